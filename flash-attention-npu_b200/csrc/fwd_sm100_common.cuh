// Argument block shared by the tcgen05 forward kernels: two query tiles a CTA and head dims above 128 (fwd_sm100.cu),
// capped scores (fwd_single_sm100.cu).
#pragma once
#include "fa_utils.cuh"
#include "fa_internal.h"
#include "sm100_ptx.cuh"
#include "tree_mask.cuh"

namespace fa {

struct alignas(64) Sm100FwdArgs {
    CUtensorMap tq, tk, tv;
    void* o;
    float* lse;
    int64_t o_sb, o_ss, o_sh;
    int64_t lse_sb, lse_sh, lse_ss;
    const int32_t* cu_q;
    const int32_t* cu_k;
    // KV-cache calls: device-resident lengths, page table, cache row of a batch entry
    const int32_t* seqused_k;
    const int32_t* block_table;
    const int32_t* cache_batch_idx;
    int64_t bt_stride;
    int page_size, s_new;
    int b, sq, sk, hq, hkv;
    int d;                               // the call's head dim (a multiple of 8): the kernels run the next of 64 / 128 / 192 / 256, the tile copies
                                         // zero-fill the columns past d and the epilogue stores d columns
    float scale_log2;
    int causal, wl, wr;
    // score transforms of the BIAS instantiation: softcap (0 = off) and alibi slopes ((hq) or (b,hq), null = off)
    float softcap, cap_in;               // cap_in = scale / softcap
    const float* alibi;
    int64_t alibi_sb;
    int kv_box;                          // rows of one K/V copy: 128, or 64 when pages are an odd multiple of 64 tokens
    int gq;                              // two-tile kernel: 1, or the query group size when a KV head's heads are stacked into the tile rows
    // split-KV (two-tile kernel, cache calls): split s of a sequence takes keys [s * keys_per_split, (s + 1) * ...) and
    // leaves a normalised fp32 partial output and its LSE for the combine kernel (nsplit = 1: final output directly)
    int nsplit, keys_per_split;          // keys_per_split is a multiple of 128
    float* o_part;                       // (nsplit, rows_all, D), rows_all = batch * sq * hq, row = (b * sq + qpos) * hq + head
    float* lse_part;                     // (nsplit, rows_all)
    int64_t rows_all;
    int chunk, nheads_grid;              // grid order, see the kernels: (batch entry, head) pairs a chunk; heads of the grid
    // A tree of drafted tokens behind the cached rows (tree_mask.cuh).  tq covers the stacked copy of q, (dim, KV head,
    // token x group, batch); rows of a tile are stacked rows, of which gq (any number) make a token.
    // TREE instantiations: splits share out the rows that the sequence has (tree_split_tiles), min_split_keys at least.
    TreeMask tree;
    int min_split_keys;
    // tree_sm100.cu: the key tiles of all sequences in one list, cut into tree_shares parts, min_split_tiles each at least
    int tree_blocks;                     // row blocks of a KV head
    int tree_shares, min_split_tiles;
};

// TREE: where the kv_box rows (what divides a page) from cache row `row` on live: (row, outermost coordinate) of the K / V maps.
// A row past the table or on a page that is not in the cache lies outside the maps: zeros.
__device__ __forceinline__ int2 tree_box(const Sm100FwdArgs& a, int row, int b) {
    if (!a.block_table) return make_int2(row, a.cache_batch_idx ? a.cache_batch_idx[b] : b);
    return make_int2(row % a.page_size, row < a.sk ? a.block_table[(int64_t)b * a.bt_stride + row / a.page_size] : -1);
}
// box number `part` of a tile
template <int NSUB>
__device__ __forceinline__ void tree_copy_box(const Sm100FwdArgs& a, const CUtensorMap* map, uint32_t dst, uint32_t full, int2 box, int part, int hk) {
#pragma unroll
    for (int s = 0; s < NSUB; ++s) sm100::tma_load_4d(dst + s * 128 * 128 + part * a.kv_box * 128, map, full, s * 64, hk, box.x, box.y);
}
// A key tile, one lane a box: `box` is the lane's, of the tile's row lane * kv_box.  The whole warp calls it.
template <int NSUB>
__device__ __forceinline__ void tree_copy_tile(const Sm100FwdArgs& a, const CUtensorMap* map, uint32_t dst, uint32_t full, int2 box, int hk, int lane) {
    if (lane == 0) sm100::mbar_expect_tx(full, NSUB * 128 * 128);
    __syncwarp();
    if (lane < 128 / a.kv_box) tree_copy_box<NSUB>(a, map, dst, full, box, lane, hk);
    __syncwarp();
}
// ... with the lane's box looked up: the tile at cache row `pos`
template <int NSUB>
__device__ __forceinline__ void tree_load_tile(const Sm100FwdArgs& a, const CUtensorMap* map, uint32_t dst, uint32_t full, int pos, int hk, int b, int lane) {
    int2 box = make_int2(0, 0);
    if (lane < 128 / a.kv_box) box = tree_box(a, pos + lane * a.kv_box, b);
    tree_copy_tile<NSUB>(a, map, dst, full, box, hk, lane);
}
// TREE: rows of the V tile at cache row n0 that no token sees may hold anything, NaN included, and 0 x NaN is NaN: rows in
// front of every window, drafted tokens that are not there, rows behind the draft.  The whole warp calls it.
template <int NSUB>
__device__ __forceinline__ void tree_clear_rows(const Sm100FwdArgs& a, unsigned char* v, int n0, int L, int b, int lane) {
    const int first = tree_first_any(a.tree, L);
    if (n0 >= first && n0 + 128 <= L) return;
    uint32_t gone[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int row = n0 + w * 32 + lane, s = row - L;
        const bool seen = s < 0 ? row >= first : s < a.tree.tokens && (a.tree.keys[b * a.tree.words + (s >> 5)] >> (s & 31) & 1);
        gone[w] = __ballot_sync(0xffffffffu, !seen);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (!gone[w]) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int chunk = i * 32 + lane;                     // 16-byte chunks of rows 32 w .. 32 w + 31, eight a row whatever the swizzle
            if (gone[w] >> (chunk >> 3) & 1) {
#pragma unroll
                for (int s = 0; s < NSUB; ++s) *reinterpret_cast<uint4*>(v + s * 128 * 128 + w * 4096 + chunk * 16) = make_uint4(0, 0, 0, 0);
            }
        }
    }
    sm100::fence_proxy_async_smem();
    __syncwarp();
}

// capped scores, head dims up to 128: one query tile a CTA, two CTAs an SM (fwd_single_sm100.cu)
int launch_fwd_single_sm100(const fa_fwd_params& p, Sm100FwdArgs& a, bool tree = false);
int fwd_single_error_flag(bool clear);
// drafted tokens, head dims up to 128 (tree_sm100.cu)
int launch_tree_sm100(const fa_fwd_params& p, const Sm100FwdArgs& a, bool dual);
int tree_sm100_error_flag(bool clear);

}  // namespace fa
