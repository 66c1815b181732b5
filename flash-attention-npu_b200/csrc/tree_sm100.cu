// Attention of drafted tokens over a cache on the tcgen05 tensor cores, head dims up to 128, sm_100a.
//
// What the two-tile forward (fwd_sm100.cu) does for a block of queries, for the stacked rows of a KV head (tree_mask.cuh), with
// the work laid out for a cache that has to be streamed once: lengths in a batch differ by factors, they are on the device, and
// a CTA a (sequence, head, split) leaves SMs idle for as long as the longest takes.  Here one CTA runs on each SM and takes an
// equal share of the key tiles.  A lane is one of the up to 256 (128) rows of a KV head; all lanes have the same list of key
// tiles, sequence after sequence, which is cut into equal shares, a CTA each.  The CTAs of all lanes for the same share are
// neighbours in the grid: they read the heads of the same cache rows, or the same rows, at the same time.  A sequence that lies
// in one share is finished there; one that the shares cut is left in pieces, at most two a CTA (the first and the last of its
// share), as normalised fp32 partials that tree_combine_kernel joins in order.  Between sequences the copies of K and V run on.
// Whole calls, graph replays, H32/8 D128: 64 tokens x 8 sequences up to 32768 rows 199 us with a CTA a split, 166 so; 26 x 16 up to
// 8192 rows 93 / 81 (337 MB: 4.1 TB/s; inside a CTA tiles come at the memory's pace, 20 us are start, ends and the two kernels
// around it).
//
// DUAL: lanes of up to 128 rows.  Both softmax groups work on the same rows, group x on key tiles x, x + 2, .. of the piece,
// and merge their results at its end.  Otherwise group x has rows 128 x .. 128 x + 127 and every tile.
//   warps 0-3 / 4-7   softmax groups (thread = row)
//   warp 8            copies, one lane a box
//   warp 9            tensor-memory allocation, MMA issue
// Tensor memory: S_0 | S_1 | O_0 | O_1, 128 columns each; P overwrites its scores.  Every wait is bounded.
#include "fwd_sm100_common.cuh"
#include "error_flags.h"

namespace fa {

using namespace sm100;

__device__ int g_tree_sm100_error = 0;

int tree_sm100_error_flag(bool clear) {
    int v = 0;
    cudaMemcpyFromSymbol(&v, g_tree_sm100_error, sizeof(int));
    if (clear) { int z = 0; cudaMemcpyToSymbol(g_tree_sm100_error, &z, sizeof(int)); }
    return v;
}

namespace {

template <int D, bool DUAL>
struct TreeSmem {
    static constexpr int kSub = 128 * 128;
    static constexpr int kTile = (D / 64) * kSub;            // a Q, K or V tile
    static constexpr int kQ = DUAL ? 1 : 2;
    static constexpr int kStages = DUAL ? 3 : 2;
    static constexpr int oQ = 0;
    static constexpr int oK = oQ + kQ * kTile;
    static constexpr int oV = oK + kStages * kTile;
    static constexpr int oMerge = oV + kStages * kTile;      // DUAL: [2 groups][exponent base, row sum][128]
    static constexpr int oBar = oMerge + (DUAL ? 2 * 2 * 128 * 4 : 0);
    static constexpr int kBytes = oBar + 224;
    // Tiles start at a multiple of 1024 bytes.  Dynamic shared memory does too where a kernel has no other, as here; three stages
    // at head dim 128 leave no room for 1024 bytes in case it did not, so the kernel checks.
    static constexpr int kSlack = 512;
    static_assert(kBytes + kSlack <= 232448, "shared memory limit of a CTA");
};
// F / E: buffer full / free.  S: scores done; P, P2: first / second half of P stored; O: all P V of a piece done; OE: O read
enum { R_Q = 0, R_QE, R_KF0, R_KE0 = R_KF0 + 3, R_VF0 = R_KE0 + 3, R_VE0 = R_VF0 + 3, R_S0 = R_VE0 + 3, R_P0 = R_S0 + 2, R_P20 = R_P0 + 2,
       R_O0 = R_P20 + 2, R_OE0 = R_O0 + 2, R_DRAIN = R_OE0 + 2, R_COUNT };

// One sequence's part in a CTA's share.
struct Piece {
    int b, L, t_lo, ntiles;
    bool whole, head;            // the sequence lies in this share as a whole; its first tile does
};
// Key tiles of sequence b
__device__ __forceinline__ int tiles_of(const Sm100FwdArgs& a, int b, int& L, int& lo) {
    int n;
    L = tree_prefix(a.seqused_k, b, a.sk);
    tree_tiles(a.tree, L, (int)min((long long)L + a.sq, (long long)a.sk), lo, n);
    return n;
}
__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ int warp_prefix(int v, int lane) {       // of lanes 0 .. lane
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
    }
    return v;
}
// A sequence in the list: its tiles, and as many entries in front of them as turning to another sequence costs a CTA (the end
// of a piece, new queries: about 4 us, a tile 1.5).  Without them the CTAs with two sequences ended 6 us after those with one.
// 0 / 1 / 2 / 3 / 5 entries, whole calls on nine kinds of batches: 978, 968, 967, 952, 948 us together.
constexpr int kTurn = 4;
__device__ __forceinline__ int entries_of(int tiles) { return tiles ? tiles + kTurn : 0; }
// Entries of the sequences in front of sequence `upto`, and of all; the whole warp calls it.  The lengths are read by every warp
// that needs them, 32 a step: one round trip for a batch of 32, and nothing to wait for but the lengths themselves.
__device__ __forceinline__ void count_entries(const Sm100FwdArgs& a, int upto, int lane, int& before, int& total) {
    before = total = 0;
    for (int i = lane; i < a.b; i += 32) {
        int L, lo;
        const int n = entries_of(tiles_of(a, i, L, lo));
        total += n;
        if (i < upto) before += n;
    }
    before = warp_sum(before);
    total = warp_sum(total);
}
// Walks over a CTA's share.  Every thread keeps its own: the lengths that it reads are the same for all.
struct Walk {
    int at, end, begin, b, L, lo, n;                         // begin: where sequence b's tiles begin in the list
    __device__ __forceinline__ void sequence(const Sm100FwdArgs& a) { n = tiles_of(a, b, L, lo); }
    // -> whether there is anything to do.  The whole warp calls it.
    __device__ __forceinline__ bool start(const Sm100FwdArgs& a, int part, int lane) {
        int before, total;
        count_entries(a, 0, lane, before, total);
        const int share = tree_share(total, a.tree_shares, a.min_split_tiles);
        if ((long long)part * share >= total) return false;
        at = part * share;
        end = (int)min((long long)at + share, (long long)total);
        // the sequence that holds entry `at` < total
        for (int i0 = 0;; i0 += 32) {
            int len = 0, first = 0;
            const int mine = i0 + lane < a.b ? tiles_of(a, i0 + lane, len, first) : 0, upto = warp_prefix(entries_of(mine), lane);
            const uint32_t behind = __ballot_sync(0xffffffffu, before + upto > at);
            if (behind) {
                const int k = __ffs(behind) - 1;
                b = i0 + k;
                L = __shfl_sync(0xffffffffu, len, k);
                lo = __shfl_sync(0xffffffffu, first, k);
                n = __shfl_sync(0xffffffffu, mine, k);
                begin = before + __shfl_sync(0xffffffffu, upto, k) - n;
                return true;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
            if (i0 + 32 >= a.b) return false;                // not reached
        }
    }
    // first tile of the share in the present sequence, and how many
    __device__ __forceinline__ int first_tile() const { return max(at - begin, 0); }
    __device__ __forceinline__ int count() const { return min(begin + n, end) - max(at, begin); }
    __device__ __forceinline__ bool next(const Sm100FwdArgs& a, Piece& p) {
        while (at < end) {
            const int t = first_tile();
            p.b = b;
            p.L = L;
            p.t_lo = lo + t;
            p.ntiles = count();
            p.head = t == 0;
            p.whole = p.head && p.ntiles == n;
            at = min(begin + n, end);
            if (at < end) {
                do { ++b; sequence(a); } while (n == 0 && b + 1 < a.b);
                begin = at + kTurn;
            }
            if (p.ntiles > 0) return true;                   // else the share ends in front of the sequence's first tile
        }
        return false;
    }
};

// true in all 256 softmax threads when `pred` holds in any of them
__device__ __forceinline__ bool any_of_256(bool pred) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.or.pred p, 1, 256, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r) : "r"((uint32_t)pred) : "memory");
    return r != 0;
}

template <typename T, int D, bool DUAL>
__global__ void __launch_bounds__(384, 1) tree_sm100_kernel(const __grid_constant__ Sm100FwdArgs a) {
    using SM = TreeSmem<D, DUAL>;
    constexpr int NST = SM::kStages;
    constexpr int NSUB = D / 64;
    constexpr int KSTEPS = D / 16;
    constexpr int ROWS = DUAL ? 128 : 256;                   // rows of a lane
    constexpr uint32_t TMEM_COLS = 512;
    constexpr int FMT = Elem<T>::kDtype == FA_BF16 ? 1 : 0;
    constexpr uint32_t IDESC_QK = umma_idesc(FMT, 128, 128, 0, 0);
    constexpr uint32_t IDESC_PV = umma_idesc(FMT, 128, D, 0, 1);
    constexpr float kRescaleThreshold = 8.f;                 // exponent bases move when a row's maximum has grown by more than 2^8

    extern __shared__ unsigned char smem_raw[];
    const uint32_t sbase = (smem_addr(smem_raw) + 1023u) & ~1023u;
    unsigned char* sgen = smem_raw + (sbase - smem_addr(smem_raw));
    const uint32_t sQ = sbase + SM::oQ, sK = sbase + SM::oK, sV = sbase + SM::oV;
    const uint32_t bars = sbase + SM::oBar;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sgen + SM::oBar + 8 * R_COUNT);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sgen + SM::oBar + 8 * R_COUNT + 8);
    auto bar = [&](int i) { return bars + 8u * i; };
    static_assert(8 * R_COUNT + 12 <= 224, "room for barriers");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int* err = &g_tree_sm100_error;
    const int failed = *err;
    if (sbase - smem_addr(smem_raw) > SM::kSlack) {          // the same for all CTAs of a launch
        if (tid == 0) atomicCAS(err, 0, 114);
        grid_wait_for_previous();
        return;
    }
    const int rows_all = a.sq * a.gq;                        // stacked rows of a KV head
    const int lanes = a.hkv * a.tree_blocks, part = blockIdx.x / lanes;
    const int hk = blockIdx.x % lanes / a.tree_blocks, r0 = blockIdx.x % a.tree_blocks * ROWS;     // KV head, first stacked row
    const bool has_b = !DUAL && rows_all - r0 > 128;         // group 1 has rows
    Walk walk;
    if (!walk.start(a, part, lane) || failed) {
        grid_wait_for_previous();                            // no grid may be done before the one in front of it
        return;
    }
    Piece p;
    int ahead = 0;                                           // copy warp: tiles asked for before anything else

    if (warp == 8) {
        if (lane == 0) {
            tma_prefetch_desc(&a.tq); tma_prefetch_desc(&a.tk); tma_prefetch_desc(&a.tv);
            for (int i = 0; i < R_COUNT; ++i) {
                const bool by_rows = i >= R_P0 && i < R_O0, read = i >= R_OE0 && i < R_DRAIN;
                mbar_init(bar(i), by_rows ? 128u : read ? (DUAL ? 256u : 128u) : 1u);
            }
            *abort_flag = 0;
            mbar_fence_init();
        }
        // The first tiles are on their way while the other warps arrive and the preparing kernel still runs: those in front of
        // the draft, which it does not write.  A lane has one box of one tile, so that the page table is looked up once.
        const int from = walk.lo + walk.first_tile();
        const int parts = 128 / a.kv_box, tile = lane / parts, part_of = lane % parts;      // up to 16 parts
        ahead = max(0, min(min(NST, 32 / parts), min(walk.count(), walk.L / 128 - from)));
        const bool busy = tile < ahead;
        int2 box = make_int2(0, 0);
        if (busy) box = tree_box(a, from * 128 + lane * a.kv_box, walk.b);
        if (lane == 0) {
            for (int j = 0; j < ahead; ++j) {
                mbar_expect_tx(bar(R_KF0 + j), SM::kTile);
                mbar_expect_tx(bar(R_VF0 + j), SM::kTile);
            }
        }
        __syncwarp();
        if (busy) {
            tree_copy_box<NSUB>(a, &a.tk, sK + tile * SM::kTile, bar(R_KF0 + tile), box, part_of, hk);
            tree_copy_box<NSUB>(a, &a.tv, sV + tile * SM::kTile, bar(R_VF0 + tile), box, part_of, hk);
        }
    } else if (warp == 9) {
        tmem_alloc(smem_addr(tmem_slot), TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_let_next_start();
    grid_wait_for_previous();                                // Q, the mask and the drafted rows are there from here on

    // registers as in the two-tile forward
    static_assert(128 * 56 + 256 * 224 <= 384 * 168, "register split exceeds the CTA's allocation");
    if (warp >= 8) {
    reg_dealloc<56>();
    if (warp == 8) {
        // whole warp: lanes leave together.  The lane's box of the next tile is looked up while this one's buffers become free.
        const int parts = 128 / a.kv_box;
        auto look_up = [&](int b, int tile) { return lane < parts ? tree_box(a, tile * 128 + lane * a.kv_box, b) : make_int2(0, 0); };
        bool ok = true;
        int J = 0;
        for (int s = 0; ok && walk.next(a, p); ++s) {
            int2 box = make_int2(0, 0), next = look_up(p.b, p.t_lo);
            for (int j = 0; j < p.ntiles && ok; ++j, ++J) {
                const int st = J % NST, use = J / NST;
                const bool asked = J < ahead;
                box = next;
                if (j + 1 < p.ntiles) next = look_up(p.b, p.t_lo + j + 1);
                if (use > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar(R_KE0 + st), (use - 1) & 1, abort_flag, err, 101));
                if (!ok) break;
                if (!asked) tree_copy_tile<NSUB>(a, &a.tk, sK + st * SM::kTile, bar(R_KF0 + st), box, hk, lane);
                if (j == 0) {                                // Q of this sequence, once no score of the last one reads the buffer
                    if (s > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar(R_QE), (s - 1) & 1, abort_flag, err, 103));
                    if (!ok) break;
                    if (lane == 0) {
                        mbar_expect_tx(bar(R_Q), has_b ? 2 * SM::kTile : SM::kTile);
#pragma unroll
                        for (int x = 0; x < SM::kQ; ++x) {
                            if (x == 1 && !has_b) break;
#pragma unroll
                            for (int c = 0; c < NSUB; ++c) tma_load_4d(sQ + x * SM::kTile + c * SM::kSub, &a.tq, bar(R_Q), c * 64, hk, r0 + x * 128, p.b);
                        }
                    }
                    __syncwarp();
                }
                if (use > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar(R_VE0 + st), (use - 1) & 1, abort_flag, err, 102));
                if (!ok) break;
                if (!asked) tree_copy_tile<NSUB>(a, &a.tv, sV + st * SM::kTile, bar(R_VF0 + st), box, hk, lane);
            }
        }
    } else if (warp == 9) {
        const uint64_t dQ0 = umma_desc(sQ, 16, 1024), dK0 = umma_desc(sK, 16, 1024), dV0 = umma_desc(sV, SM::kSub, 1024);
        bool ok = true;
        int J = 0;                                           // tile number over all pieces: what the K and V buffers count
        int uses[2] = {0, 0};                                // tiles of each softmax group: what its barriers count
        // scores of tile j of the piece (number J + j) for group x
        auto scores = [&](int x, int j) {
            umma_ss_scores<KSTEPS, SM::kSub>(tmem + x * 128, umma_desc_at(dQ0, DUAL ? 0 : x * SM::kTile), umma_desc_at(dK0, ((J + j) % NST) * SM::kTile), IDESC_QK);
            umma_commit_w(bar(R_S0 + x));
        };
        auto k_ready = [&](int j) { return mbar_wait(bar(R_KF0 + (J + j) % NST), ((J + j) / NST) & 1, abort_flag, err, 107); };
        auto k_done = [&](int j) { umma_commit_w(bar(R_KE0 + (J + j) % NST)); };
        // P V of group x in two halves of 64 keys
        auto pv = [&](int x, int j, bool more) -> bool {
            const int st = (J + j) % NST, parity = uses[x] & 1;
            if (!mbar_wait(bar(R_P0 + x), parity, abort_flag, err, 105)) return false;
            tc_fence_after();
            const uint64_t bv = umma_desc_at(dV0, st * SM::kTile);
            const uint32_t d_o = tmem + 256 + x * 128, a_p = tmem + x * 128;
            umma_ts_group4<0, 8, 0, 128>(d_o, a_p, bv, IDESC_PV, more);
            if (!mbar_wait(bar(R_P20 + x), parity, abort_flag, err, 111)) return false;
            tc_fence_after();
            umma_ts_group4<32, 8, 512, 128>(d_o, a_p, bv, IDESC_PV, 1);
            ++uses[x];
            return true;
        };
        for (int s = 0; ok && walk.next(a, p); ++s) {
            const int n = p.ntiles;
            ok = mbar_wait(bar(R_Q), s & 1, abort_flag, err, 104) && k_ready(0);
            if (!ok) break;
            tc_fence_after();
            if constexpr (DUAL) {
                auto next_scores = [&](int j) -> bool {
                    if (j > 0) {
                        if (!k_ready(j)) return false;
                        tc_fence_after();
                    }
                    scores(j & 1, j);
                    k_done(j);
                    if (j + 1 == n) umma_commit_w(bar(R_QE));
                    return true;
                };
                ok = next_scores(0);
                if (ok && n > 1) ok = next_scores(1);
                for (int j = 0; j < n && ok; ++j) {
                    const int x = j & 1, st = (J + j) % NST;
                    ok = mbar_wait(bar(R_VF0 + st), ((J + j) / NST) & 1, abort_flag, err, 106);
                    if (!ok) break;
                    tree_clear_rows<NSUB>(a, sgen + SM::oV + st * SM::kTile, (p.t_lo + j) * 128, p.L, p.b, lane);
                    if (j == 0 && s > 0) ok = mbar_wait(bar(R_OE0), (s - 1) & 1, abort_flag, err, 108);
                    if (ok) ok = pv(x, j, j > 1);
                    if (!ok) break;
                    umma_commit_w(bar(R_VE0 + st));
                    if (j + 2 < n) ok = next_scores(j + 2);
                    else umma_commit_w(bar(R_O0 + x));
                }
            } else {
                scores(0, 0);
                if (has_b) scores(1, 0);
                k_done(0);
                if (n == 1) umma_commit_w(bar(R_QE));
                for (int j = 0; j < n && ok; ++j) {
                    const int st = (J + j) % NST;
                    const bool more = j + 1 < n;
                    ok = mbar_wait(bar(R_VF0 + st), ((J + j) / NST) & 1, abort_flag, err, 106);
                    if (ok && more) ok = k_ready(j + 1);
                    if (!ok) break;
                    tree_clear_rows<NSUB>(a, sgen + SM::oV + st * SM::kTile, (p.t_lo + j) * 128, p.L, p.b, lane);
                    if (j == 0) {
                        if (s > 0) ok = mbar_wait(bar(R_OE0), (s - 1) & 1, abort_flag, err, 108);
                        if (ok && has_b && s > 0) ok = mbar_wait(bar(R_OE0 + 1), (s - 1) & 1, abort_flag, err, 109);
                        if (!ok) break;
                    }
                    ok = pv(0, j, j > 0);
                    if (!ok) break;
                    if (more) scores(0, j + 1);
                    else umma_commit_w(bar(R_O0));
                    if (has_b) {
                        ok = pv(1, j, j > 0);
                        if (!ok) break;
                    }
                    umma_commit_w(bar(R_VE0 + st));
                    if (more) {
                        if (has_b) scores(1, j + 1);
                        k_done(j + 1);
                        if (j + 2 == n) umma_commit_w(bar(R_QE));
                    } else if (has_b) {
                        umma_commit_w(bar(R_O0 + 1));
                    }
                }
            }
            J += n;
        }
        // no arrive of a commit may land after the CTA has left: wait for a last one (see the two-tile forward)
        if (ok) {
            umma_commit_w(bar(R_DRAIN));
            mbar_wait(bar(R_DRAIN), 0, abort_flag, err, 113);
        }
    }
    } else {
    reg_alloc<224>();
    // -------------------------------------------------------------------- softmax group x
    const int x = warp >> 2, r = tid & 127;
    const int x0 = DUAL ? 0 : x * 128;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_base + x * 128;
    const uint32_t t_o = tmem + lane_base + 256 + x * 128;
    const float sc = a.scale_log2;
    bool ok = true;
    const int row = r0 + x0 + r;                             // stacked row of this thread
    const bool mine = row < rows_all;
    const int qi = row / a.gq;
    const int head = hk * a.gq + row - qi * a.gq;
    int uses = 0, o1 = 0;                                    // tiles of this group so far; DUAL: pieces in which group 1 had any
    for (int s = 0; ok && (DUAL || x == 0 || has_b) && walk.next(a, p); ++s) {
        // on its way until the first masked tile or the end of the piece asks for it
        const int depth = mine ? a.tree.depth[p.b * a.tree.tokens + qi] : -1;
        auto first_key = [&] { return tree_first_key(a.tree, depth, p.L); };
        const uint32_t* tree_row = a.tree.bits + (mine ? (int64_t)(p.b * a.tree.tokens + qi) * a.tree.words : 0);
        const int all_first = tree_first_all(a.tree, p.L);
        float m_used = -INFINITY, l_run = 0.f;
        const int nt = DUAL ? (p.ntiles + 1 - x) / 2 : p.ntiles;
        for (int j = 0; j < nt; ++j) {
            const int n0 = (p.t_lo + (DUAL ? 2 * j + x : j)) * 128;
            ok = mbar_wait(bar(R_S0 + x), uses & 1, abort_flag, err, 115);
            if (!ok) break;
            ++uses;
            tc_fence_after();
            uint32_t sreg[4][32];
#pragma unroll
            for (int c = 0; c < 2; ++c) tmem_ld32(t_s + c * 32, sreg[c]);
            tmem_wait_ld();
            // the second half of the row is in flight while the first half is reduced
#pragma unroll
            for (int c = 2; c < 4; ++c) tmem_ld32(t_s + c * 32, sreg[c]);
            const bool full = n0 >= all_first && n0 + 128 <= p.L;
            float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                if (hh == 1) tmem_wait_ld();
                if (!full) {
                    const int first = first_key();
#pragma unroll
                    for (int c = 2 * hh; c < 2 * hh + 2; ++c) {
                        const uint32_t vis = first != 0x7fffffff ? tree_visible32(a.tree, tree_row, n0 + c * 32, first, p.L) : 0u;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(vis >> i & 1)) sreg[c][i] = 0xff800000u;     // -inf
                    }
                }
                // four independent chains of three-input maxima, NaN when a visible score is: the polynomial exponential loses it, and
                // the inf - inf of an infinite score
#pragma unroll
                for (int c = 2 * hh; c < 2 * hh + 2; ++c) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        mx0 = max3_nan(mx0, __uint_as_float(sreg[c][i]), __uint_as_float(sreg[c][i + 1]));
                        mx1 = max3_nan(mx1, __uint_as_float(sreg[c][i + 2]), __uint_as_float(sreg[c][i + 3]));
                        mx2 = max3_nan(mx2, __uint_as_float(sreg[c][i + 4]), __uint_as_float(sreg[c][i + 5]));
                        mx3 = max3_nan(mx3, __uint_as_float(sreg[c][i + 6]), __uint_as_float(sreg[c][i + 7]));
                    }
                }
            }
            const float m_new = max_nan(max3_nan(mx0, mx1, mx2), mx3) * sc;       // log2 domain
            if (m_used == -INFINITY) m_used = m_new;
            if (j > 0 && __any_sync(0xffffffffu, m_new > m_used + kRescaleThreshold)) {
                const float m_next = fmaxf(m_used, m_new);
                const float alpha = m_used == -INFINITY ? 1.f : ex2_approx(m_used - m_next);
                m_used = m_next;
                l_run *= alpha;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t oreg[32];
                    tmem_ld32(t_o + c * 32, oreg);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) oreg[i] = __float_as_uint(__uint_as_float(oreg[i]) * alpha);
                    tmem_st32(t_o + c * 32, oreg);
                }
            }
            const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
            const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(neg_m, neg_m);
            float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
            // P is rounded to the input type, the type that V's product on the tensor cores takes; row sums stay in fp32.  That is
            // what the output's error against 64 bits comes from: 2.1e-3 to 2.3e-3 of its 2-norm in bf16, 2.9e-4 in fp16 (with P in
            // 32 bits 1.7e-3 and 2.1e-4).
            // NPOLY of every 8 pairs take the polynomial 2^x; masked tiles none of them: the special-function path maps -inf to zero
            auto exp_phase = [&](auto npoly_c) {
                constexpr int NPOLY = decltype(npoly_c)::value;
#pragma unroll
                for (int hlf = 0; hlf < 2; ++hlf) {
                    uint32_t preg[32];
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const uint32_t* src = &sreg[2 * hlf + (g >> 1)][(g & 1) * 16];
                        static_for<0, 8>([&](auto pi) {
                            constexpr bool poly = (pi.value * NPOLY) % 8 < NPOLY;
                            const float2 xv = fma2(make_float2(__uint_as_float(src[2 * pi.value]), __uint_as_float(src[2 * pi.value + 1])), sc2, nm2);
                            float2 pv;
                            if constexpr (poly) pv = ex2_poly2(xv);
                            else pv = make_float2(ex2_approx(xv.x), ex2_approx(xv.y));
                            if constexpr (pi.value & 1) sum_b = add2(sum_b, pv); else sum_a = add2(sum_a, pv);
                            preg[g * 8 + pi.value] = Elem<T>::pack(pv.x, pv.y);
                        });
                    }
                    tmem_st32(t_s + hlf * 32, preg);
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(bar((hlf ? R_P20 : R_P0) + x));
                }
            };
            if (full) exp_phase(std::integral_constant<int, D == 128 ? 1 : 2>{});
            else exp_phase(std::integral_constant<int, 0>{});
            l_run = m_new < INFINITY ? l_run + ((sum_a.x + sum_b.x) + (sum_a.y + sum_b.y)) : m_new - m_new;
        }
        // ---- end of the piece ----
        float f_a = 1.f, f_b = 0.f;                          // DUAL: weights of the two groups' results
        if constexpr (DUAL) {
            if (ok) ok = mbar_wait(bar(R_O0), s & 1, abort_flag, err, 110);
            if (ok && p.ntiles > 1) ok = mbar_wait(bar(R_O0 + 1), o1 & 1, abort_flag, err, 112);
            o1 += p.ntiles > 1;
            // What the last piece left here has been read: the accumulators are only written again after all 256 threads have
            // let go of them.
            float* merge = reinterpret_cast<float*>(sgen + SM::oMerge);
            merge[x * 256 + r] = m_used;
            merge[x * 256 + 128 + r] = l_run;
            ok = !any_of_256(!ok);                           // both groups go on, or both leave
            const float m_a = merge[r], m_b = merge[256 + r];
            m_used = fmaxf(m_a, m_b);
            f_a = m_a == -INFINITY ? 0.f : ex2_approx(m_a - m_used);
            f_b = m_b == -INFINITY ? 0.f : ex2_approx(m_b - m_used);
            l_run = merge[128 + r] * f_a + merge[384 + r] * f_b;
        } else {
            if (ok) ok = mbar_wait(bar(R_O0 + x), s & 1, abort_flag, err, 110);
        }
        if (!ok) break;
        tc_fence_after();
        const bool there = first_key() != 0x7fffffff;
        if (!there) l_run = 0.f;                             // no token: whatever its q holds, zeros and no LSE
        // a row sum of 0 says that nothing was seen; NaN stays NaN
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
        T* orow = reinterpret_cast<T*>(a.o) + (int64_t)p.b * a.o_sb + (int64_t)qi * a.o_ss + (int64_t)head * a.o_sh;
        // partials: four columns of all rows, then the next four, so that a warp's stores lie side by side
        const int64_t piece = (int64_t)blockIdx.x * 2 + (p.head ? 1 : 0);
        float4* part_o = reinterpret_cast<float4*>(a.o_part) + piece * (D / 4) * ROWS + x0 + r;
        // DUAL: each group merges and stores one half of the columns
#pragma unroll
        for (int cc = 0; cc < (DUAL ? D / 64 : D / 32); ++cc) {
            const int c = DUAL ? x * (D / 64) + cc : cc;
            uint32_t oreg[32];
            tmem_ld32((DUAL ? t_o - x * 128 : t_o) + c * 32, oreg);
            if constexpr (DUAL) {
                uint32_t ob[32];
                tmem_ld32(t_o + (1 - x) * 128 + c * 32, ob);
                tmem_wait_ld();
                const bool both = p.ntiles > 1;              // else group 1's accumulator is not this sequence's
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float v = __uint_as_float(oreg[i]) * f_a;
                    oreg[i] = __float_as_uint(both ? fmaf(__uint_as_float(ob[i]), f_b, v) : v);
                }
            } else {
                tmem_wait_ld();
            }
            if (!there) {
#pragma unroll
                for (int i = 0; i < 32; ++i) oreg[i] = 0u;
            }
            if (mine && !p.whole) {
#pragma unroll
                for (int v = 0; v < 8; ++v)
                    __stcg(part_o + (c * 8 + v) * ROWS, make_float4(__uint_as_float(oreg[4 * v]) * inv, __uint_as_float(oreg[4 * v + 1]) * inv,
                                                                    __uint_as_float(oreg[4 * v + 2]) * inv, __uint_as_float(oreg[4 * v + 3]) * inv));
            } else if (mine) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    uint4 pk;
                    pk.x = Elem<T>::pack(__uint_as_float(oreg[8 * v + 0]) * inv, __uint_as_float(oreg[8 * v + 1]) * inv);
                    pk.y = Elem<T>::pack(__uint_as_float(oreg[8 * v + 2]) * inv, __uint_as_float(oreg[8 * v + 3]) * inv);
                    pk.z = Elem<T>::pack(__uint_as_float(oreg[8 * v + 4]) * inv, __uint_as_float(oreg[8 * v + 5]) * inv);
                    pk.w = Elem<T>::pack(__uint_as_float(oreg[8 * v + 6]) * inv, __uint_as_float(oreg[8 * v + 7]) * inv);
                    if (c * 32 + v * 8 < a.d) reinterpret_cast<uint4*>(orow + c * 32)[v] = pk;
                }
            }
        }
        // the accumulators may be written again
        tc_fence_before();
        mbar_arrive(bar(DUAL ? (int)R_OE0 : R_OE0 + x));
        if (mine && !(DUAL && x)) {
            const float lse = l_run != 0.f ? (m_used + log2f(l_run)) * kLn2 : p.whole ? INFINITY : -INFINITY;
            if (!p.whole) a.lse_part[piece * ROWS + x0 + r] = lse;
            else if (a.lse) a.lse[(int64_t)p.b * a.lse_sb + (int64_t)head * a.lse_sh + (int64_t)qi * a.lse_ss] = lse;
        }
    }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        settle_after_abort(abort_flag);
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

// Rows whose sequence was cut: its pieces in shares c0 .. c1, joined in that order.  A CTA has 32 rows of a lane, a thread 4 N
// columns of one of them, a warp the same columns of its 32 rows; PHASES warps share out the pieces.
//   many rows (two CTAs an SM with D / 8 columns a thread)   D / 8 columns: 26 tokens x 16 sequences 83.2 us a call, with 8 columns 85.5
//   fewer                                                    8 columns: 16 x 8, up to 3000 rows 35.9, with 16 columns 37.1
//   fewer, 16 shares a sequence or more                      eight warps share out the pieces: one sequence of 30000 rows of two KV
//                                                            heads 24.6, one warp 31.7; two sequences in 9 shares each 46.5 / 44.1
constexpr int kCombineRows = 32;
template <typename T, int D, int ROWS, int N, int PHASES>
__global__ void __launch_bounds__(256) tree_combine_kernel(const __grid_constant__ Sm100FwdArgs a) {
    constexpr int U = 8 / N;                                 // pieces in flight
    constexpr int WIDE = 8 / PHASES, SPLIT = D / (4 * N) / WIDE;   // column groups of a CTA, CTAs of the same rows
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows_all = a.sq * a.gq, blocks = (rows_all + kCombineRows - 1) / kCombineRows;
    const int id = blockIdx.x / SPLIT, cols = blockIdx.x % SPLIT * WIDE + warp % WIDE, phase = warp / WIDE;
    const int hk = id / blocks % a.hkv, b = id / blocks / a.hkv;
    int before, total, L, lo;
    count_entries(a, b, lane, before, total);
    const int n = tiles_of(a, b, L, lo), share = tree_share(total, a.tree_shares, a.min_split_tiles), begin = before + kTurn;
    const int c0 = n ? begin / share : 0, c1 = n ? (begin + n - 1) / share : -1;
    const int row = id % blocks * kCombineRows + lane, lanes = a.hkv * a.tree_blocks;
    const int mine = hk * a.tree_blocks + row / ROWS;
    grid_wait_for_previous();
    if (c0 == c1) return;                                    // finished by its CTA
    float m = -INFINITY, tot = 0.f;
    float4 acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    // results of weights t e^w; e^w is 0 for a piece in which the row sees nothing, whose v is not used.  A piece of a row that
    // holds NaN has a NaN w, and makes m, the sum and the output NaN.
    auto add = [&](const float (&w)[U], const float (&t)[U], const float4 (&v)[U][N]) {
        float next = m;
#pragma unroll
        for (int u = 0; u < U; ++u) next = max_nan(next, w[u]);
        if (next == -INFINITY) return;
        const float f = expf(m - next);
        m = next;
        tot *= f;
#pragma unroll
        for (int i = 0; i < N; ++i) { acc[i].x *= f; acc[i].y *= f; acc[i].z *= f; acc[i].w *= f; }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (w[u] == -INFINITY) continue;
            const float e = expf(w[u] - next);
            tot += t[u] * e;
#pragma unroll
            for (int i = 0; i < N; ++i) { acc[i].x += e * v[u][i].x; acc[i].y += e * v[u][i].y; acc[i].z += e * v[u][i].z; acc[i].w += e * v[u][i].w; }
        }
    };
    if (row < rows_all) {
        float t[U];
#pragma unroll
        for (int u = 0; u < U; ++u) t[u] = 1.f;
        for (int c = c0 + phase; c <= c1; c += PHASES * U) {
            float w[U];
            float4 v[U][N];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int cu = c + u * PHASES;
                // the piece in share c: the CTA's last one where the sequence begins in its share, else its first
                const int64_t piece = (int64_t)(cu * lanes + mine) * 2 + (cu == c0 ? 1 : 0);
                w[u] = cu <= c1 ? __ldcg(a.lse_part + piece * ROWS + row % ROWS) : -INFINITY;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (cu <= c1) v[u][i] = __ldcg(reinterpret_cast<const float4*>(a.o_part) + (piece * (D / 4) + cols * N + i) * ROWS + row % ROWS);
            }
            add(w, t, v);
        }
    }
    if constexpr (PHASES > 1) {
        __shared__ float s_m[8][32], s_tot[8][32];
        __shared__ float4 s_acc[8][N][32];
        s_m[warp][lane] = m;
        s_tot[warp][lane] = tot;
#pragma unroll
        for (int i = 0; i < N; ++i) s_acc[warp][i][lane] = acc[i];
        __syncthreads();
        if (phase) return;
        m = -INFINITY;
        tot = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < PHASES; k += U) {
            float w[U], t[U];
            float4 v[U][N];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int from = (k + u) * WIDE + warp;
                const bool there = k + u < PHASES;
                w[u] = there ? s_m[from][lane] : -INFINITY;
                t[u] = there ? s_tot[from][lane] : 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (there) v[u][i] = s_acc[from][i][lane];
            }
            add(w, t, v);
        }
    }
    if (row >= rows_all) return;
    const float inv = tot == 0.f ? 0.f : 1.f / tot;
    const int qi = row / a.gq, head = hk * a.gq + row % a.gq;
    T* orow = reinterpret_cast<T*>(a.o) + (int64_t)b * a.o_sb + (int64_t)qi * a.o_ss + (int64_t)head * a.o_sh + cols * N * 4;
#pragma unroll
    for (int i = 0; i < N; i += 2)
        if ((cols * N + i) * 4 < a.d)
            reinterpret_cast<uint4*>(orow)[i / 2] = make_uint4(Elem<T>::pack(acc[i].x * inv, acc[i].y * inv), Elem<T>::pack(acc[i].z * inv, acc[i].w * inv),
                                                               Elem<T>::pack(acc[i + 1].x * inv, acc[i + 1].y * inv), Elem<T>::pack(acc[i + 1].z * inv, acc[i + 1].w * inv));
    if (cols == 0 && a.lse)
        a.lse[(int64_t)b * a.lse_sb + (int64_t)head * a.lse_sh + (int64_t)qi * a.lse_ss] = tot == 0.f ? INFINITY : m + logf(tot);
}

template <typename T, int D, bool DUAL>
int launch_t(const fa_fwd_params& p, const Sm100FwdArgs& a) {
    cudaStream_t st = reinterpret_cast<cudaStream_t>(p.stream);
    auto kern = tree_sm100_kernel<T, D, DUAL>;
    const int smem = TreeSmem<D, DUAL>::kBytes + TreeSmem<D, DUAL>::kSlack;
    if (int e = cuda_ok(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute")) return e;
    if (int e = cuda_ok(launch_early(kern, dim3((unsigned)(a.hkv * a.tree_blocks * a.tree_shares)), 384, smem, st, a), "tree_sm100 launch")) return e;
    mark_kernel(st);
    constexpr int ROWS = DUAL ? 128 : 256;
    const int64_t blocks = (int64_t)p.b * p.hkv * ((p.sq * a.gq + kCombineRows - 1) / kCombineRows);
    const bool many = blocks >= 2 * sm_count(), cut = a.tree_shares >= 16 * a.b;
    const cudaError_t e = many ? launch_early(tree_combine_kernel<T, D, ROWS, D / 32, 1>, dim3((unsigned)blocks), 256, 0, st, a)
                        : !cut ? launch_early(tree_combine_kernel<T, D, ROWS, 2, 1>, dim3((unsigned)blocks * (D / 64)), 256, 0, st, a)
                               : launch_early(tree_combine_kernel<T, D, ROWS, 2, 8>, dim3((unsigned)blocks * (D / 8)), 256, 0, st, a);
    if (int code = cuda_ok(e, "tree_combine launch")) return code;
    mark_kernel(st);
    return FA_OK;
}
template <typename T>
int launch_dims(const fa_fwd_params& p, const Sm100FwdArgs& a, bool dual) {
    if (p.d > 64) return dual ? launch_t<T, 128, true>(p, a) : launch_t<T, 128, false>(p, a);
    return dual ? launch_t<T, 64, true>(p, a) : launch_t<T, 64, false>(p, a);
}

}  // namespace

int launch_tree_sm100(const fa_fwd_params& p, const Sm100FwdArgs& a, bool dual) {
    return p.dtype == FA_F16 ? launch_dims<__half>(p, a, dual) : launch_dims<__nv_bfloat16>(p, a, dual);
}

}  // namespace fa
