// Attention of a tree of drafted tokens over a KV cache (speculative decoding with several continuations at once): argument
// checks, launch plan and the preparing kernel; the attention itself runs on the forward kernels with the mask of
// tree_mask.cuh.  No counterpart in the reference, whose cache calls know causal and windowed masks only.
//
// With A(t) the chain of ancestors of token t and t itself, depth(t) = |A(t)| - 1 and L the cached length:
//     S(t) = {j < L} u {L + s : s in A(t)},   O(t) = sum_{j in S(t)} softmax_j(scale q_t . k_j) v_j,   LSE(t) = ln sum e^(..)
// (with a window of `left`, without the keys more than `left` positions before position L + depth(t)).  All tokens share the
// prefix, so the T x G rows of a KV head (G = query heads a KV head) are stacked into one tile: the prefix is read once a
// call, which is what bounds it, up to about 200 rows.
#include "fa_utils.cuh"
#include "fa_internal.h"
#include "rotary_axes.cuh"
#include "sm100_ptx.cuh"
#include "tree_mask.cuh"

namespace fa {

namespace {

inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

struct TreePrepArgs {
    fa_fwd_params p;
    RotaryAxes ro;                   // rd = 0: no rotation; positions null: L + depth on every axis
    const int32_t* parents;
    int64_t parents_stride_b;
    uint32_t* bits;
    int32_t* depth;
    uint32_t* keys;
    void* q_stack;                   // (b, KV head, token x group, d)
    int words, left, g;
    int uk, uv, items_k, items_kv, items;
};

// One launch in front of the attention: ancestors of every token, the new rows into the cache (keys rotated), the queries
// rotated and stacked.  Every CTA works out the tree of its sequence itself, a thread a token, by doubling: after round k a
// token knows its 2^k nearest ancestors, so eight rounds do for any tree of 256 tokens.  (Climbing one parent a step took 18 us
// for a chain of 64 tokens.)
// TT: the tables' type, T or float
template <typename T, typename TT, bool VEC>
__global__ void __launch_bounds__(kTreeMaxTokens) tree_prep_kernel(const __grid_constant__ TreePrepArgs a) {
    // what a token has climbed to: the token there, or -1 = the cached rows, -2 = no token; and over how many
    __shared__ short s_up[2][kTreeMaxTokens], s_depth[2][kTreeMaxTokens], s_parent[kTreeMaxTokens];
    __shared__ uint32_t s_bits[2][kTreeMaxWords][kTreeMaxTokens];       // CTA 0: the tokens on that way
    __shared__ uint32_t s_stored[kTreeMaxWords];
    sm100::grid_let_next_start();
    const fa_fwd_params& p = a.p;
    const int b = blockIdx.y, tid = threadIdx.x, nt = p.sq;
    const int L = tree_prefix(p.seqused_k, b, p.sk);
    const int32_t* btab = p.block_table ? p.block_table + (int64_t)b * p.block_table_stride : nullptr;
    const bool masks = blockIdx.x == 0;
    int up = -2;
    bool stored = false;
    if (tid < nt) {
        // a parent is a token in front of its child, or -1 for the last cached row; anything else: no token here, nor below it
        const int parent = a.parents[(int64_t)b * a.parents_stride_b + tid];
        up = parent >= -1 && parent < tid ? parent : -2;
        const int pos = L + tid;                             // a row outside the cache is neither written nor seen
        stored = pos < p.sk && (uint64_t)(int64_t)(btab ? btab[pos / p.page_size] : p.cache_batch_idx ? p.cache_batch_idx[b] : b) < (uint64_t)p.kv_entries;
    }
    s_up[0][tid] = (short)up;
    s_parent[tid] = (short)up;
    s_depth[0][tid] = up >= 0;
    if (masks) {
        for (int w = 0; w < a.words; ++w) s_bits[0][w][tid] = w == tid >> 5 ? 1u << (tid & 31) : 0u;
    }
    __syncthreads();
    int cur = 0;
    for (int reach = 1; reach < nt; reach *= 2, cur ^= 1) {
        const int to = s_up[cur][tid];
        s_up[cur ^ 1][tid] = (short)(to >= 0 ? s_up[cur][to] : to);
        s_depth[cur ^ 1][tid] = (short)(s_depth[cur][tid] + (to >= 0 ? s_depth[cur][to] : 0));
        if (masks) {
            for (int w = 0; w < a.words; ++w) s_bits[cur ^ 1][w][tid] = s_bits[cur][w][tid] | (to >= 0 ? s_bits[cur][w][to] : 0u);
        }
        __syncthreads();
    }
    const int depth = s_up[cur][tid] == -1 ? s_depth[cur][tid] : -1;
    const uint32_t vote = __ballot_sync(0xffffffffu, stored && depth >= 0);
    s_depth[cur ^ 1][tid] = (short)depth;                    // read below as the final depth
    if ((tid & 31) == 0) s_stored[tid >> 5] = vote;
    __syncthreads();
    const short* s_final = s_depth[cur ^ 1];
    if (masks) {
        if (tid < nt) {
            uint32_t* row = a.bits + (int64_t)(b * nt + tid) * a.words;
            if (a.left < 0 || a.left >= depth) {
                for (int w = 0; w < a.words; ++w) row[w] = depth >= 0 ? s_bits[cur][w][tid] & s_stored[w] : 0u;
            } else {                                         // a window that ends inside the tree: its first left + 1 tokens
                uint32_t seen[kTreeMaxWords];
#pragma unroll
                for (int i = 0; i < kTreeMaxWords; ++i) seen[i] = 0;
                for (int at = tid, steps = 0; steps <= a.left; at = s_parent[at], ++steps) {
#pragma unroll
                    for (int i = 0; i < kTreeMaxWords; ++i)
                        if (i == at >> 5) seen[i] |= 1u << (at & 31);
                }
#pragma unroll
                for (int i = 0; i < kTreeMaxWords; ++i)
                    if (i < a.words) row[i] = seen[i] & s_stored[i];
            }
            a.depth[b * nt + tid] = depth;
        }
        if ((tid & 31) == 0 && (tid >> 5) < a.words) a.keys[b * a.words + (tid >> 5)] = vote;
    }
    const int item = blockIdx.x * kTreeMaxTokens + tid;
    if (item >= a.items) return;
    const bool is_q = item >= a.items_kv, is_v = !is_q && item >= a.items_k;
    const int at = is_q ? item - a.items_kv : is_v ? item - a.items_k : item;
    const int heads = is_q ? p.hq : p.hkv, units = is_v ? a.uv : a.uk, n = is_v ? p.dv : p.d;
    const int u = at % units, h = at / units % heads, t = at / units / heads;
    const T* src;
    T* dst;
    if (is_q) {
        const int hk = h / a.g;
        src = reinterpret_cast<const T*>(p.q.ptr) + (int64_t)b * p.q.stride_b + (int64_t)t * p.q.stride_s + (int64_t)h * p.q.stride_h;
        dst = reinterpret_cast<T*>(a.q_stack) + (((int64_t)b * p.hkv + hk) * nt * a.g + (int64_t)t * a.g + h % a.g) * p.d;
    } else {
        if (!(s_stored[t >> 5] >> (t & 31) & 1)) return;
        const int pos = L + t;
        int64_t outer, rin;
        if (btab) {
            outer = btab[pos / p.page_size];
            rin = pos % p.page_size;
        } else {
            outer = p.cache_batch_idx ? p.cache_batch_idx[b] : b;
            rin = pos;
        }
        const fa_tensor& from = is_v ? p.v_new : p.k_new;
        const fa_tensor& to = is_v ? p.v : p.k;
        src = reinterpret_cast<const T*>(from.ptr) + (int64_t)b * from.stride_b + (int64_t)t * from.stride_s + (int64_t)h * from.stride_h;
        dst = reinterpret_cast<T*>(to.ptr) + outer * to.stride_b + rin * to.stride_s + (int64_t)h * to.stride_h;
    }
    const int rd = is_v ? 0 : a.ro.rd;
    RotaryRows rows = {};
    if (rd) rows = a.ro.positions ? rotary_rows(a.ro, b, t) : same_row(a.ro, L + max((int)s_final[t], 0));
    if constexpr (VEC) {
        const uint4* s4 = reinterpret_cast<const uint4*>(src);
        uint4* d4 = reinterpret_cast<uint4*>(dst);
        if (u < rd / 16) {
            int lo, hi;
            unit_chunks(a.ro, u, lo, hi);
            float c[8], s[8];
            load_angles<TT>(a.ro, rows, u * 8, c, s);
            uint4 ya, yb;
            turn_chunks<T>(s4[lo], s4[hi], c, s, a.ro.interleaved, ya, yb);
            d4[lo] = ya;
            d4[hi] = yb;
        } else {
            const uint4 x = s4[2 * u];
            if (2 * u + 1 < n / 8) d4[2 * u + 1] = s4[2 * u + 1];
            d4[2 * u] = x;
        }
    } else {
        for (int e = u * 16; e < min(n, u * 16 + 16); ++e) dst[e] = rd ? turn_elem<T, TT>(src, e, a.ro, rows, 1.f) : src[e];
    }
}

constexpr long kMaxGridY = 65535;

struct TreePlan {
    int nsplit, min_keys, words, sm100, shared, shares;
    size_t bits, depth, keys, q, o, lse, total;
};

// tree_sm100.cu: lanes (row blocks of KV heads), and into how many shares the list of key tiles is cut.  All CTAs do about the
// same and an SM holds one, so a call takes as long as its rounds of CTAs, each 1 / n of the list; a round also costs its start
// and its ends, put at 8 % of what the call takes at best.  8 lanes: 18 shares (144 of 148 SMs); 40 lanes: 7 (two rounds).
long lanes_of(const fa_fwd_params& p) {
    const long rows = (long)p.sq * (p.hq / p.hkv);
    return p.hkv * (rows <= 128 ? 1 : (rows + 255) / 256);
}
int shares_of(const fa_fwd_params& p) {
    const long lanes = lanes_of(p), sms = sm_count();
    long best = 1;
    double best_cost = (double)((lanes + sms - 1) / sms) * (1. + 0.08 * lanes / sms);
    for (int rounds = 1; rounds <= 3; ++rounds) {            // the most shares that so many rounds have room for
        const long n = rounds * sms / lanes;
        const double cost = n ? rounds * (1. / n + 0.08 * lanes / sms) : best_cost;
        if (cost < best_cost) { best = n; best_cost = cost; }
    }
    return (int)best;
}

// Splits of the keys.  min_keys: what a split, or a CTA's share of the key tiles, has at least.
void plan_tree(const fa_fwd_params& p, TreePlan& plan) {
    plan = {};
    const long rows = (long)p.sq * (p.hq / p.hkv);
    plan.words = (p.sq + 31) / 32;
    plan.sm100 = fwd_sm100_tree_supported(p) ? 1 : 0;
    plan.shared = plan.sm100 && fwd_sm100_tree_shared(p);
    plan.min_keys = plan.shared ? 256 : 512;
    const long base = plan.sm100 ? fwd_sm100_tree_ctas(p) : (long)p.b * p.hkv * ((rows + kGenericBM - 1) / kGenericBM);
    const long most = ((long)p.sk + plan.min_keys - 1) / plan.min_keys;
    // Splits of the kernels that do not share out the tiles: as many as run side by side, where that is enough of them, else two
    // rounds of CTAs (four of the generic kernel's), whose rest falls on SMs that short sequences left.  Head dim 256, one CTA an
    // SM, 5 / 8 / 12 / 16 sequences of 8 heads: 3 splits 81 us (8: 106), 2 96 (5: 109), 4 111 (1: 130), 3 140 (1: 165); capped at
    // head dim 128, two CTAs an SM: 7 59 (8: 78), 4 74 (5: 86), 3 79 (7: 81), 5 105 (2: 122)
    const long resident = plan.sm100 ? fwd_sm100_tree_resident(p) : 1, slots = resident * sm_count();
    const long waves = plan.sm100 ? 2 : 4;
    long n = p.num_splits > 0 ? p.num_splits : plan.sm100 && base * (resident + 1) <= slots ? slots / base : (waves * slots + base - 1) / base;
    if (n > most) n = most;
    if (n > 256) n = 256;
    if (n > 65535 / p.b) n = 65535 / p.b;                    // the general kernel's grid, and
    if (plan.sm100 && n > kMaxGridY / ((rows + 127) / 128)) n = kMaxGridY / ((rows + 127) / 128);       // the tcgen05 kernels': row blocks x splits
    plan.nsplit = (int)(n < 1 ? 1 : n);
    const size_t toks = (size_t)p.b * p.sq;
    plan.bits = 0;
    plan.depth = align256(toks * plan.words * 4);
    plan.keys = plan.depth + align256(toks * 4);
    plan.q = plan.keys + align256((size_t)p.b * plan.words * 4);
    plan.o = plan.q + align256(toks * p.hq * p.d * 2);
    if (plan.shared) {                                       // at most two pieces a CTA
        plan.shares = shares_of(p);
        // a call that asks for n splits gets shares of at least that part of the longest sequence
        if (p.num_splits > 0) plan.min_keys = (int)((((long)p.sk + 127) / 128 + p.num_splits - 1) / p.num_splits) * 128;
        const size_t pieces = plan.shares == 1 ? 0 : (size_t)lanes_of(p) * plan.shares * 2 * (rows <= 128 ? 128 : 256);
        plan.lse = plan.o + align256(pieces * (p.d <= 64 ? 64 : 128) * 4);      // partials have the kernel's head dim
        plan.total = plan.lse + align256(pieces * 4);
        return;
    }
    plan.lse = plan.o + (plan.nsplit > 1 ? align256((size_t)plan.nsplit * toks * p.hq * p.d * 4) : 0);
    plan.total = plan.lse + (plan.nsplit > 1 ? align256((size_t)plan.nsplit * toks * p.hq * 4) : 0);
}

bool tree_vec_ok(const fa_fwd_params& p) {
    if (!p.rotary_cos) return true;
    return p.rotary_dim % 16 == 0 && ((reinterpret_cast<uintptr_t>(p.rotary_cos) | reinterpret_cast<uintptr_t>(p.rotary_sin)) & 15) == 0;
}

template <typename T, typename TT>
void launch_prep(const TreePrepArgs& a, dim3 grid, cudaStream_t st) {
    if (tree_vec_ok(a.p)) tree_prep_kernel<T, TT, true><<<grid, kTreeMaxTokens, 0, st>>>(a);
    else tree_prep_kernel<T, TT, false><<<grid, kTreeMaxTokens, 0, st>>>(a);
}

int check_tensor(const char* name, const fa_tensor& t) {
    if (!t.ptr) return fail(FA_ERR_NULL, "%s is null", name);
    if (reinterpret_cast<uintptr_t>(t.ptr) & 15) return fail(FA_ERR_MISALIGNED, "%s must be 16-byte aligned", name);
    if ((t.stride_b % 8) || (t.stride_s % 8) || (t.stride_h % 8))
        return fail(FA_ERR_MISALIGNED, "%s strides must be multiples of 8 elements (16 bytes)", name);
    return FA_OK;
}

int check_tree(const fa_tree_params& t) {
    const fa_fwd_params& p = t.fwd;
    if (p.dtype != FA_F16 && p.dtype != FA_BF16) return fail(FA_ERR_BAD_DTYPE, "only fp16 and bf16 are supported");
    if (p.b < 0 || p.sq < 0 || p.sk < 0 || p.hq <= 0 || p.hkv <= 0) return fail(FA_ERR_BAD_SHAPE, "negative or zero size");
    if (p.hq % p.hkv) return fail(FA_ERR_BAD_SHAPE, "number of heads in q must be divisible by the number of heads in k/v");
    if (p.sk > kTreeMaxRows) return fail(FA_ERR_BAD_SHAPE, "a sequence of the cache has at most 2^31 - 1024 rows");
    if (p.hkv > 65535 || p.b > 65535) return fail(FA_ERR_BAD_SHAPE, "at most 65535 sequences and KV heads");
    if ((int64_t)p.sq * (p.hq / p.hkv) > kMaxGridY * 128 || (int64_t)p.sq * (p.hq + 2ll * p.hkv) * 16 > (1ll << 31) - 512)
        return fail(FA_ERR_BAD_SHAPE, "at most 2^27 heads of tokens a sequence, 8388480 of them a KV head");
    if (p.d <= 0 || p.d > 256 || p.d != p.dv || p.d % 8) return fail(FA_ERR_BAD_SHAPE, "head dimension must be a multiple of 8 in [8, 256], the same for q, k and v");
    if (p.sq > kTreeMaxTokens) return fail(FA_ERR_UNSUPPORTED, "at most %d drafted tokens a sequence", kTreeMaxTokens);
    if (p.cu_seqlens_q || p.cu_seqlens_k) return fail(FA_ERR_UNSUPPORTED, "drafted tokens are not packed");
    if (p.alibi_slopes) return fail(FA_ERR_UNSUPPORTED, "alibi is not supported with a tree of tokens");
    if (p.kv_begin || p.kv_end > 0 || p.partials_only) return fail(FA_ERR_UNSUPPORTED, "key ranges are not supported with a tree of tokens");
    if (p.num_splits < 0) return fail(FA_ERR_BAD_SHAPE, "num_splits must be >= 0");
    if (!(p.scale == p.scale) || p.softcap < 0.f) return fail(FA_ERR_BAD_SHAPE, "bad softmax_scale or softcap");
    if (int e = check_tensor("q", p.q)) return e;
    if (int e = check_tensor("k", p.k)) return e;
    if (int e = check_tensor("v", p.v)) return e;
    if (int e = check_tensor("out", p.o)) return e;
    if (!p.seqused_k) return fail(FA_ERR_NULL, "cache_seqlens is null");
    if (!t.parents) return fail(FA_ERR_NULL, "tree_parents is null");
    if (p.block_table && p.page_size <= 0) return fail(FA_ERR_BAD_SHAPE, "page_size must be positive");
    if (p.block_table && p.cache_batch_idx) return fail(FA_ERR_UNSUPPORTED, "cache_batch_idx is not used with a paged cache");
    if (p.kv_entries <= 0) return fail(FA_ERR_BAD_SHAPE, "the number of pages or cache entries must be given");
    if (!p.block_table && !p.cache_batch_idx && p.kv_entries < p.b) return fail(FA_ERR_BAD_SHAPE, "the cache has fewer entries than the batch");
    if ((p.k_new.ptr != nullptr) != (p.v_new.ptr != nullptr)) return fail(FA_ERR_NULL, "k and v must be passed together");
    if (p.k_new.ptr) {
        if (int e = check_tensor("k_new", p.k_new)) return e;
        if (int e = check_tensor("v_new", p.v_new)) return e;
    }
    if ((p.rotary_cos != nullptr) != (p.rotary_sin != nullptr)) return fail(FA_ERR_NULL, "rotary_cos and rotary_sin go together");
    if (p.rotary_cos) {
        if (p.rotary_dim <= 0 || p.rotary_dim > p.d || (p.rotary_dim % 2)) return fail(FA_ERR_BAD_SHAPE, "rotary_dim must be even and <= headdim");
        if (p.seqlen_ro <= 0) return fail(FA_ERR_BAD_SHAPE, "seqlen_ro must be positive");
        if (t.axes < 1 || t.axes > kMaxAxes) return fail(FA_ERR_BAD_SHAPE, "one to four position axes");
    }
    return FA_OK;
}

int run_tree(const fa_tree_params& t) {
    fa_fwd_params p = t.fwd;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(p.stream);
    TreePlan plan;
    plan_tree(p, plan);
    if (!p.workspace || p.workspace_bytes < plan.total)
        return fail(FA_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", plan.total, p.workspace_bytes);
    if (reinterpret_cast<uintptr_t>(p.workspace) & 15) return fail(FA_ERR_MISALIGNED, "the workspace must be 16-byte aligned");
    char* ws = reinterpret_cast<char*>(p.workspace);
    mark_kernel(st);

    TreePrepArgs a = {};
    a.p = p;
    if (p.rotary_cos) {
        a.ro.cos = p.rotary_cos;
        a.ro.sin = p.rotary_sin;
        a.ro.positions = t.positions;
        a.ro.pos_stride_axis = t.positions_stride_axis;
        a.ro.pos_stride_b = t.positions_stride_b;
        a.ro.rd = p.rotary_dim;
        a.ro.interleaved = p.rotary_interleaved;
        a.ro.rows = p.seqlen_ro;
        a.ro.axes = t.axes;
        pack_axes(a.ro, t.axis_of_pair);
    }
    a.parents = t.parents;
    a.parents_stride_b = t.parents_stride_b;
    a.bits = reinterpret_cast<uint32_t*>(ws + plan.bits);
    a.depth = reinterpret_cast<int32_t*>(ws + plan.depth);
    a.keys = reinterpret_cast<uint32_t*>(ws + plan.keys);
    a.q_stack = ws + plan.q;
    a.words = plan.words;
    a.left = p.window_left;
    a.g = p.hq / p.hkv;
    a.uk = (p.d + 15) / 16;
    a.uv = (p.dv + 15) / 16;
    a.items_k = p.k_new.ptr ? p.sq * p.hkv * a.uk : 0;
    a.items_kv = a.items_k + (p.k_new.ptr ? p.sq * p.hkv * a.uv : 0);
    a.items = a.items_kv + p.sq * p.hq * a.uk;
    const dim3 grid((a.items + kTreeMaxTokens - 1) / kTreeMaxTokens, p.b);
    const bool fp32 = p.rotary_cos && t.tables_fp32;
    if (p.dtype == FA_F16) fp32 ? launch_prep<__half, float>(a, grid, st) : launch_prep<__half, __half>(a, grid, st);
    else fp32 ? launch_prep<__nv_bfloat16, float>(a, grid, st) : launch_prep<__nv_bfloat16, __nv_bfloat16>(a, grid, st);
    mark_kernel(st);
    if (int e = cuda_ok(cudaGetLastError(), "tree_prep launch")) return e;

    TreeMask mask = {a.bits, a.depth, a.keys, p.sq, plan.words, p.window_left};
    const int64_t rows = (int64_t)p.sq * a.g;
    p.q.ptr = a.q_stack;
    p.q.stride_s = p.d;
    p.q.stride_h = rows * p.d;
    p.q.stride_b = p.hkv * rows * p.d;
    float* o_part = plan.shared || plan.nsplit > 1 ? reinterpret_cast<float*>(ws + plan.o) : nullptr;
    float* lse_part = plan.shared || plan.nsplit > 1 ? reinterpret_cast<float*>(ws + plan.lse) : nullptr;
    if (plan.shared) return launch_fwd_sm100_tree(p, mask, 1, plan.min_keys, plan.shares, o_part, lse_part);
    const int e = plan.sm100 ? launch_fwd_sm100_tree(p, mask, plan.nsplit, plan.min_keys, 1, o_part, lse_part)
                             : launch_fwd_generic_tree(p, mask, plan.nsplit, plan.min_keys, o_part, lse_part);
    if (e) return e;
    return plan.nsplit > 1 ? launch_fwd_combine(p, plan.nsplit, o_part, lse_part, 0) : FA_OK;
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" {

int fa_tree_fwd_kvcache(const fa_tree_params* t) {
    if (!t) return fail(FA_ERR_NULL, "params is null");
    if (int e = check_tree(*t)) return e;
    if (t->fwd.b == 0 || t->fwd.sq == 0) return FA_OK;
    return run_tree(*t);
}

size_t fa_tree_workspace_bytes(const fa_tree_params* t) {
    if (!t || t->fwd.b <= 0 || t->fwd.sq <= 0 || t->fwd.hq <= 0 || t->fwd.hkv <= 0 || t->fwd.d <= 0 || t->fwd.sk < 0 ||
        t->fwd.hq % t->fwd.hkv) return 0;
    TreePlan plan;
    plan_tree(t->fwd, plan);
    return plan.total;
}

}  // extern "C"
