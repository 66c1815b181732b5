// Rotary embedding of q and k with one to four position axes, forward and backward (rotary_axes.cuh has the formula; the
// backward turns by the negative angle).  The reference only rotates inside its cache call (flash_attn_npu_interface.py:1469),
// by one position a token.
//
// Bound by HBM: (Hq + Hkv) D elements a token are read and written once, 4 bytes each way together.  One launch does q and k,
// so that the tables and positions are looked up once a token: a thread keeps the eight cosines and sines of its unit (two
// 16- or 8-byte chunks that hold each other's partners) in registers and walks over heads.  16384 tokens of 32 + 8 heads of 128, bf16,
// q and k slices of one projection: 59.3 us a direction, 86 % of the copy rate; 57.0 with one axis, 6.3 for 512 tokens, 4.3 for 33.
#include <cstring>
#include "fa_utils.cuh"
#include "fa_internal.h"
#include "rotary_axes.cuh"

namespace fa {

namespace {

struct RotaryArgs {
    RotaryAxes ro;
    fa_tensor src[2], dst[2];        // q, k
    int heads[2];                    // heads of k: 0 = no k
    int d, unit, units;              // elements of a thread's unit, units of a head's row
    int lanes_h, iters, groups;      // heads side by side in a CTA's row of threads, one after the other in a thread; groups of them
    uint32_t tokens, all_tokens;     // of a sequence, of all
    int in_place;                    // columns behind the rotated ones stay where they are
    float sign;                      // -1: turn back
};

// 64 threads: 59.7 us for the above; 128: 59.8, 256: 73
constexpr int kThreads = 64;

// thread -> (unit, head lane) of a token; blockIdx.x: token x group of heads.  W: elements of a chunk, 0: element by element
template <typename T, typename TT, int W>
__global__ void __launch_bounds__(kThreads) rotary_axes_kernel(const __grid_constant__ RotaryArgs a) {
    const int heads = a.heads[0] + a.heads[1], slot_threads = a.units * a.lanes_h, slots = kThreads / slot_threads;
    if ((int)threadIdx.x >= slots * slot_threads) return;
    const uint32_t slot = blockIdx.x * (uint32_t)slots + threadIdx.x / slot_threads;
    const uint32_t token = slot / (uint32_t)a.groups;
    if (token >= a.all_tokens) return;
    const int group = (int)(slot - token * (uint32_t)a.groups);
    const int in_slot = threadIdx.x % slot_threads;
    const int u = in_slot % a.units, hl = in_slot / a.units;
    const int b = (int)(token / (uint32_t)a.tokens), t = (int)(token - (uint32_t)b * (uint32_t)a.tokens);
    const RotaryRows rows = rotary_rows(a.ro, b, t);
    const bool turned = u < (a.ro.rd + a.unit - 1) / a.unit;
    if (!turned && a.in_place) return;
    const int h0 = group * a.lanes_h * a.iters + hl;
    auto row_of = [&](int h, const T*& src, T*& dst) {
        const int w = h >= a.heads[0];
        const int hh = w ? h - a.heads[0] : h;
        const fa_tensor &x = a.src[w], &y = a.dst[w];
        src = reinterpret_cast<const T*>(x.ptr) + (int64_t)b * x.stride_b + (int64_t)t * x.stride_s + (int64_t)hh * x.stride_h;
        dst = reinterpret_cast<T*>(y.ptr) + (int64_t)b * y.stride_b + (int64_t)t * y.stride_s + (int64_t)hh * y.stride_h;
    };
    if constexpr (W > 0) {
        using C = typename ChunkOf<W>::type;
        int lo = 2 * u, hi = 2 * u + 1;
        if (turned) unit_chunks<W>(a.ro, u, lo, hi);
        const bool two = hi < a.d / W;
        // heads in flight: 2, read and written past the caches' usual policy (nothing comes back for them): 59.3 us for the above;
        // without that 61.4, with 1 / 4 / 5 heads 65.6 / 65.8 / 69, with the first heads fetched before the tables 61.4
        constexpr int N = 2;
        C xa[N], xb[N];
        T* out[N];
        auto fetch = [&](int i) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int h = h0 + (i + k) * a.lanes_h;
                out[k] = nullptr;
                if (i + k < a.iters && h < heads) {
                    const T* src;
                    row_of(h, src, out[k]);
                    xa[k] = __ldcs(reinterpret_cast<const C*>(src) + lo);
                    if (two) xb[k] = __ldcs(reinterpret_cast<const C*>(src) + hi);
                }
            }
        };
        float c[W], s[W];
        if (turned) {
            load_angles<TT, W>(a.ro, rows, u * W, c, s);
#pragma unroll
            for (int e = 0; e < W; ++e) s[e] *= a.sign;
        }
        for (int i = 0; i < a.iters; i += N) {
            fetch(i);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                if (!out[k]) continue;
                C ya = xa[k], yb = xb[k];
                if (turned) turn_chunks<T, W>(xa[k], xb[k], c, s, a.ro.interleaved, ya, yb);
                __stcs(reinterpret_cast<C*>(out[k]) + lo, ya);
                if (two) __stcs(reinterpret_cast<C*>(out[k]) + hi, yb);
            }
        }
    } else {
        // element by element; in place every pair is written by the thread that read it: units of 8 pairs, then the rest
        for (int i = 0; i < a.iters; ++i) {
            const int h = h0 + i * a.lanes_h;
            if (h >= heads) break;
            const T* src;
            T* dst;
            row_of(h, src, dst);
            const int pairs = a.ro.rd / 2;
            for (int k = u * 8; k < min(u * 8 + 8, pairs); ++k) {
                const int e = a.ro.interleaved ? 2 * k : k, f = a.ro.interleaved ? 2 * k + 1 : k + pairs;
                const T ye = turn_elem<T, TT>(src, e, a.ro, rows, a.sign), yf = turn_elem<T, TT>(src, f, a.ro, rows, a.sign);
                dst[e] = ye;
                dst[f] = yf;
            }
            if (!a.in_place)
                for (int e = max(a.ro.rd, u * 16); e < min(a.d, u * 16 + 16); ++e) dst[e] = src[e];
        }
    }
}

// elements that can be moved at once (9000 tokens of 8 + 2 heads of 256, 72 columns turned: 24.7 us with 4, element by element 141): a multiple of them in half of rotary_dim, in a row and in every stride, and aligned tables
int chunk_of(const fa_rotary_params& r, const RotaryArgs& a) {
    uintptr_t ptrs = 0;
    int64_t counts = r.rotary_dim / 2 | r.d;
    const fa_tensor* ts[4] = {&a.src[0], &a.dst[0], &a.src[1], &a.dst[1]};
    for (int i = r.hq ? 0 : 2; i < (r.hk ? 4 : 2); ++i) {
        ptrs |= reinterpret_cast<uintptr_t>(ts[i]->ptr);
        counts |= ts[i]->stride_b | ts[i]->stride_s | ts[i]->stride_h;
    }
    const uintptr_t tables = reinterpret_cast<uintptr_t>(r.cos) | reinterpret_cast<uintptr_t>(r.sin);
    for (int w = 8; w >= 4; w /= 2)
        if (counts % w == 0 && ptrs % (2 * w) == 0 && tables % (r.table_dtype == 2 ? 16 : 2 * w) == 0) return w;
    return 0;
}

template <typename T, typename TT>
int launch(const RotaryArgs& a, int w, int64_t blocks, cudaStream_t st) {
    if (w == 8) rotary_axes_kernel<T, TT, 8><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    else if (w == 4) rotary_axes_kernel<T, TT, 4><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    else rotary_axes_kernel<T, TT, 0><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    mark_kernel(st);
    return cuda_ok(cudaGetLastError(), "rotary_axes launch");
}

int run_rotary(const fa_rotary_params& r) {
    if (r.dtype != FA_F16 && r.dtype != FA_BF16) return fail(FA_ERR_BAD_DTYPE, "only fp16 and bf16 are supported");
    if (r.table_dtype != r.dtype && r.table_dtype != 2) return fail(FA_ERR_BAD_DTYPE, "the tables must have the dtype of q or fp32");
    if (r.b < 0 || r.s < 0 || r.hq < 0 || r.hk < 0 || r.hq + r.hk <= 0) return fail(FA_ERR_BAD_SHAPE, "negative or zero size");
    if (r.d <= 0 || r.d > 256 || r.d % 2) return fail(FA_ERR_BAD_SHAPE, "head dimension must be even and at most 256");
    if (r.rotary_dim <= 0 || r.rotary_dim > r.d || r.rotary_dim % 2) return fail(FA_ERR_BAD_SHAPE, "rotary_dim must be even and <= headdim");
    if (r.seqlen_ro <= 0) return fail(FA_ERR_BAD_SHAPE, "seqlen_ro must be positive");
    if (r.axes < 1 || r.axes > kMaxAxes) return fail(FA_ERR_BAD_SHAPE, "one to four position axes");
    if (!r.cos || !r.sin || !r.positions) return fail(FA_ERR_NULL, "cos, sin or positions is null");
    if (r.hq && (!r.q.ptr || !r.q_out.ptr)) return fail(FA_ERR_NULL, "q is null");
    if (r.hk && (!r.k.ptr || !r.k_out.ptr)) return fail(FA_ERR_NULL, "k is null");
    if (r.b == 0 || r.s == 0) return FA_OK;
    RotaryArgs a = {};
    a.ro.cos = r.cos;
    a.ro.sin = r.sin;
    a.ro.positions = r.positions;
    a.ro.pos_stride_axis = r.positions_stride_axis;
    a.ro.pos_stride_b = r.positions_stride_b;
    a.ro.rd = r.rotary_dim;
    a.ro.interleaved = r.interleaved;
    a.ro.rows = r.seqlen_ro;
    a.ro.axes = r.axes;
    pack_axes(a.ro, r.axis_of_pair);
    a.src[0] = r.q; a.dst[0] = r.q_out;
    a.src[1] = r.k; a.dst[1] = r.k_out;
    a.heads[0] = r.hq; a.heads[1] = r.hk;
    a.d = r.d;
    const int w = chunk_of(r, a);
    a.unit = w == 4 ? 8 : 16;
    a.units = (r.d + a.unit - 1) / a.unit;
    a.sign = r.backward ? -1.f : 1.f;
    a.in_place = (!r.hq || r.q.ptr == r.q_out.ptr) && (!r.hk || r.k.ptr == r.k_out.ptr);
    const int heads = r.hq + r.hk;
    int side = kThreads / a.units;
    // a thread turns at least four heads, so that what it looks up pays: 46125 tokens of 4 + 1 heads of 64 with three axes 14.5 us,
    // with as many lanes as there are heads 24.8
    a.lanes_h = 1;
    while (a.lanes_h * 2 <= side && a.lanes_h < 4 && a.lanes_h * 8 <= heads) a.lanes_h *= 2;
    const int per = (heads + a.lanes_h - 1) / a.lanes_h;     // heads of a thread if a token is one slot
    const int64_t tokens = (int64_t)r.b * r.s;
    // few tokens: their heads are spread over more threads, until every SM has something to do
    int groups = 1;
    while (groups * 2 <= per && tokens * groups * a.units * a.lanes_h < (int64_t)sm_count() * 512) groups *= 2;
    a.iters = (per + groups - 1) / groups;
    a.groups = groups = (per + a.iters - 1) / a.iters;
    const int slots = kThreads / (a.units * a.lanes_h);
    const int64_t blocks = (tokens * groups + slots - 1) / slots;
    if (blocks * slots >= (1ll << 31)) return fail(FA_ERR_BAD_SHAPE, "too many tokens");
    a.tokens = (uint32_t)r.s; a.all_tokens = (uint32_t)tokens;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(r.stream);
    mark_kernel(st);
    if (r.dtype == FA_F16)
        return r.table_dtype == 2 ? launch<__half, float>(a, w, blocks, st) : launch<__half, __half>(a, w, blocks, st);
    return r.table_dtype == 2 ? launch<__nv_bfloat16, float>(a, w, blocks, st) : launch<__nv_bfloat16, __nv_bfloat16>(a, w, blocks, st);
}

}  // namespace
}  // namespace fa

extern "C" int fa_rotary_axes(const fa_rotary_params* r) {
    if (!r) return fa::fail(FA_ERR_NULL, "params is null");
    return fa::run_rotary(*r);
}
