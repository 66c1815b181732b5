// Rotary embedding with one to four position axes, shared by the rotary kernel and the tree attention's preparing kernel.
//
// Pair i of a head (elements i and i + rd / 2, or 2 i and 2 i + 1 when interleaved) is turned by the angle whose cosine and
// sine stand in row positions[axis(i)] of the tables, column i:  (a, b) -> (a c - b s, a s + b c).  fp32 arithmetic with
// separately rounded products and one rounding to the element type, as in the append kernel (fwd_generic.cu), so that both
// give the same bits for the same angles.
#pragma once
#include "fa_utils.cuh"

namespace fa {

constexpr int kMaxAxes = 4;

struct RotaryAxes {
    const void* cos;                 // (rows, rd / 2), the element type or fp32
    const void* sin;
    const int32_t* positions;        // (axes, batch, tokens), or null: the caller's kernel knows the position
    int64_t pos_stride_axis, pos_stride_b;
    int rd, interleaved, rows, axes;
    uint32_t axis[8];                // two bits a pair, pairs of 16 a word
};

// host: two bits a pair from a table of one byte a pair (null: axis 0 throughout)
inline void pack_axes(RotaryAxes& r, const uint8_t* axis_of_pair) {
    for (int w = 0; w < 8; ++w) r.axis[w] = 0;
    if (!axis_of_pair) return;
    for (int i = 0; i < r.rd / 2; ++i) r.axis[i >> 4] |= (uint32_t)(axis_of_pair[i] & 3) << ((i & 15) * 2);
}

#ifdef __CUDACC__
struct RotaryRows {                  // the table rows of one token
    int row[kMaxAxes];
    __device__ __forceinline__ int of(int axis) const { return axis == 0 ? row[0] : axis == 1 ? row[1] : axis == 2 ? row[2] : row[3]; }
};
// a position outside the tables takes the nearest row, as in the append kernel
__device__ __forceinline__ int clamp_row(const RotaryAxes& r, int pos) { return max(0, min(pos, r.rows - 1)); }
__device__ __forceinline__ RotaryRows rotary_rows(const RotaryAxes& r, int b, int64_t token) {
    RotaryRows p;
#pragma unroll
    for (int a = 0; a < kMaxAxes; ++a)
        p.row[a] = a < r.axes ? clamp_row(r, r.positions[a * r.pos_stride_axis + b * r.pos_stride_b + token]) : 0;
    return p;
}
__device__ __forceinline__ RotaryRows same_row(const RotaryAxes& r, int pos) {
    RotaryRows p;
#pragma unroll
    for (int a = 0; a < kMaxAxes; ++a) p.row[a] = clamp_row(r, pos);
    return p;
}
template <typename TT> __device__ __forceinline__ float table_value(const TT* t) { return Elem<TT>::to_float(*t); }
template <> __device__ __forceinline__ float table_value<float>(const float* t) { return *t; }

// Chunks of W elements, moved at once: 16 bytes, or 8 where rotary_dim / 2 is a multiple of 4 only
template <int W> struct ChunkOf;
template <> struct ChunkOf<8> { using type = uint4; };
template <> struct ChunkOf<4> { using type = uint2; };

// cosines and sines of pairs i0 .. i0 + W - 1 (i0 a multiple of W): wide loads where one axis turns all of them
template <typename TT, int W = 8>
__device__ __forceinline__ void load_angles(const RotaryAxes& r, const RotaryRows& p, int i0, float (&c)[W], float (&s)[W]) {
    const TT* cos = reinterpret_cast<const TT*>(r.cos);
    const TT* sin = reinterpret_cast<const TT*>(r.sin);
    const int half = r.rd / 2;
    const uint32_t axes = (r.axis[i0 >> 4] >> ((i0 & 15) * 2)) & ((1u << 2 * W) - 1u);
    if (axes == (axes & 3) * (0x5555u & ((1u << 2 * W) - 1u))) {
        const int64_t at = (int64_t)p.of(axes & 3) * half + i0;
        constexpr int N = W * sizeof(TT) < 16 ? W : 16 / sizeof(TT);
        using V = typename ChunkOf<N * sizeof(TT) / 2>::type;
#pragma unroll
        for (int k = 0; k < W; k += N) {
            const V vc = *reinterpret_cast<const V*>(cos + at + k), vs = *reinterpret_cast<const V*>(sin + at + k);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                c[k + e] = table_value<TT>(reinterpret_cast<const TT*>(&vc) + e);
                s[k + e] = table_value<TT>(reinterpret_cast<const TT*>(&vs) + e);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const int64_t at = (int64_t)p.of((axes >> (2 * e)) & 3) * half + i0 + e;
            c[e] = table_value<TT>(cos + at);
            s[e] = table_value<TT>(sin + at);
        }
    }
}
__device__ __forceinline__ void turn(float a, float b, float c, float s, float& ya, float& yb) {
    ya = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    yb = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
}
// Unit u of a head's row: the two W-element chunks that hold pairs W u .. W u + W - 1.  lo, hi: chunk numbers
template <int W = 8>
__device__ __forceinline__ void unit_chunks(const RotaryAxes& r, int u, int& lo, int& hi) {
    const bool apart = u < r.rd / (2 * W) && !r.interleaved;
    lo = apart ? u : 2 * u;
    hi = apart ? u + r.rd / (2 * W) : 2 * u + 1;
}
template <typename T, int W = 8, typename C = typename ChunkOf<W>::type>
__device__ __forceinline__ void turn_chunks(const C a, const C b, const float (&c)[W], const float (&s)[W], bool interleaved, C& ya, C& yb) {
    const T *xa = reinterpret_cast<const T*>(&a), *xb = reinterpret_cast<const T*>(&b);
    uint32_t *oa = reinterpret_cast<uint32_t*>(&ya), *ob = reinterpret_cast<uint32_t*>(&yb);
    if (interleaved) {
#pragma unroll
        for (int e = 0; e < W / 2; ++e) {
            float p, q;
            turn(Elem<T>::to_float(xa[2 * e]), Elem<T>::to_float(xa[2 * e + 1]), c[e], s[e], p, q);
            oa[e] = Elem<T>::pack(p, q);
            turn(Elem<T>::to_float(xb[2 * e]), Elem<T>::to_float(xb[2 * e + 1]), c[W / 2 + e], s[W / 2 + e], p, q);
            ob[e] = Elem<T>::pack(p, q);
        }
    } else {
#pragma unroll
        for (int e = 0; e < W; e += 2) {
            float p0, q0, p1, q1;
            turn(Elem<T>::to_float(xa[e]), Elem<T>::to_float(xb[e]), c[e], s[e], p0, q0);
            turn(Elem<T>::to_float(xa[e + 1]), Elem<T>::to_float(xb[e + 1]), c[e + 1], s[e + 1], p1, q1);
            oa[e / 2] = Elem<T>::pack(p0, p1);
            ob[e / 2] = Elem<T>::pack(q0, q1);
        }
    }
}
// element e of a head's row, for other rotary dims and tables that are not aligned
template <typename T, typename TT>
__device__ __forceinline__ T turn_elem(const T* x, int e, const RotaryAxes& r, const RotaryRows& p, float sign) {
    if (e >= r.rd) return x[e];
    const int half = r.rd / 2;
    const int i = r.interleaved ? e >> 1 : e % half;
    const bool first = r.interleaved ? (e & 1) == 0 : e < half;
    const int partner = r.interleaved ? e ^ 1 : first ? e + half : e - half;
    const int64_t at = (int64_t)p.of((r.axis[i >> 4] >> ((i & 15) * 2)) & 3) * half + i;
    const float c = table_value<TT>(reinterpret_cast<const TT*>(r.cos) + at), s = sign * table_value<TT>(reinterpret_cast<const TT*>(r.sin) + at);
    float ya, yb;
    if (first) { turn(Elem<T>::to_float(x[e]), Elem<T>::to_float(x[partner]), c, s, ya, yb); return Elem<T>::from_float(ya); }
    turn(Elem<T>::to_float(x[partner]), Elem<T>::to_float(x[e]), c, s, ya, yb);
    return Elem<T>::from_float(yb);
}
#endif

}  // namespace fa
