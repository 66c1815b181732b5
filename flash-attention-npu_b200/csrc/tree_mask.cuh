// What the attention kernels need to know of a tree of drafted tokens (fa_tree_fwd_kvcache): written once a call by the
// preparing kernel (tree_attention.cu), read in the few key tiles that hold drafted tokens or a window's edge.
//
// The T drafted tokens of a sequence stand in the cache behind its L valid rows.  Token t sees the cached row j < L when
// j >= L + depth(t) - left, and the drafted row L + s when bit s of its row of `bits` is set: s is t itself or one of its
// ancestors, it could be stored, and it lies inside the window.
#pragma once
#include <stdint.h>

namespace fa {

constexpr int kTreeMaxTokens = 256;
constexpr int kTreeMaxWords = kTreeMaxTokens / 32;
// Capacity of a sequence: rows are counted in 32 bits, up to 256 tokens and the rest of a tile behind the last one
constexpr int kTreeMaxRows = 0x7fffffff - 1023;

struct TreeMask {
    const uint32_t* bits;        // (b, tokens, words): drafted tokens that a token sees
    const int32_t* depth;        // (b, tokens): number of ancestors, -1 = no token here (sees nothing)
    const uint32_t* keys;        // (b, words): drafted tokens whose rows stand in the cache
    int tokens, words;
    int left;                    // window to the left, -1 = none
};

// Entries of a CTA's share of a list of `total` key tiles
#ifdef __CUDACC__
__host__ __device__
#endif
inline int tree_share(int total, int ctas, int at_least) {
    const int even = total / ctas + (total % ctas != 0);
    return even > at_least ? even : at_least;
}

#ifdef __CUDACC__
// Length of the cached prefix: a stale or oversized entry is truncated to the capacity, as in the other cache calls.
__device__ __forceinline__ int tree_prefix(const int32_t* seqused, int b, int capacity) { return max(0, min(seqused[b], capacity)); }

// First cached row that token t of sequence b sees (the prefix ends at L): past every row where there is no token.
__device__ __forceinline__ int tree_first_key(const TreeMask& m, int depth, int L) {
    if (depth < 0) return 0x7fffffff;
    return m.left < 0 ? 0 : (int)max(0ll, (long long)L + depth - m.left);
}
__device__ __forceinline__ int tree_first_key(const TreeMask& m, int b, int t, int L) { return tree_first_key(m, m.depth[b * m.tokens + t], L); }
// ... that any token can see, and the first one that every token sees
__device__ __forceinline__ int tree_first_any(const TreeMask& m, int L) { return m.left < 0 ? 0 : (int)max(0ll, (long long)L - m.left); }
__device__ __forceinline__ int tree_first_all(const TreeMask& m, int L) { return m.left < 0 ? 0 : (int)max(0ll, (long long)L + m.tokens - 1 - m.left); }

__device__ __forceinline__ uint32_t tree_word(const uint32_t* words, int n, int w) { return w >= 0 && w < n ? words[w] : 0u; }
// 32 bits of a row of `words` from bit s on (s may be negative; bits outside are 0)
__device__ __forceinline__ uint32_t tree_bits32(const uint32_t* words, int n, int s) {
    const int w = s >> 5;
    return __funnelshift_r(tree_word(words, n, w), tree_word(words, n, w + 1), s & 31);
}
// bits [lo, hi) of a word, clipped to it
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
    lo = max(lo, 0);
    hi = min(hi, 32);
    return lo >= hi ? 0u : (0xffffffffu >> (32 - hi)) & (0xffffffffu << lo);
}
// Visible keys among cache rows base .. base + 31 of a token whose prefix keys are [first, L): one bit a key.
__device__ __forceinline__ uint32_t tree_visible32(const TreeMask& m, const uint32_t* row, int base, int first, int L) {
    uint32_t v = first >= L ? 0u : bit_range(first > base ? min(first - base, 32) : 0, L - base);
    if (base + 32 > L && base < L + m.tokens) v |= tree_bits32(row, m.words, base - L);
    return v;
}
// Key tiles of a sequence: `n` from tile `lo` on
__device__ __forceinline__ void tree_tiles(const TreeMask& m, int L, int sk, int& lo, int& n) {
    lo = tree_first_any(m, L) / 128;
    n = max(0, (sk + 127) / 128 - lo);
}
// Keys of one split: the rows that any token can see, shared out evenly in whole 128-key tiles, at least min_keys a split
// (the lengths are on the device, so every CTA works this out for its own sequence).  -> [t_lo, t_hi) in tiles
__device__ __forceinline__ void tree_split_tiles(int first, int sk, int nsplit, int split, int min_keys, int& t_lo, int& t_hi) {
    const int lo = first / 128, hi = (sk + 127) / 128;
    const int per = max(min_keys / 128, (max(hi - lo, 0) + nsplit - 1) / nsplit);
    t_lo = min(lo + split * per, hi);
    t_hi = min(t_lo + per, hi);
}
#endif

}  // namespace fa
