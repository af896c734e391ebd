// pa_mask.cuh - which keys of a paged cache a query token sees (sliding window with sinks, or a tree of drafted tokens),
// the groups of keys a call has to read, and how they are dealt out to the CTAs of the attention kernels.
#pragma once
#include "pa_common.cuh"

namespace pa {
namespace pg {

// ---------------------------------------------------------------- which keys a token sees
// Token t of set s has its own key at q0 + t (q0 = q_pos[s], or n_keys[s] - n_tok). Without a tree it sees keys j <= q0 + t,
// with a window w only j > q0 + t - w or j < sinks. With a tree it sees the keys before q0 (the window measured from
// q0 + depth, depth = its ancestors) and the drafted keys q0 + u whose bit u is set in its mask; a token with no bit set
// is padding and sees nothing.
struct View {
    const int32_t *table, *n_keys, *q_pos;   // [n_sets][max_pages], [n_sets], [n_sets] or null
    const uint64_t *tree;                    // [n_sets][n_tok] or null
    uint32_t n_sets, max_pages, n_pages, page_keys, n_tok, window, sinks;
    int *status;
};
struct Set {
    int nk, q0;   // keys held, clamped to the table's reach; key of token 0 (may be negative or past nk)
};
// the keys a row sees: [lo, hi), [0, sink) and q0 + u for each bit u
struct Row {
    int lo, hi, sink, q0;
    uint64_t bits;
};

#define PA_HD __host__ __device__ __forceinline__
PA_HD int capacity(const View &v) { return (int) (v.max_pages * v.page_keys); }   // <= 2^30
PA_HD int clampi(int64_t x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : (int) x; }
// the low n bits
PA_HD uint64_t low_bits(int64_t n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

__device__ __forceinline__ Set set_of(const View &v, uint32_t s) {
    const int n = v.n_keys[s];
    if (n < 0 || n > capacity(v)) atomicCAS(v.status, ST_OK, ST_BAD_ARGS);
    return Set{clampi(n, 0, capacity(v)), v.q_pos ? v.q_pos[s] : clampi((int64_t) n - (int) v.n_tok, INT32_MIN, INT32_MAX)};
}
PA_HD int bit_count(uint64_t b) {
#ifdef __CUDA_ARCH__
    return __popcll(b);
#else
    return __builtin_popcountll(b);
#endif
}
// the first `sinks` keys, of at most hi
PA_HD int sink_end(const View &v, int hi) { return !v.window ? 0 : v.sinks < (uint32_t) hi ? (int) v.sinks : hi; }
PA_HD Row row_from(const View &v, Set st, int64_t at, int hi, uint64_t bits) {
    Row r;
    r.hi = hi;
    r.lo = v.window ? clampi(at - (int64_t) v.window + 1, 0, hi) : 0;
    r.sink = sink_end(v, hi);
    r.q0 = st.q0;
    r.bits = bits & low_bits((int64_t) st.nk - st.q0) & ~low_bits(-(int64_t) st.q0);   // drafted keys that exist
    return r;
}
PA_HD Row row_of(const View &v, Set st, uint32_t s, uint32_t t) {
    if (!v.tree) return row_from(v, st, (int64_t) st.q0 + t, clampi((int64_t) st.q0 + t + 1, 0, st.nk), 0);
    const uint64_t b = v.tree[(uint64_t) s * v.n_tok + t] & low_bits(v.n_tok);
    if (!b) return Row{0, 0, 0, st.q0, 0};
    return row_from(v, st, (int64_t) st.q0 + bit_count(b) - 1, clampi(st.q0, 0, st.nk), b);
}
// bit i: the row sees key k0 + i
PA_HD uint64_t vis64(const Row &r, int k0) {
    uint64_t m = (low_bits((int64_t) r.hi - k0) & ~low_bits((int64_t) r.lo - k0)) | low_bits((int64_t) r.sink - k0);
    const int64_t d = (int64_t) r.q0 - k0;
    if (d >= 0) m |= d < 64 ? r.bits << d : 0;
    else m |= d > -64 ? r.bits >> -d : 0;
    return m;
}

// The groups of G keys that tokens [t0, t1] of a set see together: the sinks' groups 0 .. a-1, then groups b, b+1, ...
struct Span {
    int a, b, n;   // n groups in all
    PA_HD int group(int i) const { return i < a ? i : b + (i - a); }
};
template <int G>
PA_HD Span span_of(const View &v, Set st, uint32_t t0, uint32_t t1) {
    // a tree's tokens: depth 0 starts the window earliest, the drafted keys end at q0 + n_tok
    const int hi = clampi((int64_t) st.q0 + (v.tree ? (int64_t) v.n_tok : (int64_t) t1 + 1), 0, st.nk);
    const int lo = v.window ? clampi((int64_t) st.q0 + (v.tree ? 0 : t0) - (int64_t) v.window + 1, 0, hi) : 0;
    const int end = lo < hi ? (hi + G - 1) / G : 0;
    Span p;
    p.a = (sink_end(v, hi) + G - 1) / G;
    p.b = lo / G > p.a ? lo / G : p.a;
    p.n = p.a + (end > p.b ? end - p.b : 0);
    return p;
}

// the page of the 64-key group that holds key `key` (a page id outside the pool is reported and replaced by page 0)
__device__ __forceinline__ uint32_t page_of(const View &v, uint32_t s, uint32_t key) {
    const int32_t p = __ldg(v.table + (uint64_t) s * v.max_pages + key / v.page_keys);
    if ((uint32_t) p < v.n_pages) return (uint32_t) p;
    atomicCAS(v.status, ST_OK, ST_BAD_ARGS);
    return 0;
}
// row of the pool (within a layer) that holds key `key`
__device__ __forceinline__ uint32_t row_at(const View &v, uint32_t s, uint32_t key) {
    return page_of(v, s, key) * v.page_keys + key % v.page_keys;
}

// ---------------------------------------------------------------- parts
// The CTAs of a launch along the keys ("parts") are dealt out over the sets in proportion to the groups each has to read,
// on the device, since the lengths are only known there: `per` groups a part, so that all sets fit n_parts. (One group a
// part where the groups are few: 777 keys, window 512, us a call: 1 group 14.4, 4 groups 18.5, 8 groups 22.6.) Part c of the
// launch is also the slot its partial goes to; crange [n_sets + 1] (what the merge reads) gets the parts of every set.
struct Paged {
    View v;
    const uint8_t *k, *vr;     // the layer's rows
    uint32_t row0;             // the layer's first row in the cache's tensor maps
    uint32_t n_parts;
    uint32_t *crange;
};
// what a CTA works on (in shared memory)
struct Part {
    uint32_t set, index, of;   // part `index` of the set's `of` (0: none for this CTA)
    Set st;
};
// warp-collective; every lane gets the result
template <int G>
__device__ __forceinline__ Part find_part(const Paged &p, uint32_t c, bool write, uint32_t lane) {
    const View &v = p.v;
    Part r{0, 0, 0, {0, 0}};
    if (v.n_sets == 1) {
        const Set st = set_of(v, 0);
        const uint32_t n = (uint32_t) span_of<G>(v, st, 0, v.n_tok - 1).n;
        const uint32_t per = max(1u, (n + p.n_parts - 1) / p.n_parts), cnt = (n + per - 1) / per;
        if (write && lane < 2) p.crange[lane] = lane ? cnt : 0u;
        if (c < cnt) r = Part{0, c, cnt, st};
        return r;
    }
    uint64_t total = 0;
    for (uint32_t s = lane; s < v.n_sets; s += 32) total += (uint32_t) span_of<G>(v, set_of(v, s), 0, v.n_tok - 1).n;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    // sum of ceil(n_s / per) < total / per + n_sets <= n_parts (n_parts > n_sets, by the plan)
    const uint64_t room = p.n_parts - v.n_sets;
    const uint32_t per = max(1u, (uint32_t) ((total + room - 1) / room));
    uint32_t base = 0;
    if (write && lane == 0) p.crange[0] = 0;
    for (uint32_t s0 = 0; s0 < v.n_sets; s0 += 32) {
        const uint32_t s = s0 + lane;
        Set st{0, 0};
        uint32_t cnt = 0;
        if (s < v.n_sets) {
            st = set_of(v, s);
            cnt = ((uint32_t) span_of<G>(v, st, 0, v.n_tok - 1).n + per - 1) / per;
        }
        uint32_t end = cnt;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, end, x);
            if (lane >= (uint32_t) x) end += y;
        }
        end += base;
        if (write && s < v.n_sets) p.crange[s + 1] = end;
        const uint32_t hit = __ballot_sync(0xffffffffu, c < end && c >= end - cnt);
        if (hit) {
            const int src = __ffs((int) hit) - 1;
            r.set = s0 + (uint32_t) src;
            r.of = __shfl_sync(0xffffffffu, cnt, src);
            r.index = c - (__shfl_sync(0xffffffffu, end, src) - r.of);
            r.st.nk = __shfl_sync(0xffffffffu, st.nk, src);
            r.st.q0 = __shfl_sync(0xffffffffu, st.q0, src);
            if (!write) return r;
        }
        base = __shfl_sync(0xffffffffu, end, 31);
    }
    return r;
}

// The tokens [t0, t1] of a row tile together: a row that sees what any of them sees, and the range every one of them sees
// (padding tokens aside: their rows are emptied when they are written). Warp-collective.
struct Tile {
    Row any;
    int full_lo, full_hi, full_sink;
    // every token sees the whole group of G keys at k0
    __device__ __forceinline__ bool full(int k0, int G) const { return (k0 >= full_lo && k0 + G <= full_hi) || k0 + G <= full_sink; }
};
__device__ __forceinline__ Tile tile_of(const View &v, Set st, uint32_t s, uint32_t t0, uint32_t t1, uint32_t lane) {
    Tile r;
    if (!v.tree) {
        const Row a = row_of(v, st, s, t0);
        r.any = row_of(v, st, s, t1);
        r.full_lo = r.any.lo;
        r.full_hi = a.hi;
        r.any.lo = a.lo;
    } else {   // n_tok <= 64; the depths and the drafted keys of all tokens
        uint64_t bits = 0;
        int dmin = 64, dmax = -1;
        for (uint32_t t = lane; t < v.n_tok; t += 32) {
            const uint64_t b = v.tree[(uint64_t) s * v.n_tok + t] & low_bits(v.n_tok);
            if (!b) continue;
            bits |= b;
            dmin = min(dmin, bit_count(b) - 1);
            dmax = max(dmax, bit_count(b) - 1);
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
            bits |= __shfl_xor_sync(0xffffffffu, bits, x);
            dmin = min(dmin, __shfl_xor_sync(0xffffffffu, dmin, x));
            dmax = max(dmax, __shfl_xor_sync(0xffffffffu, dmax, x));
        }
        const int hi = dmax < 0 ? 0 : clampi(st.q0, 0, st.nk);
        r.any = row_from(v, st, (int64_t) st.q0 + dmin, hi, bits);
        r.full_hi = hi;
        r.full_lo = row_from(v, st, (int64_t) st.q0 + dmax, hi, 0).lo;
    }
    r.full_sink = sink_end(v, r.full_hi);
    return r;
}
// padding: a drafted token without a bit in its mask
__device__ __forceinline__ bool is_padding(const View &v, uint32_t s, uint32_t t) {
    return v.tree && !(v.tree[(uint64_t) s * v.n_tok + t] & low_bits(v.n_tok));
}

}  // namespace pg
}  // namespace pa
