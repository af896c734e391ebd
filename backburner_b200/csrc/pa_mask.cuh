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
    uint64_t page_mul;                       // ceil(2^40 / (page_keys / 64))
    int *status;
    // the page of a key: (key / 64) / (page_keys / 64) by a product, exact for keys below 2^30 and pages of up to 2^22 keys
    // (quotient g * m / 2^40 with m <= 2^40 / d + 1: too large by at most g / 2^40 < 2^-16 <= 1 / d, so never by a whole)
    __host__ __device__ __forceinline__ uint32_t page_index(uint32_t key) const { return (uint32_t) ((uint64_t) (key >> 6) * page_mul >> 40); }
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
PA_HD uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : ~(~0ull << n); }

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
    // drafted keys that exist; none does where q0 is 64 or more before key 0 or behind the keys, so that q0 fits 31 bits
    r.q0 = clampi(st.q0, -64, 1 << 30);
    r.bits = bits & low_bits(st.nk - r.q0) & ~low_bits(-r.q0);
    return r;
}
PA_HD Row row_of(const View &v, Set st, uint32_t s, uint32_t t) {
    if (!v.tree) return row_from(v, st, (int64_t) st.q0 + t, clampi((int64_t) st.q0 + t + 1, 0, st.nk), 0);
    const uint64_t b = v.tree[(uint64_t) s * v.n_tok + t] & low_bits(v.n_tok);
    if (!b) return Row{0, 0, 0, 0, 0};
    return row_from(v, st, (int64_t) st.q0 + bit_count(b) - 1, clampi(st.q0, 0, st.nk), b);
}
// bits [0, n) of 32
PA_HD uint32_t low32(int n) {
#ifdef __CUDA_ARCH__
    uint32_t m;
    asm("bmsk.clamp.b32 %0, 0, %1;" : "=r"(m) : "r"(n > 0 ? n : 0));
    return m;
#else
    return (uint32_t) low_bits(n < 32 ? n : 32);
#endif
}
// bit i: the row sees key k0 + i (in halves, which is short code: it stands in loops that have to stay in the instruction cache)
PA_HD uint64_t vis64(const Row &r, int k0) {
    uint32_t m[2];
    for (int h = 0; h < 2; h++) {
        const int k = k0 + 32 * h;
        m[h] = (low32(r.hi - k) & ~low32(r.lo - k)) | low32(r.sink - k);
    }
    const int d = r.q0 - k0;
    uint64_t drafts = 0;
    if (d > -64 && d < 64) drafts = d >= 0 ? r.bits << d : r.bits >> -d;
    return (((uint64_t) m[1] << 32) | m[0]) | drafts;
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

// page `index` of a set (a page id outside the pool is reported and replaced by page 0). An ordinary load, as all loads of a
// paged call's inputs: its kernels start while the stream's earlier ones run, so the inputs may be written in a kernel's
// lifetime, before its pdl_wait, and non-coherent loads (__ldg) are for data that nobody writes in it.
__device__ __forceinline__ uint32_t page_of(const View &v, uint32_t s, uint32_t index) {
    const int32_t p = v.table[(uint64_t) s * v.max_pages + index];
    if ((uint32_t) p < v.n_pages) return (uint32_t) p;
    atomicCAS(v.status, ST_OK, ST_BAD_ARGS);
    return 0;
}
// row of the pool (within a layer) that holds key `key`
__device__ __forceinline__ uint32_t row_at(const View &v, uint32_t s, uint32_t key) {
    const uint32_t i = v.page_index(key);
    return page_of(v, s, i) * v.page_keys + (key - i * v.page_keys);
}

// ---------------------------------------------------------------- parts
// The work of a launch is its units, a set's row tiles (tile_rows rows of a head each; the split-K kernel's unit is the whole
// set), each over the groups of keys its own tokens see. The CTAs along the keys ("parts") are dealt out over the units in
// proportion to their cost, on the device, since the lengths are only known there: the least `per` for which all units fit
// n_parts, by bisection. A part takes at least sqrt(groups of a unit) / 4 groups: with fewer, the merge of more parts costs
// what the shorter parts gain (split-K kernel, us a call: 777 keys, window 512: 1 group a part 14.4, 4 groups 18.5; 4,096
// keys: 1 group 24.0, 4 groups 18.5). Part c of the launch is also the slot its partial goes to, rows of one unit;
// crange [units + 1] (what the merge reads) gets the parts of every unit.
struct Paged {
    View v;
    const uint8_t *k, *vr;     // the layer's rows
    uint32_t row0;             // the layer's first row in the cache's tensor maps
    uint32_t n_parts;
    uint32_t rows, tile_rows;  // query rows per head, and of a unit
    uint32_t half_rows;        // a unit with at most so many rows leaves one of the kernel's two row tiles out
    uint32_t n_rt;             // row tiles of a set
    uint32_t *crange;
};
// a unit's part: what a CTA works on
struct Part {
    uint32_t set, rt;          // the unit
    uint32_t index, of;        // part `index` of the unit's `of` (0: none for this CTA)
    uint32_t t0, t1;           // tokens of the unit's rows
    Set st;
    // the part's groups of the unit's n (n >= of: at least one): the first n % of parts take one more
    PA_HD void share(uint32_t n, uint32_t &first, uint32_t &count) const {
        const uint32_t per = n / of, more = n - per * of;
        first = index * per + (index < more ? index : more);
        count = per + (index < more);
    }
};
// the tokens of row tile rt (row r: token r % n_tok): all of them when its rows pass the last token
PA_HD void tokens_of(const Paged &p, uint32_t rt, uint32_t &t0, uint32_t &t1) {
    const uint32_t T = p.v.n_tok, r0 = rt * p.tile_rows, n = p.rows - r0 < p.tile_rows ? p.rows - r0 : p.tile_rows;
    const uint32_t a = r0 ? r0 % T : 0;
    t0 = a + n > T ? 0u : a;
    t1 = a + n > T ? T - 1 : a + n - 1;
}
// unit u, and the cost of its groups of G keys (a group of a unit with one row tile costs 7/8 of one with two)
template <int G>
__device__ __forceinline__ uint32_t unit_of(const Paged &p, uint32_t u, Part &r) {
    r.set = p.n_rt == 1 ? u : u / p.n_rt;
    r.rt = u - r.set * p.n_rt;
    tokens_of(p, r.rt, r.t0, r.t1);
    r.st = set_of(p.v, r.set);
    return (uint32_t) span_of<G>(p.v, r.st, r.t0, r.t1).n * (p.rows - r.rt * p.tile_rows <= p.half_rows ? 7u : 8u);
}
// the bounds of a part's cost: the least that a part may take, and one with which all units fit n_parts
__device__ __forceinline__ void part_bounds(const Paged &p, uint32_t units, uint64_t total, uint32_t &lo, uint32_t &hi) {
    const uint32_t least = max(1u, (uint32_t) sqrtf((float) total / (float) (8ull * units)) / 4) * 8;
    lo = hi = max(least, (uint32_t) ((total + p.n_parts - 1) / p.n_parts));
    // sum of ceil(cost / per) < total / per + units <= n_parts at hi (n_parts > units, by the plan); 2^30 is past any
    // unit's cost
    if (units > 1) hi = max(lo, (uint32_t) min((uint64_t) 1 << 30, (total + (p.n_parts - units) - 1) / (p.n_parts - units)));
}
constexpr uint32_t UNITS_IN_WARP = 32;   // up to so many units every CTA deals them out itself, one to a lane
// Part c. Warp-collective; every lane gets the result. With more units a kernel of its own has dealt them out (deal_kernel;
// every CTA going over all of them took 6 times as long at 1,024 sets of 8 tokens) and the CTA looks its part up in crange.
template <int G>
__device__ __forceinline__ Part find_part(const Paged &p, uint32_t c, bool write, uint32_t lane) {
    const uint32_t units = p.v.n_sets * p.n_rt;
    Part mine{};
    if (units > UNITS_IN_WARP) {
        const volatile uint32_t *ends = p.crange;
        if (c >= ends[units]) return mine;
        uint32_t lo = 0, hi = units;   // ends[lo] <= c < ends[hi]
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;
            const uint32_t below = __ballot_sync(0xffffffffu, at < hi && ends[at] <= c);   // rising: a run of lanes from lane 0
            lo += (uint32_t) (__popc(below) - 1) * step;
            hi = min(hi, lo + step);
        }
        unit_of<G>(p, lo, mine);
        mine.index = c - ends[lo];
        mine.of = ends[lo + 1] - ends[lo];
        return mine;
    }
    const uint32_t cost = lane < units ? unit_of<G>(p, lane, mine) : 0;   // a lane's unit
    uint64_t total = cost;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    uint32_t lo, hi;
    part_bounds(p, units, total, lo, hi);
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2, need = __reduce_add_sync(0xffffffffu, (cost + mid - 1) / mid);
        if (need <= p.n_parts) hi = mid;
        else lo = mid + 1;
    }
    const uint32_t cnt = (cost + hi - 1) / hi;
    uint32_t end = cnt;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, end, x);
        if (lane >= (uint32_t) x) end += y;
    }
    if (write) {
        if (lane == 0) p.crange[0] = 0;
        if (lane < units) p.crange[lane + 1] = end;
    }
    Part r{};
    const uint32_t hit = __ballot_sync(0xffffffffu, c < end && c >= end - cnt);
    if (hit) {
        const int src = __ffs((int) hit) - 1;
        r.set = __shfl_sync(0xffffffffu, mine.set, src);
        r.rt = __shfl_sync(0xffffffffu, mine.rt, src);
        r.t0 = __shfl_sync(0xffffffffu, mine.t0, src);
        r.t1 = __shfl_sync(0xffffffffu, mine.t1, src);
        r.of = __shfl_sync(0xffffffffu, cnt, src);
        r.index = c - (__shfl_sync(0xffffffffu, end, src) - r.of);
        r.st.nk = __shfl_sync(0xffffffffu, mine.st.nk, src);
        r.st.q0 = __shfl_sync(0xffffffffu, mine.st.q0, src);
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
