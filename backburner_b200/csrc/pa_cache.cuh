// pa_cache.cuh - a paged device cache of quantised (or f16) key/value rows: the dealing of many units and the merge of the
// attention's partials, the append of new rows (head norm, rotation, quantisation), reading rows back, copying pages and
// compacting accepted rows. (Which keys a query token sees: pa_mask.cuh; the attention kernels: pa_decode.cuh, pa_prefill.cuh,
// pa_prefill_pair.cuh.)
//
// The cache: rows of layer i, page p, position j at base + ((i * n_pages + p) * page_keys + j) * rs, K and V alike, each
// row nkv heads of hb bytes (the row formats of pa_decode.cuh). The keys of sequence s are numbered 0, 1, ...; key j lies in
// page table[s][j / page_keys] at position j % page_keys. page_keys is a multiple of 64, so an aligned group of 64 keys
// is in one page. Lengths, positions and masks are read on the device: a captured call follows them.
#pragma once
#include "pa_common.cuh"
#include "pa_decode.cuh"
#include "pa_mask.cuh"

namespace pa {
namespace pg {

// ---------------------------------------------------------------- many units dealt out
// The same dealing as a CTA's own in find_part, for more units than a warp has lanes: one block, a unit to a thread (and every
// 1,024th after it), whose costs stay in crange until the parts' ends replace them. The bisection stops within 1/32 of the
// least cost. Bound: latency (a round is two barriers and the loads of the thread's own costs).
constexpr uint32_t DEAL_THREADS = 1024;
template <int G>
__global__ void __launch_bounds__(DEAL_THREADS) deal_kernel(const Paged p) {
    constexpr uint32_t W = DEAL_THREADS / 32;
    __shared__ uint64_t sums[W];
    __shared__ uint32_t tops[W], needs[2][W], ends[W];
    const uint32_t units = p.v.n_sets * p.n_rt, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    pdl_trigger();
    pdl_wait();
    uint64_t total = 0;
    uint32_t top = 0;
    for (uint32_t u = tid; u < units; u += DEAL_THREADS) {
        Part r{};
        const uint32_t cost = unit_of<G>(p, u, r);
        p.crange[u + 1] = cost;
        total += cost;
        top = max(top, cost);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) {
        sums[warp] = total;
        tops[warp] = top;
    }
    __syncthreads();
    total = sums[lane];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    top = __reduce_max_sync(0xffffffffu, tops[lane]);
    uint32_t lo, hi;
    part_bounds(p, units, total, lo, hi);
    hi = max(lo, min(hi, top));   // (one part a unit fits too)
    for (uint32_t round = 0; hi - lo > lo / 32; round++) {   // the same in all threads
        const uint32_t mid = lo + (hi - lo) / 2;
        uint32_t need = 0;
        for (uint32_t u = tid; u < units; u += DEAL_THREADS) need += (p.crange[u + 1] + mid - 1) / mid;
        need = __reduce_add_sync(0xffffffffu, need);
        if (lane == 0) needs[round % 2][warp] = need;
        __syncthreads();
        need = __reduce_add_sync(0xffffffffu, needs[round % 2][lane]);
        if (need <= p.n_parts) hi = mid;
        else lo = mid + 1;
    }
    if (tid == 0) p.crange[0] = 0;
    uint32_t base = 0;
    for (uint32_t u0 = 0; u0 < units; u0 += DEAL_THREADS) {
        const uint32_t u = u0 + tid;
        uint32_t end = u < units ? (p.crange[u + 1] + hi - 1) / hi : 0;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, end, x);
            if (lane >= (uint32_t) x) end += y;
        }
        __syncthreads();   // the last round's ends are read
        if (lane == 31) ends[warp] = end;
        __syncthreads();
        const uint32_t all = ends[lane];
        end += base + __reduce_add_sync(0xffffffffu, lane < warp ? all : 0);
        base += __reduce_add_sync(0xffffffffu, all);
        if (u < units) p.crange[u + 1] = end;
    }
}

// ---------------------------------------------------------------- merge of the paged attention's partials
// The log-sum-exp merge of a unit's parts (pa_merge.cuh's, over this cache's slots), giving O, m, l or f16(O / l) and lse. A
// call's merge is a chain of dependent loads (the parts' range, their l and m, their O) behind the attention kernel, so the
// first MERGE_AHEAD parts' O are loaded beside their l and m rather than after them; SPLIT warps share a row's parts.
struct MergeParams {
    const float *Op, *Mp, *Lp;      // slot c: [nkv][unit_rows][HD], [nkv][unit_rows]
    const uint32_t *crange;         // [units + 1]
    uint32_t n_sets, nkv, rows, unit_rows, n_rt;
    float *O, *M, *L;               // [n_sets][nkv][rows]...
    uint16_t *Oh;                   // or these
    float *lse;
};
template <int HD> constexpr int MERGE_AHEAD = HD == 128 ? 4 : 2;
template <int HD, int SPLIT, bool REPLY>
__global__ void __launch_bounds__(256) cache_merge_kernel(const MergeParams p) {
    constexpr int V = HD / 32, RPB = 8 / SPLIT, AHEAD = MERGE_AHEAD<HD>;
    __shared__ float s_m[8], s_l[8];
    __shared__ __align__(16) float s_acc[SPLIT > 1 ? 8 * HD : 4];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, sw = warp % SPLIT;
    const uint64_t row = (uint64_t) blockIdx.x * RPB + warp / SPLIT, per_set = (uint64_t) p.nkv * p.rows;
    const bool active = row < p.n_sets * per_set;
    const uint32_t s = active ? (uint32_t) (row / per_set) : 0, R = active ? (uint32_t) (row % per_set) : 0;
    const uint32_t h = R / p.rows, r = R - h * p.rows, rt = p.n_rt == 1 ? 0 : r / p.unit_rows;
    const uint64_t rr = (uint64_t) h * p.unit_rows + (r - rt * p.unit_rows), stride = (uint64_t) p.nkv * p.unit_rows;
    pdl_trigger();
    pdl_wait();
    const uint32_t c0 = active ? p.crange[s * p.n_rt + rt] : 0, c1 = active ? p.crange[s * p.n_rt + rt + 1] : 0;
    // this warp's parts: c0 + sw + SPLIT * i
    const uint32_t mine = c0 + sw < c1 ? (c1 - c0 - sw + SPLIT - 1) / SPLIT : 0;
    auto part = [&](uint32_t i) -> uint64_t { return (uint64_t) (c0 + sw + SPLIT * i) * stride + rr; };
    auto load_o = [&](uint32_t i, float (&o)[V]) {
        const float4 *src = reinterpret_cast<const float4 *>(p.Op + part(i) * HD + lane * V);
#pragma unroll
        for (int q = 0; q < V / 4; q++) {
            const float4 x = src[q];
            o[4 * q] = x.x; o[4 * q + 1] = x.y; o[4 * q + 2] = x.z; o[4 * q + 3] = x.w;
        }
    };
    float ahead[AHEAD][V], l0 = 0.f, m0 = -INFINITY;
    if (lane < mine) {
        l0 = p.Lp[part(lane)];
        m0 = p.Mp[part(lane)];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
        if ((uint32_t) i < mine) load_o((uint32_t) i, ahead[i]);
    float M = l0 > 0.f ? m0 : -INFINITY;
    for (uint32_t i = lane + 32; i < mine; i += 32) {
        const float l = p.Lp[part(i)], m = p.Mp[part(i)];
        if (l > 0.f) M = fmaxf(M, m);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    if (SPLIT > 1) {
        if (lane == 0) s_m[warp] = M;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SPLIT; w++) M = fmaxf(M, s_m[warp / SPLIT * SPLIT + w]);
    }
    float acc[V], L = 0.f;
#pragma unroll
    for (int q = 0; q < V; q++) acc[q] = 0.f;
    for (uint32_t b = 0; b < mine; b += 32) {
        float l = l0, m = m0;
        if (b > 0) {
            l = b + lane < mine ? p.Lp[part(b + lane)] : 0.f;
            m = b + lane < mine ? p.Mp[part(b + lane)] : -INFINITY;
        }
        const float w = l > 0.f ? ex2((m - M) * LOG2E) : 0.f;   // a part without keys may hold anything in O: not used
        L = fmaf(w, l, L);
        const uint32_t n = min(32u, mine - b);
        if (b == 0) {
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const float wi = __shfl_sync(0xffffffffu, w, i);
                if (wi != 0.f)
#pragma unroll
                    for (int q = 0; q < V; q++) acc[q] = fmaf(wi, ahead[i][q], acc[q]);
            }
        }
#pragma unroll 4
        for (uint32_t i = b == 0 ? AHEAD : 0; i < n; i++) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            float o[V];
            load_o(b + i, o);
            if (wi != 0.f)
#pragma unroll
                for (int q = 0; q < V; q++) acc[q] = fmaf(wi, o[q], acc[q]);
        }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
    if (SPLIT > 1) {   // the warps' sums, against the same M, add up in the row's first warp
#pragma unroll
        for (int q = 0; q < V / 4; q++)
            reinterpret_cast<float4 *>(s_acc + warp * HD + lane * V)[q] = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
        if (lane == 0) s_l[warp] = L;
        __syncthreads();
        if (sw != 0) return;
#pragma unroll
        for (int w = 1; w < SPLIT; w++) {
#pragma unroll
            for (int q = 0; q < V / 4; q++) {
                const float4 x = reinterpret_cast<const float4 *>(s_acc + (warp + w) * HD + lane * V)[q];
                acc[4 * q] += x.x; acc[4 * q + 1] += x.y; acc[4 * q + 2] += x.z; acc[4 * q + 3] += x.w;
            }
            L += s_l[warp + w];
        }
    }
    if (!active) return;
    // L is 0 where the row sees nothing, and NaN (a part's l is) where its scores are not numbers: no value then
    if constexpr (REPLY) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int q = 0; q < V; q += 2)
            *reinterpret_cast<uint32_t *>(p.Oh + row * HD + lane * V + q) = pack_h2(acc[q] * inv, acc[q + 1] * inv);
        if (lane == 0) p.lse[row] = L == 0.f ? -INFINITY : M + logf(L);
    } else {
        if (!(L >= 0.f))
#pragma unroll
            for (int q = 0; q < V; q++) acc[q] = L;
#pragma unroll
        for (int q = 0; q < V / 4; q++)
            reinterpret_cast<float4 *>(p.O + row * HD + lane * V)[q] = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
        if (lane == 0) {
            p.M[row] = L > 0.f ? M : L == 0.f ? -INFINITY : L;
            p.L[row] = L;
        }
    }
}

// ---------------------------------------------------------------- append: head norm, rotation, scale, quantised store
// q, k: y = x * rsqrt(mean(x^2) + eps) * w (no weight: y = x); the first `rot` dims turned in pairs by angle pos * freq;
// queries leave as f16(y * scale) in the attention calls' layout [set][nkv][gqa * n_tok][hd] (row g * n_tok + t), keys and the
// values as they are go to the cache row of key start + t. All arithmetic in fp32 (the sum of squares too), rounded
// once; the angle in fp64 turns, of which only the fraction counts, so far positions lose nothing.
struct AppendParams {
    const void *q, *k, *v;
    int64_t q_set, q_tok, k_set, k_tok, v_set, v_tok;   // strides in elements; heads are hd apart
    const void *wq, *wk;                                // [hd] of the inputs' type (w32: fp32), or null
    const double *freqs;                                // [rot / 2], radians per position
    const int32_t *start, *pos;                         // [n_sets]; [n_sets][n_tok] or null (start + t); < 0: padding
    View view;                                          // table, sizes, status
    uint8_t *K, *V;                                     // the layer's rows
    uint16_t *Qs;
    uint64_t rs, hb;
    uint32_t nkv, gqa, rot;
    float eps, scale;
    int inter, w32;
};
enum { DT_F16 = 0, DT_BF16 = 1, DT_F32 = 2 };
// 8 consecutive elements as loaded: 8 fp32 or 4 words of 16-bit pairs
template <int DT>
__device__ __forceinline__ float load1(const void *p, uint32_t i) {
    if (DT == DT_F32) return reinterpret_cast<const float *>(p)[i];
    const uint32_t x = reinterpret_cast<const uint16_t *>(p)[i];
    return DT == DT_F16 ? h2f_bits(x) : __uint_as_float(x << 16);
}
template <int DT> constexpr int RAW8 = DT == DT_F32 ? 8 : 4;
template <int DT, bool VEC>
__device__ __forceinline__ void load_raw(const uint8_t *p, uint32_t (&w)[RAW8<DT>]) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < RAW8<DT>; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(p + 4 * i);
            w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < RAW8<DT>; i++)
            w[i] = DT == DT_F32 ? *reinterpret_cast<const uint32_t *>(p + 4 * i)
                                : *reinterpret_cast<const uint16_t *>(p + 4 * i) | (uint32_t) *reinterpret_cast<const uint16_t *>(p + 4 * i + 2) << 16;
    }
}
// ... as 4 fp32 pairs
template <int DT>
__device__ __forceinline__ void unpack8(const uint32_t (&w)[RAW8<DT>], uint64_t (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (DT == DT_F32) x[e] = pack_f2(__uint_as_float(w[(2 * e) % RAW8<DT>]), __uint_as_float(w[(2 * e + 1) % RAW8<DT>]));
        else if (DT == DT_F16) x[e] = pack_f2(h2f_bits(w[e] & 0xFFFFu), h2f_bits(w[e] >> 16));
        else x[e] = pack_f2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xFFFF0000u));
    }
}
// 8 consecutive values (dims 8 * l ..) of a head into its row; the 4 lanes of a quant block are neighbours
template <int QUANT>
__device__ __forceinline__ void store_head(uint8_t *head, uint32_t l, bool write, const float (&x)[8]) {
    if (QUANT == 0) {
        if (write)
            *reinterpret_cast<uint4 *>(head + 16 * l) = make_uint4(pack_h2(x[0], x[1]), pack_h2(x[2], x[3]), pack_h2(x[4], x[5]), pack_h2(x[6], x[7]));
        return;
    }
    constexpr float TOP = QUANT == 1 ? 127.f : 7.f;
    float am = 0.f;   // NaN if a value is: then d is, and with it every value of the block
#pragma unroll
    for (int e = 0; e < 8; e++) am = max_nan(am, fabsf(x[e]));
    am = max_nan(am, __shfl_xor_sync(0xffffffffu, am, 1));
    am = max_nan(am, __shfl_xor_sync(0xffffffffu, am, 2));
    const __half dh = __float2half_rn(__fdiv_rn(am, TOP));
    const float df = __half2float(dh), id = df != 0.f ? __frcp_rn(df) : 0.f;
    uint8_t *blk = head + (l / 4) * dec::q_group_bytes(QUANT);
    const uint32_t in = l % 4;
    // x / d (Markstein's correction: a quotient off by a unit or so in the last place, its exact remainder and the rounded
    // reciprocal; a quotient that fp32 holds, as every tie of rint, comes out exactly). d = 0 gives 0; so do d = inf and d = NaN,
    // the quotients without a value among them (the conversion turns NaN into 0), so that the block reads as NaN
    const float dd = id != 0.f ? df : 0.f;
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float y = __fmul_rn(x[e], id);
        y = fmaf(fmaf(-y, dd, x[e]), id, y);
        q[e] = (uint32_t) max(-(int) TOP, min((int) TOP, __float2int_rn(y)));
    }
    if (write && in == 0) *reinterpret_cast<__half *>(blk) = dh;
    uint16_t *dst = reinterpret_cast<uint16_t *>(blk + 2 + 8 * in);   // blocks start at even bytes: 16-bit stores
    if (QUANT == 1) {
        if (write)
#pragma unroll
            for (int e = 0; e < 8; e += 2) dst[e / 2] = (uint16_t) ((q[e] & 0xFFu) | q[e + 1] << 8);
    } else {   // byte i: element i, element i + 16 (two lanes on) << 4
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint32_t own = (q[e] + 8u) | (q[e + 1] + 8u) << 8;
            w[e / 2] = own | __shfl_down_sync(0xffffffffu, own, 2) << 4;
        }
        if (write && in < 2)
#pragma unroll
            for (int i = 0; i < 4; i++) dst[i] = (uint16_t) w[i];
    }
}
constexpr int APPEND_WARPS = 4;
// heads a block takes in one step of its warps: a lane has 8 dims, so a warp has 2 heads at hd 128 and 1 at hd 256
__host__ __device__ constexpr int append_heads(int hd) { return APPEND_WARPS * 256 / hd; }
// Block = token x STEPS * append_heads heads. The heads are numbered queries, then keys, then values, each kind rounded up to
// whole warps, so that a warp's step is of one kind. A warp loads all its heads before it works on the first, and the loads
// fly while the block computes the token's angles. Bound: for long prompts issue (2 x 8,191 tokens of 40 + 8 + 8 heads, bf16 to
// Q8_0: 5,040 warp instructions a token, half of them in the heads' steps of 60 for queries and 160 for keys, the rest the
// token's own angles, weights, row and addresses; issue slots 65 % busy; the loads alone run at 6 TB/s); for single tokens a
// chain of a few loads.
// How a head's pairs meet: halves, by a shuffle to the lane half / 8 away (HALVES: half a multiple of 8); within a lane
// (PAIRS: interleaved); through shared memory, for any rot, order and alignment (ANY). A template, since the compiler runs
// the paths not taken as predicated instructions.
enum { ROT_HALVES = 0, ROT_PAIRS = 1, ROT_ANY = 2 };
template <int HD, int DT, int QUANT, int STEPS, int ROT>
__global__ void __launch_bounds__(32 * APPEND_WARPS, 6) append_kernel(const AppendParams p) {
    constexpr int LPH = HD / 8;   // lanes of a head
    constexpr int SIZE = DT == DT_F32 ? 4 : 2;
    __shared__ __align__(16) float2 cs[HD / 2];
    __shared__ __align__(16) float line[ROT == ROT_ANY ? APPEND_WARPS : 1][256];
    __shared__ __align__(16) float wsm[2][HD];   // norm weights of queries and keys (1: no norm)
    __shared__ int64_t s_at;   // byte offset of the new key's row; -1: none is stored
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, l = lane % LPH;
    const uint32_t T = p.view.n_tok, s = blockIdx.y, t = blockIdx.x;
    constexpr uint32_t HPW = 32 / LPH, HPB = append_heads(HD);   // heads of a warp's step, of a block's step
    const uint32_t uwarp = __shfl_sync(0xffffffffu, warp, 0);    // (known to be the same in all lanes)
    const uint32_t nq = p.nkv * p.gqa, nqw = (nq + HPW - 1) / HPW * HPW, nkw = (p.nkv + HPW - 1) / HPW * HPW;
    const uint32_t hw0 = blockIdx.z * (HPB * STEPS) + uwarp * HPW, sub = lane / LPH;
    const uint32_t half = p.rot / 2;
    pdl_trigger();
    pdl_wait();
    const int start = p.start[s];
    const int pos = p.pos ? p.pos[(uint64_t) s * T + t] : clampi((int64_t) start + t, -1, INT32_MAX);
    if (pos < 0) {   // padding, or without positions a key before the first one: its query rows are zero
        if (!p.pos && blockIdx.z == 0 && threadIdx.x == 0) atomicCAS(p.view.status, ST_OK, ST_BAD_ARGS);
#pragma unroll 1
        for (uint32_t h = hw0 + sub; h < hw0 + HPB * STEPS && h < nq; h += HPB)
            *reinterpret_cast<uint4 *>(p.Qs + (((uint64_t) s * nq + h) * T + t) * HD + 8 * l) = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    const uint8_t *qb = (const uint8_t *) p.q + ((int64_t) s * p.q_set + (int64_t) t * p.q_tok + 8 * l) * SIZE + sub * (HD * SIZE);
    const uint8_t *kb = (const uint8_t *) p.k + ((int64_t) s * p.k_set + (int64_t) t * p.k_tok + 8 * l) * SIZE + sub * (HD * SIZE);
    const uint8_t *vb = (const uint8_t *) p.v + ((int64_t) s * p.v_set + (int64_t) t * p.v_tok + 8 * l) * SIZE + sub * (HD * SIZE);
    uint32_t raw[STEPS][RAW8<DT>];
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const uint32_t hw = hw0 + HPB * i;
#pragma unroll
        for (int e = 0; e < RAW8<DT>; e++) raw[i][e] = 0;
        if (hw < nqw) {
            if (hw + sub < nq) load_raw<DT, ROT != ROT_ANY>(qb + hw * (HD * SIZE), raw[i]);
        } else if (hw < nqw + nkw) {
            if (hw - nqw + sub < p.nkv) load_raw<DT, ROT != ROT_ANY>(kb + (hw - nqw) * (HD * SIZE), raw[i]);
        } else if (hw < nqw + 2 * nkw) {
            if (hw - nqw - nkw + sub < p.nkv) load_raw<DT, ROT != ROT_ANY>(vb + (hw - nqw - nkw) * (HD * SIZE), raw[i]);
        }
    }
    for (uint32_t i = threadIdx.x; i < 2 * HD; i += 32 * APPEND_WARPS) {
        const void *w = i < HD ? p.wq : p.wk;
        wsm[i / HD][i % HD] = !w ? 1.f : p.w32 ? load1<DT_F32>(w, i % HD) : load1<DT>(w, i % HD);
    }
    if (threadIdx.x == 32 * APPEND_WARPS - 1) {   // the row of the new key
        const int64_t key = (int64_t) start + t;
        int64_t at = -1;
        const int32_t pg = key >= 0 && key < capacity(p.view)
                               ? p.view.table[(uint64_t) s * p.view.max_pages + (uint32_t) key / p.view.page_keys] : -1;
        if ((uint32_t) pg < p.view.n_pages) at = ((int64_t) pg * p.view.page_keys + (uint32_t) key % p.view.page_keys) * (int64_t) p.rs;
        else atomicCAS(p.view.status, ST_OK, ST_BAD_ARGS);
        s_at = at;
    }
    for (uint32_t i = threadIdx.x; i < half; i += 32 * APPEND_WARPS) {
        const double turn = (double) pos * p.freqs[i] * 0.15915494309189535;   // / (2 pi)
        const double x = 2. * (turn - rint(turn));   // half turns
        const float hi = (float) x, lo = 3.14159265f * (float) (x - hi);   // the angle's rounding, up to 2^-25 half turns
        float sn, c;
        sincospif(hi, &sn, &c);
        cs[i] = make_float2(fmaf(-lo, sn, c), fmaf(lo, c, sn));
    }
    __syncthreads();
    const int64_t at = s_at;
    // a lane has the same dims of every head: their angles stay in registers, the sine with the partner's sign
    const bool turns = 8 * l < p.rot, second = 8 * l >= half;
    uint64_t cc[4], sn[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        cc[e] = pack_f2(1.f, 1.f);
        sn[e] = 0;
        if (ROT == ROT_PAIRS) {
            const float2 c = turns && 8 * l + 2 * e < p.rot ? cs[4 * l + e] : make_float2(1.f, 0.f);
            cc[e] = pack_f2(c.x, c.x);
            sn[e] = pack_f2(-c.y, c.y);
        } else if (ROT == ROT_HALVES && turns) {
            const float2 *c = cs + 8 * l - (second ? half : 0) + 2 * e;
            cc[e] = pack_f2(c[0].x, c[1].x);
            sn[e] = second ? pack_f2(c[0].y, c[1].y) : pack_f2(-c[0].y, -c[1].y);
        }
    }
    const int from = !turns ? (int) lane : second ? (int) lane - (int) (half / 8) : (int) (lane + half / 8);
    // norm and rotation of a warp's heads; the norm's factor and the scale are multiplied in at the end
    auto head = [&](uint64_t (&x)[4], const float *w8, bool norm, float f, float (&v)[8]) {
        if (norm) {
            uint64_t s2 = mul_f2(x[0], x[0]);
#pragma unroll
            for (int e = 1; e < 4; e++) s2 = fma_f2(x[e], x[e], s2);
            float ss, s1;
            unpack_f2(s2, ss, s1);
            ss += s1;
#pragma unroll
            for (int d = LPH / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
            // (the approximation's 2 units in the last place, after a Newton step less than one)
            const float a = fmaf(ss, 1.f / HD, p.eps), r = rsqrtf(a);
            f *= fmaf(0.5f * r, fmaf(-a * r, r, 1.f), r);
            const ulonglong2 w0 = reinterpret_cast<const ulonglong2 *>(w8)[0], w1 = reinterpret_cast<const ulonglong2 *>(w8)[1];
            x[0] = mul_f2(x[0], w0.x);
            x[1] = mul_f2(x[1], w0.y);
            x[2] = mul_f2(x[2], w1.x);
            x[3] = mul_f2(x[3], w1.y);
        }
        if constexpr (ROT == ROT_ANY) {
            float *ln = line[warp] + sub * HD;
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; e++) *reinterpret_cast<uint64_t *>(ln + 8 * l + 2 * e) = x[e];
            __syncwarp();
            if (turns) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t d = 8 * l + e;
                    const bool odd = p.inter ? e % 2 : d >= half;
                    const uint32_t a = p.inter ? d / 2 : odd ? d - half : d, b = p.inter ? d ^ 1u : odd ? d - half : d + half;
                    y[e] = ln[d];
                    if (d < p.rot) y[e] = y[e] * cs[a].x + (odd ? ln[b] : -ln[b]) * cs[a].y;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = pack_f2(y[2 * e], y[2 * e + 1]);
            }
        } else {
            uint64_t y[4];   // the partners
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (ROT == ROT_PAIRS) {
                    float a, b;
                    unpack_f2(x[e], a, b);
                    y[e] = pack_f2(b, a);
                } else {
                    y[e] = __shfl_sync(0xffffffffu, (unsigned long long) x[e], from);
                }
            }
            if (turns)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (ROT == ROT_HALVES || 8 * l + 2 * e < p.rot) x[e] = fma_f2(y[e], sn[e], mul_f2(x[e], cc[e]));
        }
        const uint64_t f2 = pack_f2(f, f);
#pragma unroll
        for (int e = 0; e < 4; e++) unpack_f2(mul_f2(x[e], f2), v[2 * e], v[2 * e + 1]);
    };
    // row g * n_tok + t of KV head h / gqa
    uint16_t *dst = p.Qs + (((uint64_t) s * nq + hw0 + sub) * T + t) * HD + 8 * l;
    const uint64_t dst_step = (uint64_t) HPB * T * HD;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const uint32_t hw = hw0 + HPB * i;
        uint64_t x[4];
        float v[8];
        unpack8<DT>(raw[i], x);
        if (hw < nqw) {
            head(x, wsm[0] + 8 * l, p.wq != nullptr, p.scale, v);
            if (hw + sub < nq)
                *reinterpret_cast<uint4 *>(dst) = make_uint4(pack_h2(v[0], v[1]), pack_h2(v[2], v[3]), pack_h2(v[4], v[5]), pack_h2(v[6], v[7]));
            dst += dst_step;
        } else if (hw < nqw + nkw) {
            if (at < 0) continue;
            head(x, wsm[1] + 8 * l, p.wk != nullptr, 1.f, v);
            const uint32_t h = hw - nqw + sub;
            store_head<QUANT>(p.K + at + h * p.hb, l, h < p.nkv, v);
        } else if (hw < nqw + 2 * nkw) {
            if (at < 0) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) unpack_f2(x[e], v[2 * e], v[2 * e + 1]);
            const uint32_t h = hw - nqw - nkw + sub;
            store_head<QUANT>(p.V + at + h * p.hb, l, h < p.nkv, v);
        }
    }
}

// ---------------------------------------------------------------- reading rows back
// keys first[s] + t, t < n_tok, of every set as f16 values [n_sets][n_tok][nkv][hd], K and V. A warp takes a key; a lane gives 8
// values at a time (a 16-byte store), ROWS_UNROLL of them in flight.
constexpr int ROWS_UNROLL = 4;
struct RowsParams {
    View v;
    const int32_t *first;
    const uint8_t *K, *V;
    uint16_t *Ko, *Vo;
    uint64_t rs, hb;
    uint32_t nkv, n;      // n: keys in all
};
template <int HD, int QUANT>
__global__ void __launch_bounds__(256) rows_kernel(const RowsParams p) {
    const uint32_t i = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
    pdl_trigger();
    pdl_wait();
    if (i >= p.n) return;
    const uint32_t s = i / p.v.n_tok, t = i % p.v.n_tok, pieces = p.nkv * (HD / 8);
    const int64_t key = (int64_t) p.first[s] + t;
    const int32_t pg = key >= 0 && key < capacity(p.v) ? p.v.table[(uint64_t) s * p.v.max_pages + (uint32_t) key / p.v.page_keys] : -1;
    const bool ok = (uint32_t) pg < p.v.n_pages;
    if (!ok && lane == 0) atomicCAS(p.v.status, ST_OK, ST_BAD_ARGS);
    const uint64_t at = ok ? ((uint64_t) pg * p.v.page_keys + (uint32_t) key % p.v.page_keys) * p.rs : 0;
    for (uint32_t c = lane; c < 2 * pieces; c += 32 * ROWS_UNROLL) {   // K's pieces, then V's
        uint32_t w[ROWS_UNROLL][4], d[ROWS_UNROLL];
#pragma unroll
        for (int u = 0; u < ROWS_UNROLL; u++) {
            const uint32_t x = c + 32 * u, y = x < pieces ? x : x - pieces;
            w[u][0] = w[u][1] = w[u][2] = w[u][3] = d[u] = 0;
            if (x >= 2 * pieces || !ok) continue;
            const uint32_t piece = y % (HD / 8);
            const uint8_t *head = (x < pieces ? p.K : p.V) + at + y / (HD / 8) * p.hb;
            if (QUANT == 0) {
                const uint4 r = *reinterpret_cast<const uint4 *>(head + 16 * piece);
                w[u][0] = r.x; w[u][1] = r.y; w[u][2] = r.z; w[u][3] = r.w;
            } else {   // blocks start at even bytes: 16-bit loads
                const uint8_t *blk = head + piece / 4 * dec::q_group_bytes(QUANT);
                const uint16_t *q = reinterpret_cast<const uint16_t *>(blk + 2 + (QUANT == 1 ? 8 * (piece % 4) : 8 * (piece % 2)));
                d[u] = *reinterpret_cast<const uint16_t *>(blk);
                w[u][0] = q[0] | (uint32_t) q[1] << 16;
                w[u][1] = q[2] | (uint32_t) q[3] << 16;
            }
        }
#pragma unroll
        for (int u = 0; u < ROWS_UNROLL; u++) {
            const uint32_t x = c + 32 * u, y = x < pieces ? x : x - pieces;
            if (x >= 2 * pieces) continue;
            uint32_t o[4];
            if (QUANT == 0) {
                o[0] = w[u][0]; o[1] = w[u][1]; o[2] = w[u][2]; o[3] = w[u][3];
            } else {
                const uint32_t s2 = d[u] | d[u] << 16;
                if (QUANT == 1) {
                    dec::q8_word(w[u][0], s2, o[0], o[1]);
                    dec::q8_word(w[u][1], s2, o[2], o[3]);
                } else {   // low nibbles: the first 16 elements of the block
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint32_t n = (w[u][j] >> (y % 4 < 2 ? 0 : 4)) & 0x0F0F0F0Fu;
                        o[2 * j] = hmul2(hsub2(prmt(n, 0x64646464u, 0x4140u), 0x64086408u), s2);
                        o[2 * j + 1] = hmul2(hsub2(prmt(n, 0x64646464u, 0x4342u), 0x64086408u), s2);
                    }
                }
            }
            *reinterpret_cast<uint4 *>((x < pieces ? p.Ko : p.Vo) + ((uint64_t) i * pieces + y) * 8) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// ---------------------------------------------------------------- row moves
// Pages src[i] -> dst[i] of every layer, K and V. No page is both read and written in one call (src[i] == dst[i] aside),
// so the order does not matter. A block copies 256 x 16 B x COPY_UNROLL of one page.
constexpr int COPY_UNROLL = 4;
struct CopyParams {
    uint8_t *K, *V;
    const int32_t *src, *dst;
    uint64_t page_bytes;      // page_keys * rs, a multiple of 1024
    uint32_t n_pages, n_layers;
    int *status;
};
__global__ void __launch_bounds__(256) copy_pages_kernel(const CopyParams p) {
    pdl_trigger();
    pdl_wait();
    const int32_t a = p.src[blockIdx.y], b = p.dst[blockIdx.y];
    if ((uint32_t) a >= p.n_pages || (uint32_t) b >= p.n_pages) {
        if (threadIdx.x == 0) atomicCAS(p.status, ST_OK, ST_BAD_ARGS);
        return;
    }
    uint8_t *base = (blockIdx.z & 1 ? p.V : p.K) + (uint64_t) (blockIdx.z / 2) * p.n_pages * p.page_bytes;
    const uint4 *s = reinterpret_cast<const uint4 *>(base + a * p.page_bytes);
    uint4 *d = reinterpret_cast<uint4 *>(base + b * p.page_bytes);
    const uint64_t n = p.page_bytes / 16, i0 = (uint64_t) blockIdx.x * 256 * COPY_UNROLL + threadIdx.x;
    uint4 x[COPY_UNROLL];
#pragma unroll
    for (int u = 0; u < COPY_UNROLL; u++)
        if (i0 + 256 * u < n) x[u] = s[i0 + 256 * u];
#pragma unroll
    for (int u = 0; u < COPY_UNROLL; u++)
        if (i0 + 256 * u < n) d[i0 + 256 * u] = x[u];
}

// Rows start + path[i] -> start + i, i < count, in place, every layer, K and V; path rises strictly, so path[i] >= i. A
// thread owns 16 bytes of the row and moves them down in order: a row that is overwritten has been read by then (row
// start + i is the source of a later move j > i only if path[j] = i < j, which cannot be), also when COMPACT_BATCH rows are
// loaded before they are stored.
constexpr int COMPACT_BATCH = 8;
constexpr uint32_t COMPACT_MAX = 1024;   // tokens of a path
struct CompactParams {
    View v;
    uint8_t *K, *V;
    const int32_t *start, *path, *count;   // [n_sets], [n_sets][n_tok], [n_sets]
    int32_t *n_keys_out;                   // [n_sets]: start + count (start where the set's arguments are refused)
    uint64_t rs;
    uint32_t n_layers;
};
__global__ void __launch_bounds__(128) compact_kernel(const CompactParams p) {
    __shared__ uint32_t from[COMPACT_MAX], to[COMPACT_MAX];
    const uint32_t s = blockIdx.y, T = p.v.n_tok;
    pdl_trigger();
    pdl_wait();
    const int start = p.start[s], count = p.count[s];
    bool bad = start < 0 || count < 0 || count > (int) T || (int64_t) start + (int64_t) T > capacity(p.v);
    if (!bad)
        for (uint32_t i = threadIdx.x; i < (uint32_t) count; i += blockDim.x) {
            const int32_t x = p.path[(uint64_t) s * T + i];
            if (x < 0 || x >= (int) T || (i > 0 && p.path[(uint64_t) s * T + i - 1] >= x)) {
                bad = true;
                continue;
            }
            const uint32_t a = (uint32_t) (start + x), b = (uint32_t) start + i;
            const int32_t pa = p.v.table[(uint64_t) s * p.v.max_pages + a / p.v.page_keys];
            const int32_t pb = p.v.table[(uint64_t) s * p.v.max_pages + b / p.v.page_keys];
            if ((uint32_t) pa >= p.v.n_pages || (uint32_t) pb >= p.v.n_pages) {
                bad = true;
                continue;
            }
            from[i] = (uint32_t) pa * p.v.page_keys + a % p.v.page_keys;
            to[i] = (uint32_t) pb * p.v.page_keys + b % p.v.page_keys;
        }
    bad = __syncthreads_or(bad);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (bad) atomicCAS(p.v.status, ST_OK, ST_BAD_ARGS);
        if (p.n_keys_out) p.n_keys_out[s] = start + (bad ? 0 : count);
    }
    if (bad) return;
    const uint32_t cols = (uint32_t) (p.rs / 16);
    const uint64_t i = (uint64_t) blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (uint64_t) cols * 2 * p.n_layers) return;
    const uint32_t col = (uint32_t) (i % cols), lk = (uint32_t) (i / cols);
    uint8_t *base = (lk & 1 ? p.V : p.K) + (uint64_t) (lk / 2) * p.v.n_pages * p.v.page_keys * p.rs + 16ull * col;
    for (int j0 = 0; j0 < count; j0 += COMPACT_BATCH) {
        uint4 x[COMPACT_BATCH];
#pragma unroll
        for (int u = 0; u < COMPACT_BATCH; u++)
            if (j0 + u < count && from[j0 + u] != to[j0 + u]) x[u] = *reinterpret_cast<const uint4 *>(base + (uint64_t) from[j0 + u] * p.rs);
#pragma unroll
        for (int u = 0; u < COMPACT_BATCH; u++)
            if (j0 + u < count && from[j0 + u] != to[j0 + u]) *reinterpret_cast<uint4 *>(base + (uint64_t) to[j0 + u] * p.rs) = x[u];
    }
}

}  // namespace pg
}  // namespace pa
