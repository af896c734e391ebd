// pa_cache.cuh - a paged device cache of quantised (or f16) key/value rows: which keys a query token sees (sliding
// window with sinks, or a tree of drafted tokens), the append of new rows (head norm, rotation, quantisation), reading
// rows back, copying pages and compacting accepted rows.
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

// ---------------------------------------------------------------- elements of a head
// value i of a head row: f16(d * q), or the f16 itself
template <int QUANT>
__device__ __forceinline__ float head_value(const uint8_t *head, int i) {
    if (QUANT == 0) return __half2float(reinterpret_cast<const __half *>(head)[i]);
    const uint8_t *blk = head + (i / 32) * dec::q_group_bytes(QUANT);
    const __half d = *reinterpret_cast<const __half *>(blk);
    int q;
    if (QUANT == 1) q = (int8_t) blk[2 + i % 32];
    else q = (int) ((blk[2 + i % 16] >> (i % 32 < 16 ? 0 : 4)) & 15) - 8;
    return __half2float(__hmul(d, __int2half_rn(q)));
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
    int inter, w32, vec;                                // vec: E-element loads are aligned
};
enum { DT_F16 = 0, DT_BF16 = 1, DT_F32 = 2 };
template <int DT>
__device__ __forceinline__ float load1(const void *p, int64_t i) {
    if (DT == DT_F32) return reinterpret_cast<const float *>(p)[i];
    const uint32_t x = reinterpret_cast<const uint16_t *>(p)[i];
    return DT == DT_F16 ? h2f_bits(x) : __uint_as_float(x << 16);
}
// E consecutive elements from element i
template <int DT, int E>
__device__ __forceinline__ void load_e(const void *p, int64_t i, int vec, float (&x)[E]) {
    if (!vec) {
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = load1<DT>(p, i + e);
    } else if (DT == DT_F32) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + i + e);
            x[e] = f.x; x[e + 1] = f.y; x[e + 2] = f.z; x[e + 3] = f.w;
        }
    } else {
        uint32_t w[E / 2];
        const uint16_t *src = reinterpret_cast<const uint16_t *>(p) + i;
        if (E == 8) *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(src);
        else *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(src);
#pragma unroll
        for (int e = 0; e < E / 2; e++) {
            x[2 * e] = DT == DT_F16 ? h2f_bits(w[e] & 0xFFFFu) : __uint_as_float(w[e] << 16);
            x[2 * e + 1] = DT == DT_F16 ? h2f_bits(w[e] >> 16) : __uint_as_float(w[e] & 0xFFFF0000u);
        }
    }
}
// E consecutive values (lane's dims E * lane ..) of a head into its row: 32 / E lanes share a quant block
template <int QUANT, int E>
__device__ __forceinline__ void store_head(uint8_t *head, uint32_t lane, const float (&x)[E]) {
    if (QUANT == 0) {
#pragma unroll
        for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t *>(head + 2 * (E * lane + e)) = pack_h2(x[e], x[e + 1]);
        return;
    }
    constexpr int LB = 32 / E, TOP = QUANT == 1 ? 127 : 7;
    float am = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) am = fmaxf(am, fabsf(x[e]));
#pragma unroll
    for (int w = 1; w < LB; w <<= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, w));
    const __half dh = __float2half_rn(__fdiv_rn(am, (float) TOP));
    const float df = __half2float(dh), id = df != 0.f ? __frcp_rn(df) : 0.f;
    uint8_t *blk = head + (lane / LB) * dec::q_group_bytes(QUANT);
    const uint32_t in = lane % LB;
    int q[E];
#pragma unroll
    for (int e = 0; e < E; e++) q[e] = __float2int_rn(fmaxf(-(float) TOP, fminf((float) TOP, __fmul_rn(x[e], id))));
    if (in == 0) *reinterpret_cast<__half *>(blk) = dh;
    if (QUANT == 1) {   // blocks start at even bytes: 16-bit stores
#pragma unroll
        for (int e = 0; e < E; e += 2)
            *reinterpret_cast<uint16_t *>(blk + 2 + E * in + e) = (uint16_t) ((q[e] & 0xFF) | (q[e + 1] & 0xFF) << 8);
    } else {
        uint32_t n[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const uint32_t own = (uint32_t) (q[e] + 8);
            n[e] = own | __shfl_down_sync(0xffffffffu, own, LB / 2) << 4;   // element e + 16 is LB / 2 lanes on
        }
        if (in < LB / 2)
#pragma unroll
            for (int e = 0; e < E; e += 2) *reinterpret_cast<uint16_t *>(blk + 2 + E * in + e) = (uint16_t) (n[e] | n[e + 1] << 8);
    }
}
constexpr int APPEND_WARPS = 8;
// block = token x group of heads; a warp takes every 8th head of the group (queries, then keys, then values)
template <int HD, int DT, int QUANT>
__global__ void __launch_bounds__(32 * APPEND_WARPS) append_kernel(const AppendParams p, uint32_t heads_per_block) {
    constexpr int E = HD / 32;
    __shared__ float2 cs[HD / 2];
    __shared__ float line[APPEND_WARPS][HD];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t T = p.view.n_tok, s = blockIdx.x / T, t = blockIdx.x % T;
    const int start = p.start[s];
    const int pos = p.pos ? p.pos[blockIdx.x] : clampi((int64_t) start + t, -1, INT32_MAX);
    const uint32_t nq = p.nkv * p.gqa, h0 = blockIdx.y * heads_per_block, h1 = min(h0 + heads_per_block, nq + 2 * p.nkv);
    const uint32_t half = p.rot / 2;
    if (pos >= 0) {
        for (uint32_t i = threadIdx.x; i < half; i += 32 * APPEND_WARPS) {
            const double turn = (double) pos * p.freqs[i] * 0.15915494309189535;   // / (2 pi)
            float sn, c;
            sincospif(2.f * (float) (turn - rint(turn)), &sn, &c);
            cs[i] = make_float2(c, sn);
        }
    }
    __syncthreads();
    // the row of the new key
    const int64_t key = (int64_t) start + t;
    bool stored = pos >= 0;
    if (stored && (key < 0 || key >= capacity(p.view))) {
        atomicCAS(p.view.status, ST_OK, ST_BAD_ARGS);
        stored = false;
    }
    uint64_t at = 0;
    if (stored) {
        const int32_t pg = __ldg(p.view.table + (uint64_t) s * p.view.max_pages + (uint32_t) key / p.view.page_keys);
        if ((uint32_t) pg < p.view.n_pages) {
            at = ((uint64_t) pg * p.view.page_keys + (uint32_t) key % p.view.page_keys) * p.rs;
        } else {
            atomicCAS(p.view.status, ST_OK, ST_BAD_ARGS);
            stored = false;
        }
    }
    for (uint32_t h = h0 + warp; h < h1; h += APPEND_WARPS) {
        const bool isq = h < nq, isk = !isq && h < nq + p.nkv;
        if (!isq && !stored) continue;
        const uint32_t hh = isq ? h : isk ? h - nq : h - nq - p.nkv;
        const void *src = isq ? p.q : isk ? p.k : p.v;
        const int64_t off = (int64_t) s * (isq ? p.q_set : isk ? p.k_set : p.v_set) +
                            (int64_t) t * (isq ? p.q_tok : isk ? p.k_tok : p.v_tok) + (int64_t) hh * HD + E * lane;
        float x[E];
        if (isq && pos < 0) {
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = 0.f;
        } else {
            load_e<DT, E>(src, off, p.vec, x);
        }
        if ((isq || isk) && pos >= 0) {
            const void *w = isq ? p.wq : p.wk;
            if (w) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < E; e++) ss = fmaf(x[e], x[e], ss);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                const float inv = rsqrtf(ss * (1.f / HD) + p.eps);
#pragma unroll
                for (int e = 0; e < E; e++)
                    x[e] = x[e] * inv * (p.w32 ? load1<DT_F32>(w, E * lane + e) : load1<DT>(w, E * lane + e));
            }
            // each dim and its partner meet through the warp's line of shared memory
            __syncwarp();
#pragma unroll
            for (int e = 0; e < E; e++) line[warp][E * lane + e] = x[e];
            __syncwarp();
#pragma unroll
            for (int e = 0; e < E; e++) {
                const uint32_t d = E * lane + e;
                if (d < p.rot) {
                    const bool second = p.inter ? d & 1 : d >= half;
                    const float2 c = cs[p.inter ? d / 2 : second ? d - half : d];
                    const float y = line[warp][p.inter ? d ^ 1u : second ? d - half : d + half];
                    x[e] = second ? x[e] * c.x + y * c.y : x[e] * c.x - y * c.y;
                }
            }
        }
        if (isq) {
            const uint32_t kvh = hh / p.gqa, g = hh % p.gqa;
            uint16_t *dst = p.Qs + ((((uint64_t) s * p.nkv + kvh) * p.gqa + g) * T + t) * HD + E * lane;
#pragma unroll
            for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t *>(dst + e) = pack_h2(x[e] * p.scale, x[e + 1] * p.scale);
        } else {
            store_head<QUANT, E>((isk ? p.K : p.V) + at + hh * p.hb, lane, x);
        }
    }
}

// ---------------------------------------------------------------- reading rows back
// keys first[s] + t, t < n_tok, of every set as f16 values [n_sets][n_tok][nkv][hd]; one warp per head of a key, K and V
struct RowsParams {
    View v;
    const int32_t *first;
    const uint8_t *K, *V;
    uint16_t *Ko, *Vo;
    uint64_t rs, hb;
    uint32_t nkv;
};
template <int HD, int QUANT>
__global__ void __launch_bounds__(256) rows_kernel(const RowsParams p) {
    constexpr int E = HD / 32;
    const uint64_t w = (uint64_t) blockIdx.x * 8 + threadIdx.x / 32;
    const uint32_t lane = threadIdx.x % 32;
    const uint64_t n = (uint64_t) p.v.n_sets * p.v.n_tok * p.nkv;
    if (w >= 2 * n) return;
    const bool isv = w >= n;
    const uint64_t i = isv ? w - n : w;
    const uint32_t h = (uint32_t) (i % p.nkv);
    const uint64_t tok = i / p.nkv;
    const uint32_t s = (uint32_t) (tok / p.v.n_tok), t = (uint32_t) (tok % p.v.n_tok);
    const int64_t key = (int64_t) p.first[s] + t;
    float x[E];
    const int32_t pg = key >= 0 && key < capacity(p.v) ? __ldg(p.v.table + (uint64_t) s * p.v.max_pages + (uint32_t) key / p.v.page_keys) : -1;
    if ((uint32_t) pg < p.v.n_pages) {
        const uint8_t *head = (isv ? p.V : p.K) + ((uint64_t) pg * p.v.page_keys + (uint32_t) key % p.v.page_keys) * p.rs + h * p.hb;
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = head_value<QUANT>(head, E * lane + e);
    } else {
        atomicCAS(p.v.status, ST_OK, ST_BAD_ARGS);
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = 0.f;
    }
    uint16_t *dst = (isv ? p.Vo : p.Ko) + i * HD + E * lane;
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t *>(dst + e) = pack_h2(x[e], x[e + 1]);
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
