// pa_cache_host.h - the host side of the paged-cache entry points of include/pa_cuda.h: argument checks, plans and
// launches. Part of pa_cuda.cu, whose contexts and checks it uses.
#pragma once

namespace {

// the context's device for the length of a call; the caller's current device afterwards
struct DeviceScope {
    int before = -1;
    bool ok;
    explicit DeviceScope(int device) {
        ok = cudaGetDevice(&before) == cudaSuccess && (before == device || cudaSetDevice(device) == cudaSuccess);
        if (before == device) before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
};

// A launch that may start its prologue while the stream's previous kernel ends (every kernel launched so waits for it with
// pdl_wait before it reads or writes global memory)
template <class... A>
cudaError_t launch_pdl_cluster(uint32_t cluster, void (*kernel)(A...), dim3 grid, uint32_t threads, size_t smem, cudaStream_t st,
                               const A &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e != cudaSuccess ? e : cudaGetLastError();
}
template <class... A>
cudaError_t launch_pdl(void (*kernel)(A...), dim3 grid, uint32_t threads, size_t smem, cudaStream_t st, const A &...args) {
    return launch_pdl_cluster(1, kernel, grid, threads, smem, st, args...);
}

constexpr uint64_t kCacheMaxKeys = 1ull << 30;   // keys a page table reaches: key indexes and sums of them stay in 32 bits

int check_cache(pa_cuda_ctx *ctx, const pa_cuda_shape *sh, const pa_cuda_cache *c) {
    int rc = check_shape(ctx, sh);
    if (rc) return rc;
    if (!c || !c->k || !c->v) return fail(ctx, PA_CUDA_EINVAL, "cache is null");
    if (((uintptr_t) c->k | (uintptr_t) c->v) & 15) return fail(ctx, PA_CUDA_EINVAL, "cache K/V must be 16-byte aligned");
    if (c->page_keys == 0 || c->page_keys % 64 || c->page_keys > (1u << 22))
        return fail(ctx, PA_CUDA_EUNSUPPORTED, "page_keys must be a multiple of 64, at most 2^22");
    if (c->n_layers == 0 || c->n_pages == 0) return fail(ctx, PA_CUDA_EINVAL, "a cache needs a layer and a page");
    if (c->n_layers > 32767) return fail(ctx, PA_CUDA_EUNSUPPORTED, "more than 32,767 layers");
    // rows of the whole cache are numbered in 31 bits (tensor-map coordinates)
    if ((uint64_t) c->n_pages * c->page_keys > 0x7FFFFFFFull / c->n_layers)
        return fail(ctx, PA_CUDA_EUNSUPPORTED, "more than 2^31 - 1 rows in the cache");
    return PA_CUDA_OK;
}
int check_table(pa_cuda_ctx *ctx, const pa_cuda_cache *c, uint32_t n_sets, uint32_t max_pages) {
    if (max_pages == 0 || (uint64_t) max_pages * c->page_keys > kCacheMaxKeys)
        return fail(ctx, PA_CUDA_EINVAL, "max_pages must be >= 1 and reach at most 2^30 keys");
    if (n_sets > 65535) return fail(ctx, PA_CUDA_EUNSUPPORTED, "more than 65,535 sequences");
    return PA_CUDA_OK;
}
// whether every pointer is a multiple of n bytes (a misaligned one would fault on the device)
bool aligned(uintptr_t n, std::initializer_list<const void *> ptrs) {
    uintptr_t x = 0;
    for (const void *p : ptrs) x |= (uintptr_t) p;
    return x % n == 0;
}
// whether two device arrays of n and k int32 share a byte
bool overlap(const int32_t *a, uint64_t n, const int32_t *b, uint64_t k) {
    return a && b && (uintptr_t) a < (uintptr_t) b + 4 * k && (uintptr_t) b < (uintptr_t) a + 4 * n;
}
uint64_t page_mul(uint32_t page_keys) { return ((1ull << 40) + page_keys / 64 - 1) / (page_keys / 64); }
uint64_t layer_bytes(const pa_cuda_shape &sh, const pa_cuda_cache &c) { return (uint64_t) c.n_pages * c.page_keys * sh.rs; }

}  // namespace

struct pa_cuda_cache_plan {
    pa_cuda_ctx *ctx = nullptr;
    int device = 0;
    pa_cuda_shape sh{};
    pa_cuda_cache cache{};
    pa_cuda_mask mask{};
    uint32_t n_sets = 0, max_pages = 0;
    pa_cuda_plan d;                  // launch shape of the split-K kernel
    bool tc = false, pair = false;   // a tcgen05 kernel; on CTA pairs
    int nt = 1;                      // ... with nt tiles of 128 rows per CTA
    uint32_t n_rt = 1, unit_rows = 1;   // units of a set (row tiles; the split-K kernel: one) and their rows
    uint32_t n_parts = 1;            // CTAs along the keys = slots of partials (pa_mask.cuh)
    CUtensorMap *d_maps = nullptr;   // K and V rows of the whole cache
    float *d_part = nullptr;         // O [slot][nkv][unit_rows][hd], then m, then l
    uint32_t *d_crange = nullptr;    // [units + 1]: slots of each unit, written by every call
    const char *kernel = "";
};

namespace {

constexpr uint32_t kGroups64Overhead = 8;   // what a CTA of the tcgen05 kernel costs besides its groups, in groups

template <int HD, int Q, int W>
cudaError_t launch_decode_paged(const pa_cuda_cache_plan *p, const pa::dec::PagedParams &prm, cudaStream_t st) {
    return launch_pdl(pa::dec::decode_kernel<HD, Q, W, true>, dim3(p->n_parts, p->d.grid_y), 32 * p->d.n_consumers, p->d.smem, st, prm);
}
template <int Q, int NT, int D>
cudaError_t launch_prefill_paged(const pa_cuda_cache_plan *p, const CUtensorMap &tq, const pa::pre::PagedParams &prm, cudaStream_t st) {
    constexpr int smem = pa::pre::Smem<Q, NT, D>::TOTAL + 1024;
    return launch_pdl(pa::pre::prefill_kernel<Q, NT, D, true>, dim3(p->n_parts * p->sh.nkv), 32 * pa::pre::cta_warps(NT), smem,
                      st, tq, prm);
}
template <int Q, int NT, int D>
cudaError_t launch_pair_paged(const pa_cuda_cache_plan *p, const CUtensorMap &tq, const pa::pre::PagedParams &prm, cudaStream_t st) {
    constexpr int smem = pa::pre::PairSmem<Q, NT, D>::TOTAL + 1024;
    return launch_pdl_cluster(2, pa::pre::prefill_pair_kernel<Q, NT, D, true>, dim3(2 * p->n_parts * p->sh.nkv),
                              32 * (4 + 4 * NT + pa::pre::pair_dq_warps(D)), smem, st, tq, prm);
}
// f(kernel instance's constants) for the plan's kernel; f is a generic lambda
template <int HD, int W, class F>
auto with_quant(uint32_t quant, F &&f) {
    using std::integral_constant;
    if (quant == PA_CUDA_Q8_0) return f(integral_constant<int, HD>{}, integral_constant<int, 1>{}, integral_constant<int, W>{});
    if (quant == PA_CUDA_Q4_0) return f(integral_constant<int, HD>{}, integral_constant<int, 2>{}, integral_constant<int, W>{});
    return f(integral_constant<int, HD>{}, integral_constant<int, 0>{}, integral_constant<int, W>{});
}
template <class F>
auto with_decode(const pa_cuda_cache_plan *p, F &&f) {
    if (p->sh.hd == 128) return with_quant<128, 8>(p->sh.quant, f);
    return p->d.w == 4 ? with_quant<256, 4>(p->sh.quant, f) : with_quant<256, 8>(p->sh.quant, f);
}
template <class F>
auto with_prefill(const pa_cuda_cache_plan *p, F &&f) {
    using std::integral_constant;
    using I1 = integral_constant<int, 1>;
    using I2 = integral_constant<int, 2>;
    using D128 = integral_constant<int, 128>;
    using D256 = integral_constant<int, 256>;
    if (p->sh.hd == 256) return p->sh.quant == PA_CUDA_Q8_0 ? f(I1{}, I1{}, D256{}) : f(I2{}, I1{}, D256{});
    if (p->nt == 2) return p->sh.quant == PA_CUDA_Q8_0 ? f(I1{}, I2{}, D128{}) : f(I2{}, I2{}, D128{});
    return p->sh.quant == PA_CUDA_Q8_0 ? f(I1{}, I1{}, D128{}) : f(I2{}, I1{}, D128{});
}

template <int HD, bool REPLY>
cudaError_t launch_cache_merge(const pa_cuda_cache_plan *p, const pa::pg::MergeParams &mp, cudaStream_t st) {
    const uint64_t rows = (uint64_t) mp.n_sets * mp.nkv * mp.rows;
    // 8 warps a row where the rows alone leave SMs idle and a unit can have many parts (as launch_merge)
    if (rows * 8 <= (uint64_t) p->ctx->n_sm * 128 && p->n_parts >= 8 * p->n_sets * p->n_rt)
        return launch_pdl(pa::pg::cache_merge_kernel<HD, 8, REPLY>, dim3((unsigned) rows), 256, 0, st, mp);
    return launch_pdl(pa::pg::cache_merge_kernel<HD, 1, REPLY>, dim3((unsigned) ((rows + 7) / 8)), 256, 0, st, mp);
}

// O, m, l or Oh, lse: one of the two forms
int cache_attn(pa_cuda_cache_plan *p, uint32_t layer, const uint16_t *Qs, const int32_t *table, const int32_t *n_keys,
               const int32_t *q_pos, const uint64_t *tree, float *O, float *m, float *l, uint16_t *Oh, float *lse, void *stream) {
    if (!p) return PA_CUDA_EINVAL;
    pa_cuda_ctx *ctx = p->ctx;
    if (layer >= p->cache.n_layers) return fail(ctx, PA_CUDA_EINVAL, "layer out of range");
    if (!Qs || !table || !n_keys) return fail(ctx, PA_CUDA_EINVAL, "null argument");
    if ((p->mask.tree != 0) != (tree != nullptr)) return fail(ctx, PA_CUDA_EINVAL, "a tree plan takes the tree's masks, another plan none");
    if (!aligned(16, {Qs, O, Oh}) || !aligned(8, {tree}) || !aligned(4, {table, n_keys, q_pos, m, l, lse}))
        return fail(ctx, PA_CUDA_EINVAL, "misaligned pointer (Q and O to 16 bytes, the others to their elements)");
    DeviceScope dev(ctx->device);
    if (!dev.ok) return fail(ctx, PA_CUDA_ECUDA, "cudaSetDevice");
    cudaStream_t st = pick(ctx, stream);
    const pa_cuda_shape &sh = p->sh;
    const uint64_t rows_all = (uint64_t) sh.nkv * sh.rows, slot_rows = (uint64_t) sh.nkv * p->unit_rows;
    float *Op = p->d_part, *Mp = Op + p->n_parts * slot_rows * sh.hd, *Lp = Mp + p->n_parts * slot_rows;
    pa::pg::Paged pg{};
    pg.v.table = table;
    pg.v.n_keys = n_keys;
    pg.v.q_pos = q_pos;
    pg.v.tree = tree;
    pg.v.n_sets = p->n_sets;
    pg.v.max_pages = p->max_pages;
    pg.v.n_pages = p->cache.n_pages;
    pg.v.page_keys = p->cache.page_keys;
    pg.v.page_mul = page_mul(p->cache.page_keys);
    pg.v.n_tok = p->mask.n_tok;
    pg.v.window = p->mask.window;
    pg.v.sinks = p->mask.sinks;
    pg.v.status = ctx->d_status + 1;
    pg.k = p->cache.k + layer * layer_bytes(sh, p->cache);
    pg.vr = p->cache.v + layer * layer_bytes(sh, p->cache);
    pg.row0 = layer * p->cache.n_pages * p->cache.page_keys;
    pg.n_parts = p->n_parts;
    pg.rows = sh.rows;
    pg.tile_rows = p->unit_rows;
    pg.half_rows = p->tc && !p->pair && p->nt == 2 ? (uint32_t) pa::pre::BM : 0u;
    pg.n_rt = p->n_rt;
    pg.crange = p->d_crange;
    cudaError_t e = cudaSuccess;
    if ((uint64_t) p->n_sets * p->n_rt > pa::pg::UNITS_IN_WARP) {
        e = p->tc ? launch_pdl(pa::pg::deal_kernel<64>, dim3(1), pa::pg::DEAL_THREADS, 0, st, pg)
                  : launch_pdl(pa::pg::deal_kernel<16>, dim3(1), pa::pg::DEAL_THREADS, 0, st, pg);
        if (e != cudaSuccess) return cuda_fail(ctx, e, "cache deal launch");
        ctx->launches++;
    }
    if (p->tc) {
        CUtensorMap tq;
        if (!map_q(&tq, Qs, p->n_sets * rows_all, sh.hd)) return fail(ctx, PA_CUDA_ECUDA, "cuTensorMapEncodeTiled (Q) failed");
        pa::pre::PagedParams prm{};
        prm.pg = pg;
        prm.Qs = Qs;
        prm.kv_maps = p->d_maps;
        prm.Op = Op;
        prm.Mp = Mp;
        prm.Lp = Lp;
        prm.status = ctx->d_status;
        prm.rs = sh.rs;
        prm.hb = sh.hb;
        prm.nkv = sh.nkv;
        prm.rows = sh.rows;
        prm.n_rt = 1;
        prm.timeout_ns = ctx->timeout_ns;
        prm.stall = ctx->stall_test;
        e = with_prefill(p, [&](auto q, auto nt, auto d) {
            return p->pair ? launch_pair_paged<q.value, nt.value, d.value>(p, tq, prm, st) : launch_prefill_paged<q.value, nt.value, d.value>(p, tq, prm, st);
        });
    } else {
        pa::dec::PagedParams prm{};
        prm.pg = pg;
        prm.Qs = Qs;
        prm.Op = Op;
        prm.Mp = Mp;
        prm.Lp = Lp;
        prm.status = ctx->d_status;
        prm.rs = sh.rs;
        prm.hb = sh.hb;
        prm.nkv = sh.nkv;
        prm.rows = sh.rows;
        prm.hg = p->d.hg;
        prm.rgc = p->d.rgc;
        prm.n_rg = p->d.n_rg;
        prm.row = p->d.row;
        prm.gs = p->d.gs;
        prm.n_jobs = p->n_parts;
        prm.n_consumers = p->d.n_consumers;
        prm.timeout_ns = ctx->timeout_ns;
        prm.stall = ctx->stall_test;
        e = with_decode(p, [&](auto hd, auto q, auto w) { return launch_decode_paged<hd.value, q.value, w.value>(p, prm, st); });
    }
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cache attention launch");
    pa::pg::MergeParams mp{};
    mp.Op = Op;
    mp.Mp = Mp;
    mp.Lp = Lp;
    mp.crange = p->d_crange;
    mp.n_sets = p->n_sets;
    mp.nkv = sh.nkv;
    mp.rows = sh.rows;
    mp.unit_rows = p->unit_rows;
    mp.n_rt = p->n_rt;
    mp.O = O;
    mp.M = m;
    mp.L = l;
    mp.Oh = Oh;
    mp.lse = lse;
    if (sh.hd == 128) e = Oh ? launch_cache_merge<128, true>(p, mp, st) : launch_cache_merge<128, false>(p, mp, st);
    else e = Oh ? launch_cache_merge<256, true>(p, mp, st) : launch_cache_merge<256, false>(p, mp, st);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cache merge launch");
    ctx->launches += 2;
    return PA_CUDA_OK;
}

// the launch shape of a plan: kernel, row tiles, parts
int shape_cache_plan(pa_cuda_cache_plan *p) {
    pa_cuda_ctx *ctx = p->ctx;
    const pa_cuda_shape &sh = p->sh;
    p->d.ctx = ctx;
    p->d.sh = sh;
    int rc = plan_decode_shape(ctx, &p->d);
    if (rc) return rc;
    const bool tc_ok = sh.quant != PA_CUDA_F16 && encode_fn() != nullptr;
    if (ctx->kernel_choice >= 2 && !tc_ok) return fail(ctx, PA_CUDA_EUNSUPPORTED, "tcgen05 kernels need quantised (Q8_0 / Q4_0) rows");
    p->tc = tc_ok && (ctx->kernel_choice >= 2 || (ctx->kernel_choice == 0 && sh.rows >= (sh.hd == 128 ? kPrefillMinRows128 : kPrefillMinRows256)));
    // groups of keys that one set can have to read
    const uint32_t G = p->tc ? 64 : 16;
    const uint64_t cap = (uint64_t) p->max_pages * p->cache.page_keys;
    uint64_t groups = cap / G;
    if (p->mask.window)
        groups = std::min(groups, ((uint64_t) p->mask.window + p->mask.n_tok + G - 1) / G + 1 + std::min<uint64_t>((p->mask.sinks + (uint64_t) G - 1) / G, groups));
    if (p->tc) {
        // CTA pairs (512 rows a unit at hd 128) run a row of a group in 7/8 of the single-CTA kernel's time, if their rows are
        // real and the keys long: us single vs pair, 8 KV heads, 65,536 Q8_0 keys: 305 rows 159 vs 147, 640 rows 225 vs 308, 2,560
        // rows 884 vs 849; 2,560 rows over a window of 1,024 keys 51 vs 56, of 4,096 102 vs 98 (Q4_0 91 vs 96). hd 256, where
        // the single-CTA kernel has one tile: 240 rows x 4,096 keys 26.7 vs 24.6, 768 x 16,384 76 vs 67. Between those lengths,
        // 64 / 128 / 256 / 512 groups: 305 rows 25.7 vs 25.0, 33.0 vs 33.3, 51 vs 50, 92 vs 84; 512 rows 26.4 vs 26.4, 35.5 vs 34.7,
        // 53 vs 51, 95 vs 90; 640 rows 30 vs 36, 43 vs 54, 69 vs 90, 130 vs 171; 2,560 rows 82 vs 86, 131 vs 134, 228 vs 228, 461 vs 461;
        // hd 256, 128 and 512 groups: 144 rows 27 vs 25, 56 vs 50, 384 rows 36 vs 38, 79 vs 86, 768 rows 47 vs 44, 134 vs 120. The
        // rule's choice is within 3 % of the better one at most of them, 9 % off at worst (hd 256, 384 rows)
        const uint64_t in_pairs = ((uint64_t) sh.rows + 511) / 512 * 512, left = sh.rows % 256;
        const uint64_t single = (uint64_t) sh.rows / 256 * 256 + (left == 0 ? 0 : left <= 128 ? 224 : 256);
        const bool better = sh.hd == 256 ? sh.rows > kSingle256MaxRows : sh.rows >= kPairMinRows && groups >= 128 && 7 * in_pairs <= 8 * single;
        p->pair = ctx->kernel_choice == 3 || (ctx->kernel_choice == 0 && better);
    }
    uint64_t parts, units;
    if (p->tc) {
        const uint32_t tile = (uint32_t) pa::pre::BM * (p->pair ? 2u : 1u), ctas = p->pair ? 2 : 1;
        p->nt = sh.hd == 128 && sh.rows > tile ? 2 : 1;
        p->unit_rows = tile * p->nt;
        p->n_rt = (sh.rows + p->unit_rows - 1) / p->unit_rows;
        units = (uint64_t) p->n_sets * p->n_rt;
        static const char *names[2][2] = {{"pa::pre::prefill_kernel<1 tile, paged>", "pa::pre::prefill_kernel<2 tiles, paged>"},
                                          {"pa::pre::prefill_pair_kernel<1 tile, paged>", "pa::pre::prefill_pair_kernel<2 tiles, paged>"}};
        p->kernel = names[p->pair][p->nt - 1];
        const uint64_t y = (uint64_t) sh.nkv * ctas;   // CTAs of a part
        // the count that minimises waves x (groups of a part + a CTA's overhead), all units as long as they can be; parts
        // that are left over by equal units' remainders are counted out
        const uint64_t spare = units > 1 ? units : 0;
        uint64_t best = ~0ull;
        parts = units;
        for (uint64_t c = std::max<uint64_t>(1, units); c <= spare + std::max<uint64_t>(1, 8ull * ctx->n_sm / y); c++) {
            const uint64_t per = (groups + c / units - 1) / (c / units);
            const uint64_t cost = ((c / units * units * y + ctx->n_sm - 1) / ctx->n_sm) * (per + kGroups64Overhead);
            if (cost < best) { best = cost; parts = c; }
        }
        // as many as the waves hold anyway (units differ in length)
        const uint64_t waves = (parts * y + ctx->n_sm - 1) / ctx->n_sm;
        parts = std::max(parts, waves * ctx->n_sm / y);
        if ((2 * units + parts) * y > 0x7FFFFFFFull) return fail(ctx, PA_CUDA_EUNSUPPORTED, "too many rows and sets in one call");
    } else {
        // f16 rows have this kernel for every row count: with many, a CTA's warps share fewer heads' keys between more
        // rows (us with as many heads as fit and so: 8 sets x 8,192 keys, 8 heads x 16 rows 95 vs 72, 32 rows 197 vs 129; hd 256,
        // 2 sets x 4,096 keys, 512 tokens x 4 heads x 6 2,378 vs 1,279)
        if (sh.quant == PA_CUDA_F16 && p->d.n_rg > 1 && (rc = plan_decode_shape(ctx, &p->d, std::max(1u, p->d.w / p->d.n_rg)))) return rc;
        if (p->d.grid_y > 65535) return fail(ctx, PA_CUDA_EUNSUPPORTED, "too many head/row groups");
        p->kernel = "pa::dec::decode_kernel<paged>";
        int per_sm = 1;
        const cudaError_t e = with_decode(p, [&](auto hd, auto q, auto w) {
            auto *k = pa::dec::decode_kernel<hd.value, q.value, w.value, true>;
            // the limit is the function's, shared by every plan of the instance: all that a block can have
            cudaFuncAttributes a{};
            cudaError_t r = cudaFuncGetAttributes(&a, k);
            if (r == cudaSuccess) r = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem - (int) a.sharedSizeBytes);
            if (r == cudaSuccess) r = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, 32 * (int) p->d.n_consumers, p->d.smem);
            return r;
        });
        if (e != cudaSuccess) return cuda_fail(ctx, e, "cache plan: split-K kernel attributes");
        // as many CTAs as run at once
        parts = std::max<uint64_t>(1, (uint64_t) ctx->n_sm * std::max(1, per_sm) / p->d.grid_y);
        units = p->n_sets;
        p->unit_rows = sh.rows;
        // (or, where there are about as many sets, that many four times, since few sets can be cut then and the longest one
        // would be what the call takes: us without and with, 1 token, 256 sets of 512 to 4,096 keys 449 vs 317, 1,024 of up to
        // 2,048 704 vs 684; 64 sets, which are cut anyway, 95 vs 106)
        if (2 * units > parts) parts *= 4;
    }
    parts = std::min(parts, units * std::max<uint64_t>(1, groups));
    p->n_parts = (uint32_t) (units > 1 ? std::max(parts, units + 1) : parts);   // find_part: one more than the units
    return PA_CUDA_OK;
}

template <int HD, int DT, int Q, int STEPS, int ROT>
cudaError_t launch_append_s(const pa::pg::AppendParams &a, cudaStream_t st) {
    constexpr uint32_t w = 256 / HD, per = pa::pg::append_heads(HD) * STEPS;   // heads of a warp's step, of a block
    const uint32_t heads = (a.nkv * a.gqa + w - 1) / w * w + 2 * ((a.nkv + w - 1) / w * w);
    const dim3 grid(a.view.n_tok, a.view.n_sets, (heads + per - 1) / per);
    return launch_pdl(pa::pg::append_kernel<HD, DT, Q, STEPS, ROT>, grid, 32 * pa::pg::APPEND_WARPS, 0, st, a);
}
template <int HD, int DT, int Q>
cudaError_t launch_append_h(const pa::pg::AppendParams &a, uint32_t steps, int rot, cudaStream_t st) {
    using namespace pa::pg;
    if (rot == ROT_ANY) return launch_append_s<HD, DT, Q, 1, ROT_ANY>(a, st);
    if (steps == 1) return rot == ROT_PAIRS ? launch_append_s<HD, DT, Q, 1, ROT_PAIRS>(a, st) : launch_append_s<HD, DT, Q, 1, ROT_HALVES>(a, st);
    constexpr int S = DT == DT_F32 ? 4 : 8;   // (8 heads of fp32 do not fit the registers)
    return rot == ROT_PAIRS ? launch_append_s<HD, DT, Q, S, ROT_PAIRS>(a, st) : launch_append_s<HD, DT, Q, S, ROT_HALVES>(a, st);
}
template <int HD, int DT>
cudaError_t launch_append_q(const pa::pg::AppendParams &a, uint32_t quant, uint32_t steps, int rot, cudaStream_t st) {
    return quant == PA_CUDA_Q8_0   ? launch_append_h<HD, DT, 1>(a, steps, rot, st)
           : quant == PA_CUDA_Q4_0 ? launch_append_h<HD, DT, 2>(a, steps, rot, st)
                                   : launch_append_h<HD, DT, 0>(a, steps, rot, st);
}
template <int HD>
cudaError_t launch_append(const pa::pg::AppendParams &a, uint32_t dtype, uint32_t quant, uint32_t steps, int rot, cudaStream_t st) {
    return dtype == PA_CUDA_T_F16    ? launch_append_q<HD, pa::pg::DT_F16>(a, quant, steps, rot, st)
           : dtype == PA_CUDA_T_BF16 ? launch_append_q<HD, pa::pg::DT_BF16>(a, quant, steps, rot, st)
                                     : launch_append_q<HD, pa::pg::DT_F32>(a, quant, steps, rot, st);
}
template <int HD>
cudaError_t launch_rows(const pa::pg::RowsParams &a, uint32_t quant, cudaStream_t st) {
    const dim3 grid((a.n + 7) / 8);
    return launch_pdl(quant == PA_CUDA_Q8_0 ? pa::pg::rows_kernel<HD, 1> : quant == PA_CUDA_Q4_0 ? pa::pg::rows_kernel<HD, 2> : pa::pg::rows_kernel<HD, 0>,
                      grid, 256, 0, st, a);
}

}  // namespace

extern "C" {

int pa_cuda_cache_plan_create(pa_cuda_ctx *ctx, const pa_cuda_shape *shape, const pa_cuda_cache *cache, uint32_t n_sets,
                              uint32_t max_pages, const pa_cuda_mask *mask, pa_cuda_cache_plan **out) {
    if (!ctx || !out) return PA_CUDA_EINVAL;
    *out = nullptr;
    int rc = check_cache(ctx, shape, cache);
    if (rc || (rc = check_table(ctx, cache, n_sets, max_pages))) return rc;
    if (n_sets == 0) return fail(ctx, PA_CUDA_EINVAL, "n_sets must be >= 1");
    if (!mask || mask->n_tok == 0 || shape->rows % mask->n_tok) return fail(ctx, PA_CUDA_EINVAL, "rows must be a multiple of n_tok >= 1");
    if (mask->window > kCacheMaxKeys) return fail(ctx, PA_CUDA_EINVAL, "window above 2^30 keys (0: none)");
    if (mask->sinks && !mask->window) return fail(ctx, PA_CUDA_EINVAL, "sinks without a window");
    if (mask->tree && mask->n_tok > 64) return fail(ctx, PA_CUDA_EUNSUPPORTED, "a tree has at most 64 tokens");
    if (mask->tree && mask->window && mask->window < mask->n_tok)
        return fail(ctx, PA_CUDA_EUNSUPPORTED, "a tree needs a window of at least n_tok keys");
    if (ctx->qk_domain == PA_CUDA_QK_INT8)
        return fail(ctx, PA_CUDA_EUNSUPPORTED, "the int8-domain QK does not cover the paged cache");
    if ((uint64_t) n_sets * shape->nkv * shape->rows > 0x7FFFFFFFull)
        return fail(ctx, PA_CUDA_EUNSUPPORTED, "more than 2^31 - 1 query rows in a call");
    auto *p = new (std::nothrow) pa_cuda_cache_plan();
    if (!p) return fail(ctx, PA_CUDA_ENOMEM, "plan");
    p->ctx = ctx;
    p->device = ctx->device;
    p->sh = *shape;
    p->cache = *cache;
    p->mask = *mask;
    p->n_sets = n_sets;
    p->max_pages = max_pages;
    DeviceScope dev(ctx->device);
    if (!dev.ok) rc = fail(ctx, PA_CUDA_ECUDA, "cudaSetDevice");
    if (rc || (rc = shape_cache_plan(p))) {
        delete p;
        return rc;
    }
    cudaError_t e = cudaMalloc((void **) &p->d_part, (uint64_t) p->n_parts * shape->nkv * p->unit_rows * (shape->hd + 2) * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc((void **) &p->d_crange, ((uint64_t) n_sets * p->n_rt + 1) * sizeof(uint32_t));
    if (e == cudaSuccess && p->tc) {
        const uint32_t rows = cache->n_layers * cache->n_pages * cache->page_keys;
        const uint32_t raw = (uint32_t) pa::pre::raw_row_bytes((int) shape->quant, (int) shape->hd);
        CUtensorMap maps[2];
        // a CTA of a pair loads half of each block's K rows and all of its V rows
        if (!map_rows(&maps[0], cache->k, shape->rs, rows, raw, p->pair ? pa::pre::BN / 2 : pa::pre::BN) || !map_rows(&maps[1], cache->v, shape->rs, rows, raw, pa::pre::BN)) {
            pa_cuda_cache_plan_destroy(p);
            return fail(ctx, PA_CUDA_ECUDA, "cuTensorMapEncodeTiled (K/V rows) failed");
        }
        if ((e = cudaMalloc((void **) &p->d_maps, sizeof maps)) == cudaSuccess)
            e = cudaMemcpy(p->d_maps, maps, sizeof maps, cudaMemcpyHostToDevice);
        if (e == cudaSuccess)
            e = with_prefill(p, [&](auto q, auto nt, auto d) {
                if (p->pair) {
                    constexpr int smem = pa::pre::PairSmem<q.value, nt.value, d.value>::TOTAL + 1024;
                    return cudaFuncSetAttribute(pa::pre::prefill_pair_kernel<q.value, nt.value, d.value, true>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
                }
                constexpr int smem = pa::pre::Smem<q.value, nt.value, d.value>::TOTAL + 1024;
                return cudaFuncSetAttribute(pa::pre::prefill_kernel<q.value, nt.value, d.value, true>,
                                            cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            });
    }
    if (e != cudaSuccess) {
        pa_cuda_cache_plan_destroy(p);
        cudaGetLastError();
        return fail(ctx, e == cudaErrorMemoryAllocation ? PA_CUDA_ENOMEM : PA_CUDA_ECUDA, std::string("cache plan: ") + cudaGetErrorString(e));
    }
    *out = p;
    return PA_CUDA_OK;
}
const char *pa_cuda_cache_plan_kernel(const pa_cuda_cache_plan *plan) { return plan ? plan->kernel : ""; }
void pa_cuda_cache_plan_destroy(pa_cuda_cache_plan *plan) {
    if (!plan) return;
    DeviceScope dev(plan->device);
    if (plan->d_part) cudaFree(plan->d_part);
    if (plan->d_crange) cudaFree(plan->d_crange);
    if (plan->d_maps) cudaFree(plan->d_maps);
    delete plan;
}

int pa_cuda_cache_attn(pa_cuda_cache_plan *plan, uint32_t layer, const uint16_t *Qs, const int32_t *table, const int32_t *n_keys,
                       const int32_t *q_pos, const uint64_t *tree, float *O, float *m, float *l, void *stream) {
    if (plan && (!O || !m || !l)) return fail(plan->ctx, PA_CUDA_EINVAL, "null argument");
    return cache_attn(plan, layer, Qs, table, n_keys, q_pos, tree, O, m, l, nullptr, nullptr, stream);
}
int pa_cuda_cache_attn_reply(pa_cuda_cache_plan *plan, uint32_t layer, const uint16_t *Qs, const int32_t *table,
                             const int32_t *n_keys, const int32_t *q_pos, const uint64_t *tree, uint16_t *Oh, float *lse,
                             void *stream) {
    if (plan && (!Oh || !lse)) return fail(plan->ctx, PA_CUDA_EINVAL, "null argument");
    return cache_attn(plan, layer, Qs, table, n_keys, q_pos, tree, nullptr, nullptr, nullptr, Oh, lse, stream);
}

int pa_cuda_cache_append(pa_cuda_ctx *ctx, const pa_cuda_shape *shape, const pa_cuda_cache *cache, uint32_t layer,
                         const pa_cuda_append *in, uint32_t n_sets, uint32_t n_tok, const int32_t *table, uint32_t max_pages,
                         const int32_t *start, uint16_t *Qs, void *stream) {
    if (!ctx) return PA_CUDA_EINVAL;
    int rc = check_cache(ctx, shape, cache);
    if (rc || (rc = check_table(ctx, cache, n_sets, max_pages))) return rc;
    if (layer >= cache->n_layers) return fail(ctx, PA_CUDA_EINVAL, "layer out of range");
    if (n_sets == 0 || n_tok == 0) return PA_CUDA_OK;
    if (!in || !in->q || !in->k || !in->v || !table || !start || !Qs) return fail(ctx, PA_CUDA_EINVAL, "null argument");
    if (shape->rows % n_tok) return fail(ctx, PA_CUDA_EINVAL, "rows must be a multiple of n_tok");
    if ((uint64_t) n_sets * n_tok > 0x7FFFFFFFull) return fail(ctx, PA_CUDA_EUNSUPPORTED, "more than 2^31 - 1 tokens");
    if (in->dtype > PA_CUDA_T_F32 || in->w_dtype > PA_CUDA_T_F32 || (in->w_dtype != in->dtype && in->w_dtype != PA_CUDA_T_F32))
        return fail(ctx, PA_CUDA_EUNSUPPORTED, "inputs are f16, bf16 or f32; weights of the inputs' type or f32");
    if (in->rot % 2 || in->rot > shape->hd || (in->rot && !in->freqs))
        return fail(ctx, PA_CUDA_EINVAL, "rot must be even, at most hd, with rot / 2 frequencies");
    const uint64_t size = in->dtype == PA_CUDA_T_F32 ? 4 : 2;
    if (!aligned(16, {Qs}) || !aligned(8, {in->freqs}) || !aligned(4, {table, start, in->pos}) || !aligned(size, {in->q, in->k, in->v}) ||
        !aligned(in->w_dtype == PA_CUDA_T_F32 ? 4 : 2, {in->wq, in->wk}))
        return fail(ctx, PA_CUDA_EINVAL, "misaligned pointer (Q to 16 bytes, the others to their elements)");
    DeviceScope dev(ctx->device);
    if (!dev.ok) return fail(ctx, PA_CUDA_ECUDA, "cudaSetDevice");
    pa::pg::AppendParams a{};
    a.q = in->q;
    a.k = in->k;
    a.v = in->v;
    a.q_set = in->q_set;
    a.q_tok = in->q_tok;
    a.k_set = in->k_set;
    a.k_tok = in->k_tok;
    a.v_set = in->v_set;
    a.v_tok = in->v_tok;
    a.wq = in->wq;
    a.wk = in->wk;
    a.freqs = in->freqs;
    a.start = start;
    a.pos = in->pos;
    a.view.table = table;
    a.view.n_sets = n_sets;
    a.view.max_pages = max_pages;
    a.view.n_pages = cache->n_pages;
    a.view.page_keys = cache->page_keys;
    a.view.page_mul = page_mul(cache->page_keys);
    a.view.n_tok = n_tok;
    a.view.status = ctx->d_status + 1;
    a.K = cache->k + layer * layer_bytes(*shape, *cache);
    a.V = cache->v + layer * layer_bytes(*shape, *cache);
    a.Qs = Qs;
    a.rs = shape->rs;
    a.hb = shape->hb;
    a.nkv = shape->nkv;
    a.gqa = shape->rows / n_tok;
    a.rot = in->rot;
    a.eps = in->eps;
    a.scale = in->scale;
    a.inter = in->interleaved != 0;
    a.w32 = in->w_dtype == PA_CUDA_T_F32;
    // 16-byte loads where every head and the weights start on such a boundary
    uint64_t odd = (uintptr_t) in->q | (uintptr_t) in->k | (uintptr_t) in->v | (uintptr_t) in->wq | (uintptr_t) in->wk;
    for (int64_t x : {in->q_set, in->q_tok, in->k_set, in->k_tok, in->v_set, in->v_tok}) odd |= (uint64_t) x * size;
    const int rot = odd % 16 ? pa::pg::ROT_ANY : a.inter ? pa::pg::ROT_PAIRS : a.rot % 16 ? pa::pg::ROT_ANY : pa::pg::ROT_HALVES;
    const uint64_t tokens = (uint64_t) n_sets * n_tok, heads = (uint64_t) shape->nkv * (a.gqa + 2);
    if (heads > 65535) return fail(ctx, PA_CUDA_EUNSUPPORTED, "too many heads");
    // steps of a block's warps: one while the blocks that gives run at once (latency), else eight (64 heads at hd 128)
    const uint64_t per = pa::pg::append_heads((int) shape->hd);
    const uint32_t steps = tokens * ((heads + per - 1) / per) <= 8ull * ctx->n_sm ? 1 : 8;
    PA_CK(shape->hd == 128 ? launch_append<128>(a, in->dtype, shape->quant, steps, rot, pick(ctx, stream))
                           : launch_append<256>(a, in->dtype, shape->quant, steps, rot, pick(ctx, stream)),
          "append launch");
    ctx->launches++;
    return PA_CUDA_OK;
}

int pa_cuda_cache_rows(pa_cuda_ctx *ctx, const pa_cuda_shape *shape, const pa_cuda_cache *cache, uint32_t layer, uint32_t n_sets,
                       uint32_t n_tok, const int32_t *table, uint32_t max_pages, const int32_t *first, uint16_t *K, uint16_t *V,
                       void *stream) {
    if (!ctx) return PA_CUDA_EINVAL;
    int rc = check_cache(ctx, shape, cache);
    if (rc || (rc = check_table(ctx, cache, n_sets, max_pages))) return rc;
    if (layer >= cache->n_layers) return fail(ctx, PA_CUDA_EINVAL, "layer out of range");
    if (n_sets == 0 || n_tok == 0) return PA_CUDA_OK;
    if (!table || !first || !K || !V) return fail(ctx, PA_CUDA_EINVAL, "null argument");
    if (!aligned(16, {K, V}) || !aligned(4, {table, first})) return fail(ctx, PA_CUDA_EINVAL, "misaligned pointer (K and V to 16 bytes, the others to 4)");
    const uint64_t keys = (uint64_t) n_sets * n_tok;
    if (keys > 0x7FFFFFFFull) return fail(ctx, PA_CUDA_EUNSUPPORTED, "too many rows in one call");
    DeviceScope dev(ctx->device);
    if (!dev.ok) return fail(ctx, PA_CUDA_ECUDA, "cudaSetDevice");
    pa::pg::RowsParams a{};
    a.v.table = table;
    a.v.n_sets = n_sets;
    a.v.max_pages = max_pages;
    a.v.n_pages = cache->n_pages;
    a.v.page_keys = cache->page_keys;
    a.v.page_mul = page_mul(cache->page_keys);
    a.v.n_tok = n_tok;
    a.v.status = ctx->d_status + 1;
    a.first = first;
    a.K = cache->k + layer * layer_bytes(*shape, *cache);
    a.V = cache->v + layer * layer_bytes(*shape, *cache);
    a.Ko = K;
    a.Vo = V;
    a.rs = shape->rs;
    a.hb = shape->hb;
    a.nkv = shape->nkv;
    a.n = (uint32_t) keys;
    PA_CK(shape->hd == 128 ? launch_rows<128>(a, shape->quant, pick(ctx, stream)) : launch_rows<256>(a, shape->quant, pick(ctx, stream)),
          "cache rows launch");
    ctx->launches++;
    return PA_CUDA_OK;
}

int pa_cuda_cache_copy_pages(pa_cuda_ctx *ctx, const pa_cuda_shape *shape, const pa_cuda_cache *cache, const int32_t *src,
                             const int32_t *dst, uint32_t n, void *stream) {
    if (!ctx) return PA_CUDA_EINVAL;
    int rc = check_cache(ctx, shape, cache);
    if (rc) return rc;
    if (n == 0) return PA_CUDA_OK;
    if (!src || !dst) return fail(ctx, PA_CUDA_EINVAL, "null argument");
    if (!aligned(4, {src, dst})) return fail(ctx, PA_CUDA_EINVAL, "misaligned pointer");
    DeviceScope dev(ctx->device);
    if (!dev.ok) return fail(ctx, PA_CUDA_ECUDA, "cudaSetDevice");
    pa::pg::CopyParams a{};
    a.K = cache->k;
    a.V = cache->v;
    a.page_bytes = cache->page_keys * shape->rs;
    a.n_pages = cache->n_pages;
    a.n_layers = cache->n_layers;
    a.status = ctx->d_status + 1;
    const uint64_t per = 256ull * 16 * pa::pg::COPY_UNROLL, x = (a.page_bytes + per - 1) / per;
    if (x > 0x7FFFFFFFull) return fail(ctx, PA_CUDA_EUNSUPPORTED, "pages too large");
    for (uint32_t i = 0; i < n; i += 65535) {
        a.src = src + i;
        a.dst = dst + i;
        const dim3 grid((unsigned) x, std::min<uint32_t>(65535, n - i), 2 * cache->n_layers);
        PA_CK(launch_pdl(pa::pg::copy_pages_kernel, grid, 256, 0, pick(ctx, stream), a), "copy pages launch");
        ctx->launches++;
    }
    return PA_CUDA_OK;
}

int pa_cuda_cache_compact(pa_cuda_ctx *ctx, const pa_cuda_shape *shape, const pa_cuda_cache *cache, uint32_t n_sets,
                          uint32_t n_tok, const int32_t *table, uint32_t max_pages, const int32_t *start, const int32_t *path,
                          const int32_t *count, int32_t *n_keys_out, void *stream) {
    if (!ctx) return PA_CUDA_EINVAL;
    int rc = check_cache(ctx, shape, cache);
    if (rc || (rc = check_table(ctx, cache, n_sets, max_pages))) return rc;
    if (n_sets == 0) return PA_CUDA_OK;
    if (n_tok == 0 || n_tok > pa::pg::COMPACT_MAX) return fail(ctx, PA_CUDA_EUNSUPPORTED, "a path has 1 to 1,024 tokens");
    if (!table || !start || !path || !count) return fail(ctx, PA_CUDA_EINVAL, "null argument");
    if (!aligned(4, {table, start, path, count, n_keys_out})) return fail(ctx, PA_CUDA_EINVAL, "misaligned pointer");
    // (every block of a set reads them, one writes n_keys_out)
    if (overlap(n_keys_out, n_sets, start, n_sets) || overlap(n_keys_out, n_sets, count, n_sets) ||
        overlap(n_keys_out, n_sets, path, (uint64_t) n_sets * n_tok) || overlap(n_keys_out, n_sets, table, (uint64_t) n_sets * max_pages))
        return fail(ctx, PA_CUDA_EINVAL, "n_keys_out overlaps an input");
    DeviceScope dev(ctx->device);
    if (!dev.ok) return fail(ctx, PA_CUDA_ECUDA, "cudaSetDevice");
    pa::pg::CompactParams a{};
    a.v.table = table;
    a.v.n_sets = n_sets;
    a.v.max_pages = max_pages;
    a.v.n_pages = cache->n_pages;
    a.v.page_keys = cache->page_keys;
    a.v.page_mul = page_mul(cache->page_keys);
    a.v.n_tok = n_tok;
    a.v.status = ctx->d_status + 1;
    a.K = cache->k;
    a.V = cache->v;
    a.start = start;
    a.path = path;
    a.count = count;
    a.n_keys_out = n_keys_out;
    a.rs = shape->rs;
    a.n_layers = cache->n_layers;
    const uint64_t threads = shape->rs / 16 * 2 * cache->n_layers;
    const dim3 grid((unsigned) ((threads + 127) / 128), n_sets);
    PA_CK(launch_pdl(pa::pg::compact_kernel, grid, 128, 0, pick(ctx, stream), a), "compact launch");
    ctx->launches++;
    return PA_CUDA_OK;
}

}  // extern "C"
