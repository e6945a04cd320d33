// thk_kv8.cpp — the 8-bit K/V cache of include/thk.h: handle, argument checks, launches (kernels: thk_kv8.hip).
#include "thk_internal.hpp"
#include "thk_kv8.hpp"
#include <new>

struct thk_kv8 {
    thk_ctx* ctx = nullptr;
    int64_t n_ctx = 0;
    Kv8View view{};
    void* mem = nullptr;        // one allocation: codes, scales, tail rows
    size_t mem_bytes = 0;
    float2* ml = nullptr;       // per-row softmax statistics of an attention call that counts weights
    float* part_o = nullptr;    // parts of rows that are split over the positions
    float2* part_ml = nullptr;
    int64_t part_rows = 0;      // rows x parts they hold; the selection of long sets uses part_o too
    unsigned* counters = nullptr;
    float* scores = nullptr;    // [H][padded n_ctx]: a single row's scores, for the weight count (groups of up to kKv8ScoredHeads heads)
};

namespace {
// The context's device is current inside a call and the caller's own afterwards.
struct DeviceScope {
    int old = -1;
    hipError_t err;
    explicit DeviceScope(int device) {
        err = hipGetDevice(&old);
        if (err == hipSuccess && old != device) err = hipSetDevice(device); else old = -1;
    }
    ~DeviceScope() { if (old >= 0) (void)hipSetDevice(old); }
};
bool overlap(const void* a, size_t na, const void* b, size_t nb) { return a && b && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
// Parts that T positions are cut into at most: a tile for every wave, no more than one wave joins.
int64_t max_parts(int64_t T, int64_t D) {
    const int64_t tiles = (T + kKv8Tile - 1) / kKv8Tile, waves = kv8_split_waves((int)D);
    return std::min<int64_t>((tiles + waves - 1) / waves, 64);
}

// An allocation, a free or a blocking call inside a stream capture would break the capture: refused before anything is touched.
int refuse_capture(thk_ctx* ctx, const char* what) {
    hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
    HIPCHK(ctx, hipStreamIsCapturing(ctx->stream, &s));
    if (s != hipStreamCaptureStatusNone) return fail(ctx, THK_ERR_STATE, "%s: the context's stream is being captured", what);
    return THK_OK;
}
}  // namespace

extern "C" int thk_kv8_create(thk_ctx* ctx, int64_t n_ctx, int64_t H, int64_t H_kv, int64_t D, thk_kv8** out) {
    if (!ctx || !out) return THK_ERR_INVALID;
    *out = nullptr;
    REQUIRE(ctx, n_ctx > 0 && n_ctx <= (1 << 26), "thk_kv8_create: n_ctx=%lld outside 1 .. 2^26", (long long)n_ctx);
    REQUIRE(ctx, H > 0 && H <= 1024 && H_kv > 0 && H % H_kv == 0, "thk_kv8_create: %lld heads on %lld K/V heads (at most 1024, a multiple)", (long long)H, (long long)H_kv);
    REQUIRE(ctx, valid_head_dim(D), "thk_kv8_create: head dim %lld not in {64,128,256}", (long long)D);
    DeviceScope dev(ctx->device);
    HIPCHK(ctx, dev.err);
    const int rc = refuse_capture(ctx, "thk_kv8_create");
    if (rc != THK_OK) return rc;
    thk_kv8* kv = new (std::nothrow) thk_kv8();
    if (!kv) return fail(ctx, THK_ERR_OOM, "thk_kv8_create: out of host memory");
    kv->ctx = ctx; kv->n_ctx = n_ctx;
    Kv8View& v = kv->view;
    v.n_blk = (int)((n_ctx + kKv8Pad - 1) / kKv8Pad) * (kKv8Pad / kKv8Block);
    v.H = (int)H; v.Hkv = (int)H_kv; v.D = (int)D;
    const size_t codes = (size_t)H_kv * v.n_blk * kKv8Block * D, scales = up256((size_t)H_kv * v.n_blk * 4), tail = (size_t)2 * H_kv * kKv8Block * D * 4;
    // The workspace is what calls on this cache can ask for: no more rows than positions, no more parts than its length is cut into.
    const int64_t rows = n_ctx < kKv8RowSlab ? n_ctx : kKv8RowSlab, parts = max_parts(n_ctx, D);
    kv->part_rows = n_ctx > kKv8SliceFrom ? kKv8SliceRows : parts > 1 ? std::min<int64_t>(kKv8SplitRows, parts * rows * H) : 0;
    const size_t at = up256((size_t)2 * H_kv * sizeof(int2)), ml = up256((size_t)rows * H * sizeof(float2)), part_o = (size_t)kv->part_rows * D * 4;
    const size_t part_ml = up256((size_t)kv->part_rows * sizeof(float2)), scores_bytes = H / H_kv <= kKv8ScoredHeads ? (size_t)H * v.n_blk * kKv8Block * 4 : 0;
    kv->mem_bytes = 2 * codes + 2 * scales + tail + at + ml + part_o + part_ml + kKv8Groups * 4 + scores_bytes;
    hipError_t e = hipMalloc(&kv->mem, kv->mem_bytes);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        const size_t bytes = kv->mem_bytes;
        delete kv;
        return fail(ctx, e == hipErrorOutOfMemory ? THK_ERR_OOM : THK_ERR_HIP, "thk_kv8_create: hipMalloc(%zu): %s", bytes, hipGetErrorString(e));
    }
    char* p = (char*)kv->mem;
    v.k = (int8_t*)p; p += codes;
    v.v = (int8_t*)p; p += codes;
    v.ks = (float*)p; p += scales;
    v.vs = (float*)p; p += scales;
    v.tail = (float*)p; p += tail;
    v.tail_at = (int2*)p; p += at;
    kv->ml = (float2*)p; p += ml;
    kv->part_o = (float*)p; p += part_o;
    kv->part_ml = (float2*)p; p += part_ml;
    kv->counters = (unsigned*)p; p += kKv8Groups * 4;
    kv->scores = (float*)p;
    e = hipMemsetAsync(kv->mem, 0, kv->mem_bytes, ctx->stream);
    if (e == hipSuccess) e = hipMemsetAsync(v.tail_at, 0xFF, (size_t)2 * H_kv * sizeof(int2), ctx->stream);     // no block is open
    if (e != hipSuccess) {
        (void)hipFree(kv->mem);
        delete kv;
        return fail(ctx, THK_ERR_HIP, "thk_kv8_create: hipMemsetAsync: %s", hipGetErrorString(e));
    }
    *out = kv;
    return THK_OK;
}
extern "C" int thk_kv8_destroy(thk_kv8* kv) {
    if (!kv) return THK_OK;
    DeviceScope dev(kv->ctx->device);
    const int rc = refuse_capture(kv->ctx, "thk_kv8_destroy");
    if (rc != THK_OK) return rc;
    (void)hipStreamSynchronize(kv->ctx->stream);
    (void)hipFree(kv->mem);
    delete kv;
    return THK_OK;
}
extern "C" int64_t thk_kv8_bytes(const thk_kv8* kv) { return kv ? (int64_t)kv->mem_bytes : 0; }
extern "C" int64_t thk_kv8_n_ctx(const thk_kv8* kv) { return kv ? kv->n_ctx : 0; }

extern "C" int thk_kv8_append(thk_kv8* kv, const float* k, const float* v, int64_t pos, int64_t n_tok) {
    if (!kv) return THK_ERR_INVALID;
    thk_ctx* ctx = kv->ctx;
    REQUIRE(ctx, k && v && pos >= 0 && n_tok > 0, "thk_kv8_append: bad arguments");
    REQUIRE(ctx, pos <= kv->n_ctx && n_tok <= kv->n_ctx - pos, "thk_kv8_append: positions [%lld, %lld + %lld) outside the cache of %lld", (long long)pos, (long long)pos,
            (long long)n_tok, (long long)kv->n_ctx);
    REQUIRE(ctx, aligned16(k) && aligned16(v), "thk_kv8_append: k and v must be 16-byte aligned");
    DeviceScope dev(ctx->device);
    HIPCHK(ctx, dev.err);
    HIPCHK(ctx, launch_kv8_append(kv->view, k, v, pos, n_tok, ctx->stream));
    return THK_OK;
}
extern "C" int thk_kv8_read(thk_kv8* kv, int64_t pos, int64_t n_tok, float* k_out, float* v_out) {
    if (!kv) return THK_ERR_INVALID;
    thk_ctx* ctx = kv->ctx;
    REQUIRE(ctx, (k_out || v_out) && pos >= 0 && n_tok > 0, "thk_kv8_read: bad arguments");
    REQUIRE(ctx, pos <= kv->n_ctx && n_tok <= kv->n_ctx - pos, "thk_kv8_read: positions [%lld, %lld + %lld) outside the cache of %lld", (long long)pos, (long long)pos,
            (long long)n_tok, (long long)kv->n_ctx);
    REQUIRE(ctx, aligned16(k_out) && aligned16(v_out), "thk_kv8_read: k_out and v_out must be 16-byte aligned");
    const size_t bytes = (size_t)n_tok * kv->view.Hkv * kv->view.D * 4;
    REQUIRE(ctx, !overlap(k_out, bytes, v_out, bytes), "thk_kv8_read: k_out and v_out overlap");
    DeviceScope dev(ctx->device);
    HIPCHK(ctx, dev.err);
    HIPCHK(ctx, launch_kv8_read(kv->view, pos, n_tok, k_out, v_out, ctx->stream));
    return THK_OK;
}

// rows [0, M) at positions n_past + i, in slabs of kKv8RowSlab rows (the statistics of a slab fit the cache's workspace)
static int kv8_attention(thk_kv8* kv, const char* what, const float* q, int64_t n_past, int64_t M, const float* mass_in, float* mass_out, float* out) {
    thk_ctx* ctx = kv->ctx;
    REQUIRE(ctx, q && out, "%s: null pointer", what);
    REQUIRE(ctx, (mass_in != nullptr) == (mass_out != nullptr), "%s: mass_in and mass_out go together", what);
    REQUIRE(ctx, aligned16(q) && aligned16(out) && aligned16(mass_in) && aligned16(mass_out), "%s: pointers must be 16-byte aligned", what);
    const size_t row = (size_t)kv->view.H * kv->view.D, rows = (size_t)M * row * 4;
    const size_t weights = ((size_t)(kv->view.Hkv - 1) * kv->n_ctx + n_past + M) * 4;                  // up to the last entry that is touched
    REQUIRE(ctx, !overlap(q, rows, out, rows), "%s: q and out overlap", what);
    REQUIRE(ctx, mass_in == mass_out || !overlap(mass_in, weights, mass_out, weights), "%s: mass_in and mass_out overlap and are not the same array", what);
    REQUIRE(ctx, !overlap(out, rows, mass_in, weights) && !overlap(out, rows, mass_out, weights) && !overlap(q, rows, mass_out, weights), "%s: the weights overlap q or out", what);
    DeviceScope dev(ctx->device);
    HIPCHK(ctx, dev.err);
    for (int64_t i = 0; i < M; i += kKv8RowSlab) {
        Kv8Attn a{};
        a.c = kv->view; a.q = q + i * row; a.out = out + i * row;
        a.n_past = (int)(n_past + i); a.M = (int)(M - i < kKv8RowSlab ? M - i : kKv8RowSlab);
        if (mass_out) { a.ml = kv->ml; a.mass_in = mass_in; a.mass_out = mass_out; a.mass_ld = kv->n_ctx; a.mass_n = (int)(n_past + M); }
        bool scored = false;
        const int64_t G = a.c.H / a.c.Hkv, cols = a.M * G, cg = (cols + 15) / 16, groups = cg * a.c.Hkv;      // workgroups without a split
        // Few columns: split over the positions, a tile of 64 a wave in turn; many: whole rows, tiles shared by a workgroup.  32 heads of 128, split and
        // rows: no past, 512 groups 11.2 and 10.7 us, 768 17.6 and 12.9; over 1024 positions 22.6 and 29.3, 34.2 and 32.3; over 8192 91 and 148, 138 and 155.
        // The rule does not look at the length: 768 groups over 8192 positions would be 17 us faster split.
        if (groups <= kKv8Groups) {
            Kv8Split sp{};
            const int64_t T = a.n_past + a.M;
            const int64_t n = std::min(256 / groups, max_parts(T, a.c.D));              // one workgroup on every CU
            sp.n = n < 1 ? 1 : (int)n; sp.part_o = kv->part_o; sp.part_ml = kv->part_ml;
            sp.stream = cg == 1 && 2 * T * a.c.Hkv * a.c.D >= (64 << 20);  // twice what the L2s hold: 112 -> 100 us at 65535 x 32 heads; at 2047 x 40 heads 10.4 -> 11.1
            // Joined inside the launch where the last workgroup has little to do: 4096 positions, 32 heads on 8, 10.4 -> 9.7 us, at 8192 10.8 -> 11.3; and
            // the weights counted there, too: 2048 positions 17.4 -> 13.2 us, 8192 19.6 -> 23.3.
            const bool inside = sp.n * std::min<int64_t>(cols, 16) <= 64, count = mass_out && a.M == 1 && G <= kKv8ScoredHeads;
            const bool count_inside = inside && T <= 4096;
            scored = count && (count_inside || sp.n > 1);
            if (scored) { sp.scores = kv->scores; sp.scores_ld = (int64_t)a.c.n_blk * kKv8Block; }
            if (scored ? count_inside : inside && sp.n > 1) sp.counters = kv->counters;
            HIPCHK(ctx, launch_kv8_attn_split(a, sp, ctx->stream));
        } else {
            a.halves = true;
            HIPCHK(ctx, launch_kv8_attn_tile(a, ctx->stream));
        }
        if (mass_out && !scored) HIPCHK(ctx, launch_kv8_attn_mass(a, ctx->stream));
        mass_in = mass_out;
    }
    return THK_OK;
}
extern "C" int thk_kv8_attn_decode(thk_kv8* kv, const float* q, int64_t T, const float* mass_in, float* mass_out, float* out) {
    if (!kv) return THK_ERR_INVALID;
    REQUIRE(kv->ctx, T > 0 && T <= kv->n_ctx, "thk_kv8_attn_decode: T=%lld outside 1 .. %lld", (long long)T, (long long)kv->n_ctx);
    return kv8_attention(kv, "thk_kv8_attn_decode", q, T - 1, 1, mass_in, mass_out, out);
}
extern "C" int thk_kv8_attn_prefill(thk_kv8* kv, const float* q, int64_t n_past, int64_t M, const float* mass_in, float* mass_out, float* out) {
    if (!kv) return THK_ERR_INVALID;
    REQUIRE(kv->ctx, n_past >= 0 && M > 0 && n_past <= kv->n_ctx && M <= kv->n_ctx - n_past, "thk_kv8_attn_prefill: rows [%lld, %lld + %lld) outside the cache of %lld",
            (long long)n_past, (long long)n_past, (long long)M, (long long)kv->n_ctx);
    return kv8_attention(kv, "thk_kv8_attn_prefill", q, n_past, M, mass_in, mass_out, out);
}
extern "C" int thk_kv8_evict(thk_kv8* src, int64_t T, int64_t n_keep, int64_t n_sink, int64_t n_recent, const float* mass_in, thk_kv8* dst, float* mass_out, int32_t* kept) {
    if (!src || !dst) return THK_ERR_INVALID;
    thk_ctx* ctx = src->ctx;
    REQUIRE(ctx, src != dst, "thk_kv8_evict: source and destination are the same cache");
    REQUIRE(ctx, dst->ctx == ctx, "thk_kv8_evict: the caches belong to different contexts");
    REQUIRE(ctx, dst->view.Hkv == src->view.Hkv && dst->view.D == src->view.D, "thk_kv8_evict: the caches differ in K/V heads or head dim");
    REQUIRE(ctx, T > 0 && T <= src->n_ctx && n_keep > 0 && n_keep <= T && n_keep <= dst->n_ctx, "thk_kv8_evict: T=%lld n_keep=%lld for caches of %lld and %lld", (long long)T,
            (long long)n_keep, (long long)src->n_ctx, (long long)dst->n_ctx);
    REQUIRE(ctx, n_sink >= 0 && n_recent >= 0 && n_sink <= n_keep && n_recent <= n_keep - n_sink, "thk_kv8_evict: n_sink=%lld + n_recent=%lld exceed n_keep=%lld", (long long)n_sink,
            (long long)n_recent, (long long)n_keep);
    REQUIRE(ctx, mass_in && kept, "thk_kv8_evict: null pointer");
    REQUIRE(ctx, mass_in != mass_out, "thk_kv8_evict: mass_out must not be mass_in");
    REQUIRE(ctx, aligned16(mass_in) && aligned16(mass_out) && aligned16(kept), "thk_kv8_evict: pointers must be 16-byte aligned");
    const size_t in = ((size_t)(src->view.Hkv - 1) * src->n_ctx + T) * 4, to = ((size_t)(src->view.Hkv - 1) * dst->n_ctx + n_keep) * 4, list = (size_t)src->view.Hkv * n_keep * 4;
    REQUIRE(ctx, !overlap(mass_in, in, mass_out, to) && !overlap(mass_in, in, kept, list) && !overlap(mass_out, to, kept, list), "thk_kv8_evict: mass_in, mass_out and kept overlap");
    DeviceScope dev(ctx->device);
    HIPCHK(ctx, dev.err);
    HIPCHK(ctx, launch_kv8_select(src->view.Hkv, (int)T, (int)n_keep, (int)n_sink, (int)n_recent, mass_in, src->n_ctx, mass_out, dst->n_ctx, kept,
                                  reinterpret_cast<unsigned*>(src->part_o), src->part_rows * src->view.D, ctx->stream));
    HIPCHK(ctx, launch_kv8_move(src->view, dst->view, (int)n_keep, kept, ctx->stream));
    return THK_OK;
}
