// Host-only stand-ins for what thk_kv8.cpp calls: memory on the host, launches written down instead of made.  Built by test_kv8_host.py.
#include "../token-hawk_amd/csrc/thk_internal.hpp"
#include "../token-hawk_amd/csrc/thk_kv8.hpp"

static int g_device = 0, g_capturing = 0, g_malloc_fails = 0, g_launch_fails = 0;
static std::string g_log;
static void note(const char* fmt, ...) {
    char b[256]; va_list ap; va_start(ap, fmt); vsnprintf(b, sizeof b, fmt, ap); va_end(ap);
    g_log += std::to_string(g_device) + ":" + b + ";";
}
static hipError_t launched() { return g_launch_fails ? hipErrorLaunchFailure : hipSuccess; }

extern "C" hipError_t hipGetDevice(int* d) { *d = g_device; return hipSuccess; }
extern "C" hipError_t hipSetDevice(int d) { g_device = d; return hipSuccess; }
#undef hipMalloc
extern "C" hipError_t hipMalloc(void** p, size_t n) { if (g_malloc_fails) return hipErrorOutOfMemory; *p = malloc(16); note("malloc %zu", n); return hipSuccess; }
extern "C" hipError_t hipFree(void* p) { free(p); note("free"); return hipSuccess; }
extern "C" hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t) { return hipSuccess; }
extern "C" hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) { *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone; return hipSuccess; }
extern "C" hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
extern "C" hipError_t hipGetLastError(void) { return hipSuccess; }
extern "C" const char* hipGetErrorString(hipError_t) { return "stub"; }

int fail(thk_ctx* ctx, int code, const char* fmt, ...) {
    char b[512]; va_list ap; va_start(ap, fmt); vsnprintf(b, sizeof b, fmt, ap); va_end(ap);
    ctx->err = b;
    return code;
}
int valid_head_dim(int64_t D) { return D == 64 || D == 128 || D == 256; }
int64_t tun(thk_ctx*, const char*) { return 0; }

namespace thk {
hipError_t launch_kv8_append(const Kv8View&, const float*, const float*, int64_t pos, int64_t n, hipStream_t) { note("append %lld %lld", (long long)pos, (long long)n); return launched(); }
hipError_t launch_kv8_read(const Kv8View&, int64_t pos, int64_t n, float*, float*, hipStream_t) { note("read %lld %lld", (long long)pos, (long long)n); return launched(); }
hipError_t launch_kv8_select(int Hkv, int T, int keep, int sink, int recent, const float*, int64_t li, float*, int64_t lo, int32_t*, unsigned*, int64_t, hipStream_t) {
    note("select %d %d %d %d %d %lld %lld", Hkv, T, keep, sink, recent, (long long)li, (long long)lo); return launched();
}
hipError_t launch_kv8_move(const Kv8View&, const Kv8View&, int keep, const int32_t*, hipStream_t) { note("move %d", keep); return launched(); }
hipError_t launch_kv8_attn_tile(const Kv8Attn& a, hipStream_t) { note("tile %d %d", a.n_past, a.M); return launched(); }
hipError_t launch_kv8_attn_split(const Kv8Attn& a, const Kv8Split& sp, hipStream_t) {
    const size_t rows = (size_t)a.M * a.c.H * (sp.n > 1 ? sp.n : 0);       // parts and statistics have to fit between their arrays' starts
    if ((const char*)(sp.part_o + rows * a.c.D) > (const char*)sp.part_ml || (a.ml && (const char*)(a.ml + (size_t)a.M * a.c.H) > (const char*)sp.part_o)) return hipErrorOutOfMemory;
    if (sp.counters ? (const char*)(sp.part_ml + rows) > (const char*)sp.counters : sp.scores && (const char*)(sp.part_ml + rows) > (const char*)sp.scores) return hipErrorOutOfMemory;
    note("split %d %d %d", a.n_past, a.M, sp.n); return launched(); }
hipError_t launch_kv8_attn_mass(const Kv8Attn& a, hipStream_t) { note("mass %d %d %d%s", a.n_past, a.M, a.mass_n, a.mass_in == a.mass_out ? " in place" : ""); return launched(); }
}

extern "C" thk_ctx* stub_ctx(int device) { thk_ctx* c = new thk_ctx(); c->device = device; return c; }
extern "C" const char* stub_error(thk_ctx* c) { return c->err.c_str(); }
extern "C" void stub_set(int device, int capturing, int malloc_fails, int launch_fails) { g_device = device; g_capturing = capturing; g_malloc_fails = malloc_fails; g_launch_fails = launch_fails; }
extern "C" int stub_device(void) { return g_device; }
extern "C" const char* stub_log(void) { static std::string out; out = g_log; g_log.clear(); return out.c_str(); }
