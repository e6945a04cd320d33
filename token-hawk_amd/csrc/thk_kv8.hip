// thk_kv8.hip — kernels of the 8-bit K/V cache: append (quantise), read (dequantise), attention over the codes, eviction.
// Layout: thk_kv8.hpp.  All sums, softmax statistics and scales are f32; the codes are the only 8-bit values.
#include "thk_device.hpp"
#include "thk_kv8.hpp"

namespace thk {

// ---------------------------------------------------------------- quantiser
// A block's scale is f32(amax / 127), its codes rint(x * f32(127 / amax)).  fma with 1.5 * 2^23 rounds the exact product once, to the
// nearest integer (ties to even): the code does not depend on a rounding of the product, and the low byte of the sum's bits is the code.
// amax below 2^-100 counts as zero (127 / amax would leave the f32 range); an amax that is not finite gives the block a NaN scale, so
// that whoever reads it sees NaN and not a clipped number.
struct Quant { float inv, scale; };
__device__ __forceinline__ Quant quant_of(unsigned amax_bits) {
    const float amax = __builtin_bit_cast(float, amax_bits);
    if (amax_bits >= 0x7F800000u) return {0.f, __builtin_bit_cast(float, 0x7FC00000u)};
    if (amax < 0x1p-100f) return {0.f, 0.f};
    return {127.f / amax, amax / 127.f};
}
__device__ __forceinline__ unsigned quant_code(float x, float inv) { return __builtin_bit_cast(unsigned, fmaf(x, inv, 12582912.f)) & 0xFFu; }
__device__ __forceinline__ unsigned abs_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7FFFFFFFu; }   // orders magnitudes; NaN above infinity

// maximum over the workgroup's 256 threads; sm: 4 words
__device__ __forceinline__ unsigned block_max_u32(unsigned v, unsigned* sm) {
#pragma unroll
    for (int o = 32; o; o >>= 1) { const unsigned u = (unsigned)__shfl_xor((int)v, o); v = u > v ? u : v; }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    const unsigned a = sm[0] > sm[1] ? sm[0] : sm[1], b = sm[2] > sm[3] ? sm[2] : sm[3];
    return a > b ? a : b;
}

// The 256 threads of a workgroup hold a block's 16 x D numbers, D / 16 each: for K thread t has row t / 16, dimensions
// (t % 16) * D/16 + i; for V dimension t % D, rows (t / D) * D/16 + i.  Either way a thread's codes are D / 16 contiguous bytes.
template <int D, bool V> __device__ __forceinline__ int el_row(int i) { return V ? (int)(threadIdx.x / D) * (D / 16) + i : (int)(threadIdx.x >> 4); }
template <int D, bool V> __device__ __forceinline__ int el_dim(int i) { return V ? (int)(threadIdx.x % D) : (int)(threadIdx.x & 15) * (D / 16) + i; }
template <int D, bool V> __device__ __forceinline__ int code_at() { return V ? (int)(threadIdx.x % D) * 16 + (int)(threadIdx.x / D) * (D / 16) : (int)threadIdx.x * (D / 16); }

template <int D> __device__ __forceinline__ void put_codes(int8_t* p, const unsigned (&q)[D / 16]) {
    unsigned* w = reinterpret_cast<unsigned*>(p);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) w[i] = q[4 * i] | (q[4 * i + 1] << 8) | (q[4 * i + 2] << 16) | (q[4 * i + 3] << 24);
}

// ---------------------------------------------------------------- append
// One workgroup per block, head and K | V: reads the block's older rows (unrounded where tail still holds them, else as the values of
// their codes), the new ones from x [n][Hkv][D], and writes the whole block anew.  Because the open block is always requantised from
// unrounded rows, n calls of one token leave the same bits as one call of n.  The last block's rows go to tail; when the call spans
// several blocks the first workgroup also takes the last block, after the first: nobody else reads or writes tail.
template <int D, bool V>
__device__ void append_block(const Kv8View& c, int h, int b, const float* x, int64_t pos, int64_t n, bool last, unsigned* sm) {
    const int64_t p0 = (int64_t)b * kKv8Block;
    const int r0 = pos > p0 ? (int)(pos - p0) : 0;                                                  // rows before the new ones
    const int r1 = pos + n < p0 + kKv8Block ? (int)(pos + n - p0) : kKv8Block;                      // end of the new ones
    const size_t hb = (size_t)h * c.n_blk + b;
    int8_t* codes = (V ? c.v : c.k) + hb * (kKv8Block * D) + code_at<D, V>();
    float* scale = (V ? c.vs : c.ks) + hb;
    float* tail = c.tail + ((size_t)(V ? c.Hkv : 0) + h) * (kKv8Block * D);
    int2* at = c.tail_at + (V ? c.Hkv : 0) + h;
    float xs[D / 16];
    unsigned m = 0;
    int held = 0;
    float old = 0.f;
    if (r0 > 0) { const int2 t = *at; held = t.x == b ? t.y : 0; old = *scale; }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const int r = el_row<D, V>(i), d = el_dim<D, V>(i);
        float e = 0.f;
        if (r >= r0 && r < r1) e = x[((size_t)(p0 + r - pos) * c.Hkv + h) * D + d];
        else if (r < r0) e = r < held ? tail[r * D + d] : (float)codes[i] * old;
        xs[i] = e;
        const unsigned a = abs_bits(e);
        m = a > m ? a : m;
    }
    const Quant qz = quant_of(block_max_u32(m, sm));
    unsigned q[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) q[i] = qz.inv == 0.f ? 0u : quant_code(xs[i], qz.inv);
    put_codes<D>(codes, q);
    if (threadIdx.x == 0) *scale = qz.scale;
    if (last) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) tail[el_row<D, V>(i) * D + el_dim<D, V>(i)] = xs[i];
        if (threadIdx.x == 0) *at = int2{b, r1};
    }
}
template <int D, bool V>
__device__ __forceinline__ void append_body(const Kv8View& c, const float* x, int64_t pos, int64_t n) {
    __shared__ unsigned sm[4];
    const int h = blockIdx.y, b0 = (int)(pos / kKv8Block), b1 = (int)((pos + n - 1) / kKv8Block);
    append_block<D, V>(c, h, b0 + blockIdx.x, x, pos, n, b0 + (int)blockIdx.x == b1, sm);
    if (blockIdx.x == 0 && b1 > b0) append_block<D, V>(c, h, b1, x, pos, n, true, sm);
}
template <int D>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8View c, const float* __restrict__ k, const float* __restrict__ v, int64_t pos, int64_t n) {
    if (blockIdx.z == 0) append_body<D, false>(c, k, pos, n);
    else append_body<D, true>(c, v, pos, n);
}

// ---------------------------------------------------------------- read
template <int D, bool V>
__device__ __forceinline__ void read_body(const Kv8View& c, int64_t pos, int64_t n, float* out) {
    const int h = blockIdx.y, b = (int)(pos / kKv8Block) + blockIdx.x;
    const size_t hb = (size_t)h * c.n_blk + b;
    const int8_t* codes = (V ? c.v : c.k) + hb * (kKv8Block * D) + code_at<D, V>();
    const float s = (V ? c.vs : c.ks)[hb];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const int64_t p = (int64_t)b * kKv8Block + el_row<D, V>(i);
        if (p >= pos && p < pos + n) out[((size_t)(p - pos) * c.Hkv + h) * D + el_dim<D, V>(i)] = (float)codes[i] * s;
    }
}
template <int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8View c, int64_t pos, int64_t n, float* __restrict__ k_out, float* __restrict__ v_out) {
    if (blockIdx.z == 0) { if (k_out) read_body<D, false>(c, pos, n, k_out); }
    else if (v_out) read_body<D, true>(c, pos, n, v_out);
}

// ---------------------------------------------------------------- eviction
// Weights as unsigned keys, heaviest first: order-preserving, -0 = +0, NaN (the weight of a row nobody could attend) below everything.
__device__ __forceinline__ unsigned mass_key(float x) {
    const unsigned b = __builtin_bit_cast(unsigned, x + 0.f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// Exclusive prefix sum over 1024 threads; *total gets the sum.  sm: 16 words
__device__ __forceinline__ unsigned block_scan_1024(unsigned v, unsigned* sm, unsigned* total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const unsigned u = (unsigned)__shfl_up((int)s, o); if (lane >= o) s += u; }
    __syncthreads();
    if (lane == 63) sm[w] = s;
    __syncthreads();
    unsigned before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) { const unsigned t = sm[i]; if (i < w) before += t; all += t; }
    *total = all;
    return before + s - v;
}
// One workgroup per K/V head: the n_keep - n_sink - n_recent heaviest of the middle positions by radix selection (four passes of 8 bits,
// histograms in LDS), ties to the lowest position, then the kept positions in ascending order.
__global__ __launch_bounds__(1024) void kv8_select_kernel(int T, int n_keep, int n_sink, int n_recent, const float* __restrict__ mass_in, int64_t ld_in,
                                                          float* __restrict__ mass_out, int64_t ld_out, int32_t* __restrict__ kept) {
    __shared__ unsigned hist[256], sm[16], pick[2];
    const int h = blockIdx.x, tid = threadIdx.x, lo = n_sink, hi = T - n_recent;
    const float* mass = mass_in + (size_t)h * ld_in;
    unsigned need = (unsigned)(n_keep - n_sink - n_recent), prefix = 0;     // of the positions whose key starts with prefix, the `need` heaviest stay
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int t = lo + tid; t < hi; t += 1024) {
            const unsigned key = mass_key(mass[t]);
            if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);    // integer: the order changes nothing
        }
        __syncthreads();
        unsigned total;
        const unsigned mine = tid < 256 ? hist[255 - tid] : 0u;              // thread i: the bucket of digit 255 - i
        const unsigned above = block_scan_1024(mine, sm, &total);
        if (tid < 256 && above < need && need <= above + mine) { pick[0] = 255u - tid; pick[1] = need - above; }
        if (tid == 0 && need == 0) { pick[0] = 255u; pick[1] = 0u; }
        __syncthreads();
        prefix = (prefix << 8) | pick[0];
        need = pick[1];
        __syncthreads();
    }
    // every thread takes a contiguous share of the positions: heavier ones stay, of those equal to the threshold the first `need`
    const int per = (T + 1023) / 1024, t0 = tid * per < T ? tid * per : T, t1 = t0 + per < T ? t0 + per : T;
    unsigned eq = 0, dummy;
    for (int t = t0; t < t1; ++t) if (t >= lo && t < hi) eq += mass_key(mass[t]) == prefix;
    unsigned rank = block_scan_1024(eq, sm, &dummy);
    unsigned cnt = 0, r = rank;
    for (int t = t0; t < t1; ++t) {
        if (t < lo || t >= hi) { ++cnt; continue; }
        const unsigned key = mass_key(mass[t]);
        cnt += key > prefix || (key == prefix && r < need);
        r += key == prefix;
    }
    unsigned at = block_scan_1024(cnt, sm, &dummy);
    r = rank;
    for (int t = t0; t < t1; ++t) {
        bool stay = t < lo || t >= hi;
        if (!stay) {
            const unsigned key = mass_key(mass[t]);
            stay = key > prefix || (key == prefix && r < need);
            r += key == prefix;
        }
        if (stay) { kept[(size_t)h * n_keep + at] = t; if (mass_out) mass_out[(size_t)h * ld_out + at] = mass[t]; ++at; }
    }
}
// One workgroup per destination block, head and K | V: gathers the 16 kept rows as values and quantises them anew.  Sixteen rows that were
// one block stay as they are (codes and scale), so that what eviction leaves in place does not drift.
template <int D, bool V>
__device__ __forceinline__ void move_body(const Kv8View& s, const Kv8View& d, int n_keep, const int32_t* kept, unsigned* sm, int* src) {
    const int h = blockIdx.y, b = blockIdx.x, rows = n_keep - b * kKv8Block < kKv8Block ? n_keep - b * kKv8Block : kKv8Block;
    if (threadIdx.x < kKv8Block) src[threadIdx.x] = (int)threadIdx.x < rows ? kept[(size_t)h * n_keep + b * kKv8Block + threadIdx.x] : -1;
    __syncthreads();
    const bool whole = src[0] % kKv8Block == 0 && src[15] == src[0] + 15;
    const int8_t* from = (V ? s.v : s.k) + (size_t)h * s.n_blk * (kKv8Block * D);
    const float* sc = (V ? s.vs : s.ks) + (size_t)h * s.n_blk;
    const size_t hb = (size_t)h * d.n_blk + b;
    float xs[D / 16];
    unsigned q[D / 16], m = 0;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const int p = src[el_row<D, V>(i)], dim = el_dim<D, V>(i);
        int code = 0;
        float scale = 0.f;
        if (p >= 0) { code = V ? from[((size_t)(p >> 4) * D + dim) * 16 + (p & 15)] : from[(size_t)p * D + dim]; scale = sc[p >> 4]; }
        q[i] = (unsigned)code & 0xFFu;
        xs[i] = (float)code * scale;
        const unsigned a = abs_bits(xs[i]);
        m = a > m ? a : m;
    }
    const Quant qz = quant_of(block_max_u32(m, sm));
    float scale = qz.scale;
    if (whole) scale = sc[src[0] >> 4];
    else {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) q[i] = qz.inv == 0.f ? 0u : quant_code(xs[i], qz.inv);
    }
    put_codes<D>((V ? d.v : d.k) + hb * (kKv8Block * D) + code_at<D, V>(), q);
    if (threadIdx.x == 0) (V ? d.vs : d.ks)[hb] = scale;
    if ((b + 1) * kKv8Block >= n_keep) {
        float* tail = d.tail + ((size_t)(V ? d.Hkv : 0) + h) * (kKv8Block * D);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) tail[el_row<D, V>(i) * D + el_dim<D, V>(i)] = xs[i];
        if (threadIdx.x == 0) d.tail_at[(V ? d.Hkv : 0) + h] = int2{b, rows};
    }
}
template <int D>
__global__ __launch_bounds__(256) void kv8_move_kernel(Kv8View s, Kv8View d, int n_keep, const int32_t* __restrict__ kept) {
    __shared__ unsigned sm[4];
    __shared__ int src[16];
    if (blockIdx.z == 0) move_body<D, false>(s, d, n_keep, kept, sm, src);
    else move_body<D, true>(s, d, n_keep, kept, sm, src);
}

// ---------------------------------------------------------------- attention, one workgroup per (row, head)
// Block by block: 16 threads share a position's score, then every thread adds its dimension's share with the running maximum and sum
// of the softmax.  Scores carry log2(e), so that the weights are exp2.
static const float kLog2e = 1.44269504088896340736f;
template <int D>
__device__ __forceinline__ float block_score(const Kv8View& c, const float* q, int hkv, int b, float scale) {     // of position 16 b + tid / 16, in all 16 threads of it
    const size_t hb = (size_t)hkv * c.n_blk + b;
    const int8_t* k = c.k + hb * (kKv8Block * D) + threadIdx.x * (D / 16);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) s = fmaf((float)k[i], q[(threadIdx.x & 15) * (D / 16) + i], s);
    return row16_sum(s) * (c.ks[hb] * scale);
}
template <int D>
__global__ __launch_bounds__(256) void kv8_attn_rows_kernel(Kv8Attn a, float scale) {
    __shared__ float qs[D], ss[16], acc[256];
    const Kv8View& c = a.c;
    const int h = blockIdx.x, row = blockIdx.y, hkv = h / (c.H / c.Hkv), tid = threadIdx.x, T = a.n_past + row + 1;
    const float* q = a.q + ((size_t)row * c.H + h) * D;
    for (int d = tid; d < D; d += 256) qs[d] = q[d];
    __syncthreads();
    float m = -INFINITY, l = 0.f, o = 0.f;
    constexpr int NG = 256 / D, PT = 16 / NG;                               // thread: dimension tid % D, positions (tid / D) * PT + i of the block
    for (int b = 0; b * kKv8Block < T; ++b) {
        const float s = block_score<D>(c, qs, hkv, b, scale);
        if ((tid & 15) == 0) ss[tid >> 4] = b * kKv8Block + (tid >> 4) < T ? s : -INFINITY;
        __syncthreads();
        float mb = m;
#pragma unroll
        for (int t = 0; t < 16; ++t) mb = fmaxf(mb, ss[t]);
        const float mu = mb == -INFINITY ? 0.f : mb, al = exp2f(m - mu);
        const size_t hb = (size_t)hkv * c.n_blk + b;
        const int8_t* v = c.v + hb * (kKv8Block * D) + (tid % D) * 16 + (tid / D) * PT;
        const float vs = c.vs[hb];
        float ob = 0.f, lb = 0.f;
#pragma unroll
        for (int t = 0; t < 16; ++t) lb += exp2f(ss[t] - mu);
#pragma unroll
        for (int i = 0; i < PT; ++i) ob = fmaf(exp2f(ss[(tid / D) * PT + i] - mu), (float)v[i], ob);
        o = fmaf(o, al, ob * vs); l = fmaf(l, al, lb); m = mb;
        __syncthreads();
    }
    acc[tid] = o;
    __syncthreads();
    if (tid < D) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) t += acc[g * D + tid];
        a.out[((size_t)row * c.H + h) * D + tid] = t / l;
    }
    if (tid == 0 && a.ml) a.ml[(size_t)row * c.H + h] = float2{m, l};
}
// mass_out = mass_in + the softmax weights of every row and head of the group; one workgroup per block and K/V head, rows and heads in order
template <int D>
__global__ __launch_bounds__(256) void kv8_attn_mass_kernel(Kv8Attn a, float scale) {
    __shared__ float qs[D];
    const Kv8View& c = a.c;
    const int b = blockIdx.x, hkv = blockIdx.y, G = c.H / c.Hkv, tid = threadIdx.x, t = b * kKv8Block + (tid >> 4);
    float sum = 0.f;
    for (int row = 0; row < a.M; ++row) {
        if (b * kKv8Block > a.n_past + row) continue;
        for (int g = 0; g < G; ++g) {
            const int h = hkv * G + g;
            __syncthreads();
            for (int d = tid; d < D; d += 256) qs[d] = a.q[((size_t)row * c.H + h) * D + d];
            __syncthreads();
            const float s = block_score<D>(c, qs, hkv, b, scale);
            const float2 ml = a.ml[(size_t)row * c.H + h];
            if (t <= a.n_past + row) sum += exp2f(s - ml.x) / ml.y;
        }
    }
    if ((tid & 15) == 0 && t < a.mass_n) a.mass_out[(size_t)hkv * a.mass_ld + t] = a.mass_in[(size_t)hkv * a.mass_ld + t] + sum;
}

// ---------------------------------------------------------------- launchers
#define KV8_BY_DIM(D, EXPR)                                   \
    switch (D) {                                              \
        case 64: { constexpr int kD = 64; EXPR; break; }      \
        case 128: { constexpr int kD = 128; EXPR; break; }    \
        case 256: { constexpr int kD = 256; EXPR; break; }    \
        default: return hipErrorInvalidValue;                 \
    }

hipError_t launch_kv8_append(const Kv8View& c, const float* k, const float* v, int64_t pos, int64_t n, hipStream_t st) {
    const int64_t blocks = (pos + n - 1) / kKv8Block - pos / kKv8Block + 1;
    const dim3 grid((unsigned)(blocks > 1 ? blocks - 1 : 1), c.Hkv, 2);
    KV8_BY_DIM(c.D, hipLaunchKernelGGL(kv8_append_kernel<kD>, grid, dim3(256), 0, st, c, k, v, pos, n));
    return hipGetLastError();
}
hipError_t launch_kv8_read(const Kv8View& c, int64_t pos, int64_t n, float* k_out, float* v_out, hipStream_t st) {
    const dim3 grid((unsigned)((pos + n - 1) / kKv8Block - pos / kKv8Block + 1), c.Hkv, 2);
    KV8_BY_DIM(c.D, hipLaunchKernelGGL(kv8_read_kernel<kD>, grid, dim3(256), 0, st, c, pos, n, k_out, v_out));
    return hipGetLastError();
}
hipError_t launch_kv8_select(int Hkv, int T, int n_keep, int n_sink, int n_recent, const float* mass_in, int64_t ld_in, float* mass_out, int64_t ld_out, int32_t* kept,
                             hipStream_t st) {
    hipLaunchKernelGGL(kv8_select_kernel, dim3(Hkv), dim3(1024), 0, st, T, n_keep, n_sink, n_recent, mass_in, ld_in, mass_out, ld_out, kept);
    return hipGetLastError();
}
hipError_t launch_kv8_move(const Kv8View& src, const Kv8View& dst, int n_keep, const int32_t* kept, hipStream_t st) {
    const dim3 grid((unsigned)((n_keep + kKv8Block - 1) / kKv8Block), src.Hkv, 2);
    KV8_BY_DIM(src.D, hipLaunchKernelGGL(kv8_move_kernel<kD>, grid, dim3(256), 0, st, src, dst, n_keep, kept));
    return hipGetLastError();
}
hipError_t launch_kv8_attn_rows(const Kv8Attn& a, hipStream_t st) {
    KV8_BY_DIM(a.c.D, hipLaunchKernelGGL(kv8_attn_rows_kernel<kD>, dim3(a.c.H, a.M), dim3(256), 0, st, a, kLog2e / sqrtf((float)kD)));
    return hipGetLastError();
}
hipError_t launch_kv8_attn_mass(const Kv8Attn& a, hipStream_t st) {
    const unsigned blocks = (unsigned)((a.mass_n + kKv8Block - 1) / kKv8Block);
    KV8_BY_DIM(a.c.D, hipLaunchKernelGGL(kv8_attn_mass_kernel<kD>, dim3(blocks, a.c.Hkv), dim3(256), 0, st, a, kLog2e / sqrtf((float)kD)));
    return hipGetLastError();
}

}  // namespace thk
