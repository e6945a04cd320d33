// thk_kv8.hip — kernels of the 8-bit K/V cache: append (quantise), read (dequantise), attention over the codes, eviction.
// Layout: thk_kv8.hpp.  All sums, softmax statistics and scales are f32; the codes are the only 8-bit values.
#include "thk_device.hpp"
#include "thk_kv8.hpp"
#include <algorithm>
#include <type_traits>

namespace thk {

__device__ __forceinline__ float as_f(unsigned v) { return __builtin_bit_cast(float, v); }
__device__ __forceinline__ unsigned as_u(float v) { return __builtin_bit_cast(unsigned, v); }

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

template <int D> __device__ __forceinline__ void get_codes(const int8_t* p, int (&q)[D / 16]) {
    int w[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) w[i] = reinterpret_cast<const int*>(p)[i];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) q[i] = (int)(int8_t)(w[i / 4] >> (8 * (i % 4)));
}
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
// Bound by memory: 16381 tokens on 32 heads of 128, 537 MB in and 134 MB out, 140 us, the rate of a large copy (4.8 TB/s).  A single token: the
// launch (3.5 us); all its sources are asked for before one is chosen, so that it waits for memory once.
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
    const size_t ld = (size_t)c.Hkv * D;
    const float* src = x + (p0 - pos) * (int64_t)ld + (size_t)h * D;        // row r of the block: src + r ld (the new rows only)
    if (r0 == 0 && r1 == kKv8Block) {                                      // all rows are new: no choice, all loads at once
        if (V) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) xs[i] = __builtin_nontemporal_load(src + (size_t)el_row<D, V>(0) * ld + i * ld + el_dim<D, V>(0));
        } else {
#pragma unroll
            for (int i = 0; i < D / 16; i += 4) {
                const f4 v = __builtin_nontemporal_load(reinterpret_cast<const f4*>(src + (size_t)el_row<D, V>(0) * ld + el_dim<D, V>(0) + i));
                xs[i] = v[0]; xs[i + 1] = v[1]; xs[i + 2] = v[2]; xs[i + 3] = v[3];
            }
        }
    } else {                                                               // every source is read (rows out of reach: the nearest that exists), then one is taken
        const int2 t = *at;
        const float old = *scale;
        float xn[D / 16], xt[D / 16];
        int xc[D / 16];
        get_codes<D>(codes, xc);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const int r = el_row<D, V>(i), d = el_dim<D, V>(i);
            xn[i] = src[(size_t)min(max(r, r0), r1 - 1) * ld + d];
            xt[i] = tail[r * D + d];
        }
        const int held = t.x == b ? t.y : 0;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const int r = el_row<D, V>(i);
            xs[i] = r >= r1 ? 0.f : r >= r0 ? xn[i] : r < held ? xt[i] : (float)xc[i] * old;
        }
    }
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) { const unsigned u = abs_bits(xs[i]); m = u > m ? u : m; }
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
// value = code * scale, a block per workgroup as for append.  Bound by the f32 stores: 16386 positions on 32 heads 152 us (4.4 TB/s).
template <int D, bool V>
__device__ __forceinline__ void read_body(const Kv8View& c, int64_t pos, int64_t n, float* out) {
    const int h = blockIdx.y, b = (int)(pos / kKv8Block) + blockIdx.x;
    const size_t hb = (size_t)h * c.n_blk + b;
    const int8_t* codes = (V ? c.v : c.k) + hb * (kKv8Block * D) + code_at<D, V>();
    const float s = (V ? c.vs : c.ks)[hb];
    float xs[D / 16];
    int q[D / 16];
    get_codes<D>(codes, q);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) xs[i] = (float)q[i] * s;
    const int64_t p0 = (int64_t)b * kKv8Block - pos, ld = (int64_t)c.Hkv * D;
    float* to = out + p0 * ld + (int64_t)h * D + el_dim<D, V>(0);          // row r of the block: to + r ld
    if (V) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const int r = el_row<D, V>(i);
            if (p0 + r >= 0 && p0 + r < n) to[r * ld] = xs[i];
        }
    } else if (p0 + el_row<D, V>(0) >= 0 && p0 + el_row<D, V>(0) < n) {
#pragma unroll
        for (int i = 0; i < D / 16; i += 4) *reinterpret_cast<f4*>(to + el_row<D, V>(0) * ld + i) = f4{xs[i], xs[i + 1], xs[i + 2], xs[i + 3]};
    }
}
template <int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8View c, int64_t pos, int64_t n, float* __restrict__ k_out, float* __restrict__ v_out) {
    if (blockIdx.z == 0) { if (k_out) read_body<D, false>(c, pos, n, k_out); }
    else if (v_out) read_body<D, true>(c, pos, n, v_out);
}

// ---------------------------------------------------------------- eviction
// Weights as unsigned keys, heaviest first: order-preserving, -0 = +0, NaN (the weight of a row nobody could attend) below everything but the
// 0 of a position that does not exist; the positions that stay whatever their weight have the largest.
static const unsigned kKeyStays = 0xFFFFFFFFu;
__device__ __forceinline__ unsigned mass_key(float x) {
    const unsigned b = as_u(x + 0.f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 1u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_mass(unsigned k) { return as_f(k == 1u ? 0x7FC00000u : (k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k); }
// The n_keep largest keys of a head by radix selection, ties to the lowest position, then the kept positions in ascending order.
//   W waves; thread t takes positions 4 t .. 4 t + 3 of every 256 W.
//   Histograms in LDS, in interleaved copies by lane (the weights' leading bits take few values, and copies in one bank would not help);
//   thread t sums the buckets of one stretch, heaviest first.
//   What stays is one ballot per 64 keys; the ballots' bit counts, summed up over waves, say where each thread's kept positions go.
template <int W> __device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* sm, unsigned* total) {     // exclusive prefix sum over 64 W threads; sm: W words
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const unsigned u = (unsigned)__shfl_up((int)s, o); if (lane >= o) s += u; }
    __syncthreads();
    if (lane == 63) sm[w] = s;
    __syncthreads();
    unsigned before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) { const unsigned t = sm[i]; if (i < w) before += t; all += t; }
    *total = all;
    return before + s - v;
}
struct Weights {                                                           // of one head; positions outside [lo, hi) stay, positions from end on do not exist
    const float* mass;
    int lo, hi, end;
    __device__ __forceinline__ void load4(int t, unsigned (&k)[4]) const {
        typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
        f4 v;
        if (t + 3 < end) v = *reinterpret_cast<const f4u*>(mass + t);
        else v = f4{mass[min(t, end - 1)], mass[min(t + 1, end - 1)], mass[min(t + 2, end - 1)], mass[end - 1]};
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = t + j >= end ? 0u : t + j < lo || t + j >= hi ? kKeyStays : mass_key(v[j]);
    }
};
// Of the keys that start with prefix, `same` of them, the `need` heaviest stay; the bits of all keys below prefix's are still open.
struct Pick { unsigned prefix, need, same; };
static const Pick kOnlyThose = {kKeyStays, 1u, 1u};                        // nothing but what stays in any case
// The next `bits` of the threshold from the counts of their values, thread t holding those of mask - (t PT + i).  to: 3 words
template <int W, int PT> __device__ __forceinline__ Pick pick_bits(const unsigned (&c)[PT], int bits, Pick p, unsigned* sm, unsigned* to) {
    const unsigned mask = (1u << bits) - 1;
    unsigned mine = 0, total;
#pragma unroll
    for (int i = 0; i < PT; ++i) mine += c[i];
    unsigned above = block_scan<W>(mine, sm, &total);
#pragma unroll
    for (int i = 0; i < PT; ++i) {
        if (above < p.need && p.need <= above + c[i]) { to[0] = mask - (threadIdx.x * PT + i); to[1] = p.need - above; to[2] = c[i]; }
        above += c[i];
    }
    __syncthreads();
    return Pick{(p.prefix << bits) | to[0], to[1], to[2]};
}
// The kept positions of [t0, end) in order.  each(t0, f) calls f(group, position, keys) for this thread's groups of four from t0, Q at most and none that begins behind end; cnt: Q W words
template <int W, int Q, typename Each>
__device__ __forceinline__ void place_kept(int t0, int end, Pick p, unsigned ties_before, unsigned kept_before, const float* mass, int32_t* kept, float* mass_out, unsigned* sm,
                                           unsigned* cnt, Each each) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, tid = threadIdx.x;
    // stays: heavier than the threshold, or equal to it and among the first `need` of those
    const bool all_ties = p.need == p.same;                                // then nobody's rank matters
    const unsigned long long below = (1ull << lane) - 1;
    unsigned all;
    auto place = [&](const bool (&f)[4], int (&at)[4]) {                   // places of the set flags within the wave's 256 positions, and their number
        unsigned long long b[4];
        int n = 0, base = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { b[j] = __ballot(f[j]); n += (int)__popcll(b[j]); base += (int)__popcll(b[j] & below); }
#pragma unroll
        for (int j = 0; j < 4; ++j) { at[j] = base; base += f[j]; }
        return n;
    };
    auto sum_up = [&](unsigned before, int groups) {                       // cnt -> what lies before each of its entries
        __syncthreads();
        static_assert(Q * W <= 64 * W, "one entry a thread");
        const unsigned v = block_scan<W>(tid < groups * W ? cnt[tid] : 0u, sm, &all) + before;
        if (tid < Q * W) cnt[tid] = v;
        __syncthreads();
    };
#pragma unroll 1
    for (; t0 < end; t0 += Q * 256 * W) {
        const int groups = min(Q, (end - t0 + 256 * W - 1) / (256 * W));   // those that `each` visits
        unsigned long long ties = 0;                                       // bit 4 q + j: equal to the threshold and among the first
        if (!all_ties) {
            each(t0, [&](int q, int, const unsigned (&k)[4]) {
                bool f[4]; int at[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = k[j] == p.prefix;
                const int n = place(f, at);
                if (lane == 0) cnt[q * W + w] = (unsigned)n;
            });
            sum_up(ties_before, groups);
            ties_before += all;
            each(t0, [&](int q, int, const unsigned (&k)[4]) {
                bool f[4]; int at[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = k[j] == p.prefix;
                place(f, at);
#pragma unroll
                for (int j = 0; j < 4; ++j) ties |= (unsigned long long)(f[j] && cnt[q * W + w] + (unsigned)at[j] < p.need) << (4 * q + j);
            });
            __syncthreads();
        }
        auto stays = [&](int q, const unsigned (&k)[4], bool (&f)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = all_ties ? k[j] >= p.prefix : k[j] > p.prefix || (ties >> (4 * q + j) & 1);
        };
        each(t0, [&](int q, int, const unsigned (&k)[4]) {
            bool f[4];
            stays(q, k, f);
            int n = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) n += (int)__popcll(__ballot(f[j]));
            if (lane == 0) cnt[q * W + w] = (unsigned)n;
        });
        sum_up(kept_before, groups);
        kept_before += all;
        each(t0, [&](int q, int t, const unsigned (&k)[4]) {
            bool f[4]; int at[4];
            stays(q, k, f);
            place(f, at);
            const unsigned base = cnt[q * W + w];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (f[j]) {
                    kept[base + (unsigned)at[j]] = t + j;
                    if (mass_out) mass_out[base + (unsigned)at[j]] = k[j] == kKeyStays ? mass[t + j] : key_mass(k[j]);
                }
        });
        __syncthreads();
    }
}
// One workgroup per head.  With N > 0 (T <= 64 W N) a thread's N keys stay in LDS, else every pass reads the weights again, 64 a thread at a time.
// (Registers would hold them too, but loops over them have to be unrolled, and then spill.)  Bound by one CU's instruction issue and its barriers:
// 512 positions 7 us with 4 waves and 8 bits a pass (11 bits: 9.6), 32768 with 16 waves 28 us.
template <int W, int N, int BITS>
__global__ __launch_bounds__(64 * W) void kv8_select_kernel(int T, int n_keep, int n_sink, int n_recent, const float* __restrict__ mass_in, int64_t ld_in,
                                                            float* __restrict__ mass_out, int64_t ld_out, int32_t* __restrict__ kept) {
    constexpr int Q = (N > 0 ? N : 64) / 4, R = 2, B = 1 << BITS, PT = (B + 64 * W - 1) / (64 * W);     // groups of four a thread and sweep; copies; buckets; buckets a thread
    __shared__ unsigned hist[B * R], sm[W], to[3], cnt[Q * W];
    extern __shared__ __align__(16) char smem[];
    uint4* keys = reinterpret_cast<uint4*>(smem);                          // [Q][64 W]
    const int h = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const Weights m{mass_in + (size_t)h * ld_in, n_sink, T - n_recent, T};
    if (N > 0) {                                                           // read by the thread that writes them
#pragma unroll 4
        for (int q = 0; q < min(Q, (T + 256 * W - 1) / (256 * W)); ++q) {
            unsigned k[4];
            m.load4((q * 64 * W + tid) * 4, k);
            keys[q * 64 * W + tid] = uint4{k[0], k[1], k[2], k[3]};
        }
    }
    auto each = [&](int t0, auto f) {                                      // f(group, position, keys) over the sweep from t0
        const int groups = min(Q, (T - t0 + 256 * W - 1) / (256 * W));     // nothing lies behind them
        for (int q = 0; q < groups; ++q) {
            unsigned k[4];
            const int t = t0 + (q * 64 * W + tid) * 4;
            if (N > 0) { const uint4 v = keys[q * 64 * W + tid]; k[0] = v.x; k[1] = v.y; k[2] = v.z; k[3] = v.w; }
            else m.load4(t, k);
            f(q, t, k);
        }
    };
    Pick p{0, (unsigned)(n_keep - n_sink - n_recent), 0};                  // what stays in any case is not counted
    int shift = 32;
    if (p.need == 0) { p = kOnlyThose; shift = 0; }
#pragma unroll 1
    while (shift > 0) {
        const int bits = shift < BITS ? shift : BITS, prev = shift;
        const bool first = shift == 32;
        shift -= bits;
        const unsigned mask = (1u << bits) - 1;
        for (int i = tid; i < B * R; i += 64 * W) hist[i] = 0;
        __syncthreads();
        for (int t0 = 0; t0 < T; t0 += Q * 256 * W)
            each(t0, [&](int, int, const unsigned (&k)[4]) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k[j] - 1 < kKeyStays - 1 && (first || (k[j] >> prev) == p.prefix)) atomicAdd(&hist[((k[j] >> shift) & mask) * R + lane % R], 1u);    // integers: the order changes nothing
            });
        __syncthreads();
        unsigned c[PT];
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const int d = (int)mask - (tid * PT + i);
            c[i] = 0;
            if (d >= 0) { const uint2 v = *reinterpret_cast<const uint2*>(hist + d * R); c[i] = v.x + v.y; }
        }
        p = pick_bits<W, PT>(c, bits, p, sm, to);
    }
    place_kept<W, Q>(0, T, p, 0u, 0u, m.mass, kept + (size_t)h * n_keep, mass_out ? mass_out + (size_t)h * ld_out : nullptr, sm, cnt, each);
}
// Long sets on few heads: a head's positions are cut into gridDim.x slices, a workgroup each, and a launch for each of the threshold's three parts
// (11, 11 and 10 bits) leaves the slices' counts for the next one, where every workgroup adds them up; the fourth places what stays.
//   count  [3][heads][slices][2048]   of the part's values, heaviest first
//   above  [2][heads][slices]         a slice's keys above the first (second) part of the threshold
//   picks  [2][heads][4]              the threshold after the first (second) part
struct Slices { unsigned *count, *above, *picks; };
template <int PART>
__global__ __launch_bounds__(1024) void kv8_select_slice_kernel(int T, int slice, int n_keep, int n_sink, int n_recent, const float* __restrict__ mass_in, int64_t ld_in,
                                                                float* __restrict__ mass_out, int64_t ld_out, int32_t* __restrict__ kept, Slices s) {
    constexpr int W = 16, Q = 2, R = 4;
    constexpr int shift = PART == 0 ? 21 : PART == 1 ? 10 : 0, bits = PART < 2 ? 11 : 10, known = PART == 0 ? 0 : shift + bits, prev_bits = PART == 3 ? 10 : 11;
    __shared__ unsigned hist[PART < 3 ? 2048 * R : 1], sm[W], to[3], tied, cnt[Q * W];
    const int h = blockIdx.y, id = blockIdx.x, n = gridDim.x, tid = threadIdx.x, lane = tid & 63, heads = gridDim.y;
    const int t0 = min(id * slice, T), end = min(t0 + slice, T);
    const Weights m{mass_in + (size_t)h * ld_in, n_sink, T - n_recent, end};
    auto each = [&](int t0, auto f) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            unsigned k[4];
            const int t = t0 + (q * 64 * W + tid) * 4;
            if (t0 + q * 256 * W >= end) break;
            m.load4(t, k);
            f(q, t, k);
        }
    };
    Pick p{0, (unsigned)(n_keep - n_sink - n_recent), 0};
    unsigned kept_before = 0, ties_before = 0;
    const bool only_those = p.need == 0;
    if (only_those) {
        if (PART < 3) return;
        p = kOnlyThose;
    } else if (PART > 0) {                                                        // the previous part: thread t has its values 2 t and 2 t + 1, heaviest first
        const uint2* c = reinterpret_cast<const uint2*>(s.count + ((size_t)(PART - 1) * heads + h) * n * 2048) + tid;
        unsigned all[2] = {0, 0}, early[2] = {0, 0}, mine[2] = {0, 0};     // of all slices, of those before this one, of this one
        for (int i = 0; i < n; ++i) {
            const uint2 v = c[(size_t)i * 1024];
            all[0] += v.x; all[1] += v.y;
            if (i < id) { early[0] += v.x; early[1] += v.y; }
            if (i == id) { mine[0] = v.x; mine[1] = v.y; }
        }
        if (PART > 1) { const unsigned* q = s.picks + ((size_t)(PART - 2) * heads + h) * 4; p = Pick{q[0], q[1], q[2]}; }
        p = pick_bits<W, 2>(all, prev_bits, p, sm, to);
        const unsigned at = ((1u << prev_bits) - 1) - (p.prefix & ((1u << prev_bits) - 1));    // the place of the threshold's value
        auto heavier = [&](const unsigned (&v)[2]) { return (2u * tid < at ? v[0] : 0u) + (2u * tid + 1 < at ? v[1] : 0u); };
        if (PART < 3) {
            unsigned above;
            (void)block_scan<W>(heavier(mine), sm, &above);
            if (tid == 0) {
                s.above[((size_t)(PART - 1) * heads + h) * n + id] = above;
                if (id == 0) { unsigned* q = s.picks + ((size_t)(PART - 1) * heads + h) * 4; q[0] = p.prefix; q[1] = p.need; q[2] = p.same; }
            }
        } else {
            unsigned x = heavier(early);
            for (int i = tid; i < id; i += 1024) x += s.above[(size_t)h * n + i] + s.above[((size_t)heads + h) * n + i];
            (void)block_scan<W>(x, sm, &kept_before);
            if (2u * tid == (at & ~1u)) tied = early[at & 1];
            __syncthreads();
            ties_before = tied;
            kept_before += min(ties_before, p.need);
        }
    }
    kept_before += (unsigned)(min(t0, m.lo) + max(t0 - m.hi, 0));          // stay in any case, before this slice
    if (PART < 3) {
        for (int i = tid; i < 2048 * R / 4; i += 1024) reinterpret_cast<uint4*>(hist)[i] = uint4{0, 0, 0, 0};
        __syncthreads();
        for (int t = t0; t < end; t += Q * 256 * W)
            each(t, [&](int, int t, const unsigned (&k)[4]) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k[j] - 1 < kKeyStays - 1 && (PART == 0 || (k[j] >> known) == p.prefix)) atomicAdd(&hist[((k[j] >> shift) & ((1u << bits) - 1)) * R + lane % R], 1u);
            });
        __syncthreads();
        unsigned c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = (1 << bits) - 1 - (2 * tid + i);
            const uint4 v = reinterpret_cast<const uint4*>(hist)[max(d, 0)];
            c[i] = d >= 0 ? v.x + v.y + v.z + v.w : 0u;
        }
        reinterpret_cast<uint2*>(s.count + (((size_t)PART * heads + h) * n + id) * 2048)[tid] = uint2{c[0], c[1]};
    } else
        place_kept<W, Q>(t0, end, p, ties_before, kept_before, m.mass, kept + (size_t)h * n_keep, mass_out ? mass_out + (size_t)h * ld_out : nullptr, sm, cnt, each);
}
// One workgroup per destination block, head and K | V: gathers the 16 kept rows as values and quantises them anew.  Sixteen rows that were
// one block stay as they are (codes and scale), so that what eviction leaves in place does not drift.  A V row is a byte of every 16 (the layout
// attention wants), so sparse selections read all of V: 4099 of 32768 positions on 32 heads, 134 MB of V and 51 MB else, 47 us.
template <int D, bool V>
__device__ __forceinline__ void move_body(const Kv8View& s, const Kv8View& d, int n_keep, const int32_t* kept, unsigned* sm, int* src) {
    const int h = blockIdx.y, b = blockIdx.x, rows = n_keep - b * kKv8Block < kKv8Block ? n_keep - b * kKv8Block : kKv8Block;
    if (threadIdx.x < kKv8Block) src[threadIdx.x] = (int)threadIdx.x < rows ? kept[(size_t)h * n_keep + b * kKv8Block + threadIdx.x] : -1;
    __syncthreads();
    const bool whole = src[0] % kKv8Block == 0 && src[15] == src[0] + 15;
    const int8_t* from = (V ? s.v : s.k) + (size_t)h * s.n_blk * (kKv8Block * D);
    const float* sc = (V ? s.vs : s.ks) + (size_t)h * s.n_blk;
    const size_t hb = (size_t)h * d.n_blk + b;
    float xs[D / 16], sc_[D / 16];
    unsigned q[D / 16], m = 0;
    int code[D / 16];
    if (V) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {                                 // rows behind the last kept one read position 0: all loads at once
            const int p = max(src[el_row<D, V>(i)], 0);
            code[i] = from[((size_t)(p >> 4) * D + el_dim<D, V>(0)) * 16 + (p & 15)];
            sc_[i] = sc[p >> 4];
        }
    } else {
        const int p = max(src[el_row<D, V>(0)], 0);
        get_codes<D>(from + (size_t)p * D + el_dim<D, V>(0), code);
        const float s0 = sc[p >> 4];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) sc_[i] = s0;
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const bool in = src[el_row<D, V>(i)] >= 0;
        q[i] = in ? (unsigned)code[i] & 0xFFu : 0u;
        xs[i] = in ? (float)code[i] * sc_[i] : 0.f;
        const unsigned u = abs_bits(xs[i]);
        m = u > m ? u : m;
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

static const float kLog2e = 1.44269504088896340736f;      // scores carry log2(e): the weights are exp2

// a * b rounded to f32, whatever it goes to: a score has to be the same number where it is compared and where the maximum is taken from it.
// Fused into the difference, the largest one's weight would be 2^(half a step of the maximum) and not 1.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// ---------------------------------------------------------------- attention of few rows: i8 matrix instructions, split over the positions
// out_n = sum_t p_nt v_t with p = softmax(q_n . k_t), for up to 16 (row, head) columns n that read one K/V head.  Both products run on
// v_mfma_i32_16x16x64_i8 with the cache's codes as they are - no conversion - and the f32 operand (q, then the weights) as a fixed-point
// number of three balanced base-256 digits: x = d2 2^16 + d1 2^8 + d0, each digit an i8 operand of its own product, the three i32 sums
// exact.  q is fixed relative to its column's largest entry (23 bits with the sign), the weights p * v_scale relative to the largest of their column
// in the tile of 64 positions (a power of two, 21 to 22 bits).  Both lie above f32's own rounding, which short sums show (64 positions 6.7e-7 from the
// 64-bit result in norm, elementary f32 operations 3.5e-7); over 2047 positions the two are alike, over 65535 the fewer f32 additions count (8.7e-7, 2.2e-6).
// Operand layout (A: row = lane % 16, B: column = lane % 16, both 16 consecutive k per lane of chunk lane / 16; result: column lane % 16,
// rows 4 (lane / 16) + i).  The k order is free as long as A and B share it, and the row order of the first product is chosen so that
// lane chunk c ends up with the scores of the 16 positions of block c: then one K scale and one V scale per lane serve a whole tile, and
// the second product's B operand is what the lane already holds - no exchange between lanes.
// Long caches are bound by memory: 65535 positions on 32 heads, 537 MB in 89 us (6.0 TB/s; the bare reads in this pattern reach 6.9), 131071 on 8
// heads for 64 query heads 47 us with the joining launch.  Short ones are a chain of latencies (launch, load, one tile, join of the waves, from 513
// positions on join of the parts): 64 positions 4.4 us, 512 on 32 heads with weights 8.0 us (one part, 32 workgroups: 224 CUs have nothing to do),
// 2047 on 40 heads 9.7 us.
typedef int i4 __attribute__((ext_vector_type(4)));
struct U2 { unsigned a, b; };
// Between them, a and b hold a value and that of the lane 16 (32) away, in every lane.  The swap works on two registers: the empty asm keeps
// the compiler from giving it the same one twice, which would leave the value where it is.
__device__ __forceinline__ U2 pair16(unsigned v) {
    unsigned w = v;
    asm("" : "+v"(w));
    const auto r = __builtin_amdgcn_permlane16_swap(v, w, false, false);
    return {r[0], r[1]};
}
__device__ __forceinline__ U2 pair32(unsigned v) {
    unsigned w = v;
    asm("" : "+v"(w));
    const auto r = __builtin_amdgcn_permlane32_swap(v, w, false, false);
    return {r[0], r[1]};
}
// over the four lanes of a column
__device__ __forceinline__ float chunks_max(float v) {
    U2 r = pair16(as_u(v));
    r = pair32(as_u(fmaxf(as_f(r.a), as_f(r.b))));
    return fmaxf(as_f(r.a), as_f(r.b));
}
__device__ __forceinline__ unsigned chunks_max_bits(unsigned v) {
    U2 r = pair16(v);
    r = pair32(r.a > r.b ? r.a : r.b);
    return r.a > r.b ? r.a : r.b;
}
__device__ __forceinline__ float chunks_sum(float v) {
    U2 r = pair16(as_u(v));
    r = pair32(as_u(as_f(r.a) + as_f(r.b)));
    return as_f(r.a) + as_f(r.b);
}
// Four numbers x + 0x8080, with SIGNED x + 0x408080, |x| < 0x3F7F80: their digits, four to a word.
template <bool SIGNED>
__device__ __forceinline__ void pack_digits(unsigned e0, unsigned e1, unsigned e2, unsigned e3, int& d2, int& d1, int& d0) {
    const unsigned a = __builtin_amdgcn_perm(e1, e0, 0x05040100u), b = __builtin_amdgcn_perm(e3, e2, 0x05040100u);     // bytes: e0.0 e0.1 e1.0 e1.1
    const unsigned u = __builtin_amdgcn_perm(e1, e0, 0x0C0C0602u), w = __builtin_amdgcn_perm(e3, e2, 0x06020C0Cu);
    d0 = (int)(__builtin_amdgcn_perm(b, a, 0x06040200u) ^ 0x80808080u);
    d1 = (int)(__builtin_amdgcn_perm(b, a, 0x07050301u) ^ 0x80808080u);
    d2 = (int)(u | w);
    if (SIGNED) { const unsigned t = (u | w) ^ 0x40404040u; d2 = (int)(t | (t & 0x40404040u) << 1); }      // bytes 0 .. 127, less 64
}
__device__ __forceinline__ float join_digits(int i2, int i1, int i0) { return fmaf((float)i2, 65536.f, (float)(i1 * 256 + i0)); }   // |i1| <= 256 * 2^14: no overflow

// q of a column as a B operand wants it: x[4 kc + i] are dimensions 64 kc + 16 (lane / 16) + 4 i + 0 .. 3 (q points to the chunk's first)
template <int D>
__device__ __forceinline__ void load_q(const float* q, bool valid, f4 (&x)[D / 16]) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) x[i] = valid ? reinterpret_cast<const f4*>(q)[(i / 4) * 16 + i % 4] : f4{0.f, 0.f, 0.f, 0.f};
}
// Digits of 4 N numbers of a lane as fixed point relative to the largest of their column, as put(word, d2, d1, d0); returns its step.  One fma makes a
// digit triple: 22 bits and the sign, half a step is 2^-23 of the largest entry (a step more cost three instructions each, 9 % of the weight count).
template <int N, typename Max, typename Put>
__device__ __forceinline__ float digits_of(const f4 (&x)[N], Max column_max, Put put) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) { const unsigned a = abs_bits(x[i][j]); m = a > m ? a : m; }
    m = column_max(m);
    const float amax = as_f(m);
    const bool some = amax >= 0x1p-100f;                                   // also false for NaN
    const float inv = some && m < 0x7F800000u ? 4161000.f / amax : 0.f;    // x + 2^22 + 0x8080 is the mantissa of the sum below: it has to stay under 2^23
#pragma unroll
    for (int i = 0; i < N; ++i) {
        unsigned e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = as_u(fmaf(x[i][j], inv, 12615808.f));
        int d2, d1, d0;
        pack_digits<true>(e[0], e[1], e[2], e[3], d2, d1, d0);
        put(i, d2, d1, d0);
    }
    if (m >= 0x7F800000u) return as_f(0x7FC00000u);                        // a query that is not finite: every score is NaN
    return some ? amax / 4161000.f : 0.f;
}
template <int D>
__device__ __forceinline__ float q_digits(const f4 (&x)[D / 16], i4 (&qd)[3][D / 64]) {
    return digits_of<D / 16>(x, chunks_max_bits, [&](int i, int d2, int d1, int d0) { qd[2][i / 4][i % 4] = d2; qd[1][i / 4][i % 4] = d1; qd[0][i / 4][i % 4] = d0; });
}
template <int CTRL> __device__ __forceinline__ unsigned dpp_max(unsigned v) {
    const unsigned u = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
    return u > v ? u : v;
}
template <int L> __device__ __forceinline__ unsigned row_max_bits(unsigned v) {      // over aligned groups of L = 16, 32 or 64 lanes
    v = dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(v))));
    if (L >= 32) { const U2 r = pair16(v); v = r.a > r.b ? r.a : r.b; }
    if (L >= 64) { const U2 r = pair32(v); v = r.a > r.b ? r.a : r.b; }
    return v;
}
// What one workgroup leaves for another inside a launch is written and read past the XCDs' own L2s (agent scope).
__device__ __forceinline__ void put2(float* p, float x, float y) { st_agent_u64(reinterpret_cast<unsigned long long*>(p), (unsigned long long)as_u(y) << 32 | as_u(x)); }
__device__ __forceinline__ float2 get2(const float* p) { const unsigned long long v = ld_agent_u64(reinterpret_cast<const unsigned long long*>(p)); return {as_f((unsigned)v), as_f((unsigned)(v >> 32))}; }

template <bool NT> __device__ __forceinline__ i4 load16(const void* p) {
    if (NT) return __builtin_nontemporal_load(reinterpret_cast<const i4*>(p));
    return *reinterpret_cast<const i4*>(p);
}
// W waves, a tile each in turn.  NT: codes that will not be read again soon (many more than the caches hold) go past them.
template <int D, int W, bool NT>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void kv8_attn_split_kernel(Kv8Attn a, Kv8Split sp, float scale) {
    constexpr int KC = D / 64, NG = D / 16;
    __shared__ float so[W][16][D + 4], sml[W][16][2], fin[2][16];     // fin: maximum and 1 / sum of the columns, once they are final
    __shared__ int last;
    const Kv8View& c = a.c;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 15, ch = lane >> 4;
    const int split = blockIdx.x, hkv = blockIdx.y, col = blockIdx.z * 16 + n, G = c.H / c.Hkv, cols = a.M * G;
    const bool valid = col < cols, one = a.M == 1;                   // one row: no division (a launch of a single token is short enough to feel them)
    const int row = one ? 0 : col / G, last_row = one ? 0 : min((int)blockIdx.z * 16 + 15, cols - 1) / G;
    const int T = a.n_past + last_row + 1, first_lim = one ? a.n_past : a.n_past + (int)blockIdx.z * 16 / G, lim = valid ? a.n_past + row : T - 1;   // positions <= lim are seen
    const int tiles = (T + kKv8Tile - 1) / kKv8Tile, per = (tiles + sp.n - 1) / sp.n, t1 = min((split + 1) * per, tiles);
    const size_t orow = valid ? (size_t)row * c.H + hkv * G + (col - row * G) : 0;
    auto out_row = [&](int cc) { const int i = one ? 0 : cc / G; return (size_t)i * c.H + hkv * G + (cc - i * G); };

    // q's digits, by all threads together (a wave alone would spend as long on one column as on sixteen): a thread has four dimensions
    constexpr int QL = D / 4 + 4;                                    // words of a column in LDS, padded against bank conflicts
    __shared__ unsigned sq[3][16][QL];
    __shared__ float sqf[16];
    const int nv = min(cols - (int)blockIdx.z * 16, 16);
    constexpr int QN = (16 * (D / 4) + 64 * W - 1) / (64 * W);
    f4 qx[QN];
#pragma unroll
    for (int k = 0; k < QN; ++k) {
        const int j = threadIdx.x + k * 64 * W;
        if (j < nv * (D / 4)) qx[k] = reinterpret_cast<const f4*>(a.q + out_row(blockIdx.z * 16 + j / (D / 4)) * D)[j % (D / 4)];
    }
    const int8_t* kb = c.k + ((size_t)hkv * c.n_blk * kKv8Block + 16 * (n >> 2) + (n & 3)) * D + ch * 16;
    const int8_t* vb = c.v + (((size_t)hkv * c.n_blk + ch) * D + n) * 16;
    const float *ksb = c.ks + (size_t)hkv * c.n_blk + ch, *vsb = c.vs + (size_t)hkv * c.n_blk + ch;
    i4 kr[4][KC], vr[NG];
    float ks = 0.f, vs = 0.f;
    auto load_k = [&](int t) {
        const int8_t* p = kb + (size_t)t * (kKv8Tile * D);
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) kr[g][kc] = load16<NT>(p + (4 * g) * D + kc * 64);
        ks = ksb[(size_t)t * 4];
    };
    auto load_v = [&](int t) {
        const int8_t* p = vb + (size_t)t * (kKv8Tile * D);
#pragma unroll
        for (int g = 0; g < NG; ++g) vr[g] = load16<NT>(p + g * 256);
        vs = vsb[(size_t)t * 4];
    };
    int t = split * per + w;
    if (t < t1) { load_k(t); load_v(t); }
#pragma unroll
    for (int k = 0; k < QN; ++k) {
        const int j = threadIdx.x + k * 64 * W, cn = j / (D / 4);
        if (j < nv * (D / 4)) {
            const f4 x[1] = {qx[k]};
            const float step = digits_of<1>(x, row_max_bits<D / 4>, [&](int, int d2, int d1, int d0) { sq[2][cn][j % (D / 4)] = d2; sq[1][cn][j % (D / 4)] = d1; sq[0][cn][j % (D / 4)] = d0; });
            if (j % (D / 4) == 0) sqf[cn] = step * scale;
        }
    }
    __syncthreads();
    i4 qd[3][KC];                                                    // columns behind the last: whatever is there, times 0
#pragma unroll
    for (int d = 0; d < 3; ++d)
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) qd[d][kc] = *reinterpret_cast<const i4*>(&sq[d][n][16 * kc + 4 * ch]);
    const float qf = valid ? sqf[n] : 0.f;
    float m = -INFINITY, l = 0.f;
    f4 o[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) o[g] = f4{0.f, 0.f, 0.f, 0.f};
    // One tile; `more` is a constant in each of its two uses: with a branch around the loads the compiler would wait for all of them wherever it
    // waits for any.
    auto step = [&](auto more) {
        float s[16];
        const float kf = qf * ks;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            i4 acc[3];
#pragma unroll
            for (int d = 0; d < 3; ++d) {
                acc[d] = i4{0, 0, 0, 0};
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[g][kc], qd[d][kc], acc[d], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * g + i] = rounded_product(join_digits(acc[2][i], acc[1][i], acc[0][i]), kf);
            if (g & 1) __builtin_amdgcn_sched_barrier(0);            // two groups in flight: more only cost registers
        }
        if (decltype(more)::value) load_k(t + W);
        const int pos = t * kKv8Tile + ch * 16;
        if (t * kKv8Tile + kKv8Tile - 1 > first_lim) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = pos + i <= lim ? s[i] : -INFINITY;
        }
        if (sp.scores && valid) {
            float* ps = sp.scores + orow * sp.scores_ld + pos;
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                if (sp.counters) { put2(ps + i, s[i], s[i + 1]); put2(ps + i + 2, s[i + 2], s[i + 3]); }     // read in this launch
                else *reinterpret_cast<f4*>(ps + i) = f4{s[i], s[i + 1], s[i + 2], s[i + 3]};
            }
        }
        float sm = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) sm = fmaxf(sm, s[i]);
        const float mn = fmaxf(m, chunks_max(sm)), mu = mn == -INFINITY ? 0.f : mn;
        if (__any(mn != m)) {                                        // a new maximum in some column: rare after the first tiles
            const float al = __builtin_amdgcn_exp2f(m - mu);
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[g][i] *= al;
            l *= al;
            m = mn;
        }
        float ls = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) { s[i] = __builtin_amdgcn_exp2f(s[i] - mu); ls += s[i]; }
        l += ls;
        // weights p * vs in steps of 2^(e - 22), e the exponent of the tile's largest: whole numbers below 2^22.  Blocks no row of this
        // column sees (p = 0 throughout) must not bring in their scale, which may be NaN.  For e p counts as 2^-106 at least: vs in these steps stays finite.
        const float vsu = pos <= lim ? vs : 0.f;
        const float wm = as_f(chunks_max_bits(as_u(fmaxf(__builtin_amdgcn_exp2f(sm - mu), 0x1p-106f) * vsu)));
        const int e = __builtin_amdgcn_frexp_expf(wm);
        const float fac = ldexpf(vsu, 22 - e), f = ldexpf(1.f, e - 22) + (wm - wm);                  // wm - wm: 0, or NaN if wm is not finite
        i4 pd[3];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            unsigned x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = as_u(fmaf(s[4 * g + i], fac, 8421504.f));             // 2^23 + 0x8080: the mantissa is x + 0x8080
            int d2, d1, d0;
            pack_digits<false>(x[0], x[1], x[2], x[3], d2, d1, d0);
            pd[2][g] = d2; pd[1][g] = d1; pd[0][g] = d0;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const i4 z = i4{0, 0, 0, 0};
            const i4 a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(vr[g], pd[2], z, 0, 0, 0);
            const i4 a1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(vr[g], pd[1], z, 0, 0, 0);
            const i4 a0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(vr[g], pd[0], z, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[g][i] = fmaf(f, join_digits(a2[i], a1[i], a0[i]), o[g][i]);
            if (g & 1) __builtin_amdgcn_sched_barrier(0);
        }
        if (decltype(more)::value) load_v(t + W);
    };
    for (; t + W < t1; t += W) step(std::true_type{});
    if (t < t1) step(std::false_type{});
    l = chunks_sum(l);
    // join the waves: columns n, dimensions 16 g + 4 ch + i
    if (valid) {
#pragma unroll
        for (int g = 0; g < NG; ++g) *reinterpret_cast<f4*>(&so[w][n][16 * g + 4 * ch]) = o[g];
        if (ch == 0) { sml[w][n][0] = m; sml[w][n][1] = l; }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < nv * (D / 4); j += 64 * W) {
        const int cn = j / (D / 4), d = (j % (D / 4)) * 4, cc = blockIdx.z * 16 + cn;
        const size_t r = out_row(cc);
        float mm = sml[0][cn][0];
#pragma unroll
        for (int i = 1; i < W; ++i) mm = fmaxf(mm, sml[i][cn][0]);
        const float mu = mm == -INFINITY ? 0.f : mm;
        f4 sum = f4{0.f, 0.f, 0.f, 0.f};
        float ll = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float e = __builtin_amdgcn_exp2f(sml[i][cn][0] - mu);
            const f4 v = *reinterpret_cast<const f4*>(&so[i][cn][d]);
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] = fmaf(v[k], e, sum[k]);
            ll = fmaf(sml[i][cn][1], e, ll);
        }
        if (sp.n == 1) {
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] = sum[k] / ll;
            *reinterpret_cast<f4*>(a.out + r * D + d) = sum;
        } else if (!sp.counters) {
            *reinterpret_cast<f4*>(sp.part_o + (r * sp.n + split) * D + d) = sum;
        } else {
            float* po = sp.part_o + (r * sp.n + split) * D + d;
            put2(po, sum[0], sum[1]); put2(po + 2, sum[2], sum[3]);
        }
        if (d == 0) {
            if (sp.n == 1) {
                fin[0][cn] = mm; fin[1][cn] = 1.f / ll;
                if (a.ml) a.ml[r] = float2{mm, ll};
            } else put2(reinterpret_cast<float*>(sp.part_ml + r * sp.n + split), mm, ll);
        }
    }
    if (!sp.counters) return;
    // The workgroup that finishes last for its columns joins the splits (in their order, whoever comes last) and counts the weights.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                 // this thread's parts and scores are where the others can see them
    __syncthreads();
    if (sp.n > 1) {
        unsigned* counter = sp.counters + blockIdx.z * gridDim.y + hkv;
        if (threadIdx.x == 0) last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)sp.n - 1;
        __syncthreads();
        if (!last) return;
        if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);    // as the next launch expects it
    }
    // everything the first round of either loop needs is asked for before anything is waited for
    const int tw = threadIdx.x * 2;
    const bool early = sp.scores && nv == 1 && tw < a.mass_n;
    float2 s0 = {0.f, 0.f}, in0 = {0.f, 0.f};
    if (early) {
        s0 = get2(sp.scores + (size_t)(hkv * G) * sp.scores_ld + tw);
        in0 = {a.mass_in[(size_t)hkv * a.mass_ld + tw], a.mass_in[(size_t)hkv * a.mass_ld + min(tw + 1, a.mass_n - 1)]};
    }
    if (sp.n > 1) {
        for (int j = threadIdx.x; j < nv * (D / 2); j += 64 * W) {
            const int cn = j / (D / 2), d = (j % (D / 2)) * 2;
            const size_t r = out_row(blockIdx.z * 16 + cn);
            const float* po = sp.part_o + r * sp.n * D + d;
            const float* pm = reinterpret_cast<const float*>(sp.part_ml + r * sp.n);
            float mm = -INFINITY, ll = 0.f, x = 0.f, y = 0.f;
            for (int i0 = 0; i0 < sp.n; i0 += 8) {
                float2 v[8], ml[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) { const int k = min(i0 + i, sp.n - 1); ml[i] = get2(pm + 2 * k); v[i] = get2(po + (size_t)k * D); }
                float mn = mm;
#pragma unroll
                for (int i = 0; i < 8; ++i) mn = fmaxf(mn, ml[i].x);
                const float mu = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(mm - mu);
                x *= al; y *= al; ll *= al; mm = mn;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i0 + i < sp.n) {
                        const float e = __builtin_amdgcn_exp2f(ml[i].x - mu);
                        x = fmaf(v[i].x, e, x); y = fmaf(v[i].y, e, y); ll = fmaf(ml[i].y, e, ll);
                    }
            }
            *reinterpret_cast<float2*>(a.out + r * D + d) = float2{x / ll, y / ll};
            if (d == 0) { fin[0][cn] = mm; fin[1][cn] = 1.f / ll; if (a.ml) a.ml[r] = float2{mm, ll}; }
        }
        __syncthreads();
    }
    if (sp.scores)                                                   // one row: columns are the heads of the group
        for (int t2 = tw; t2 < a.mass_n; t2 += 128 * W) {
            const bool have = early && t2 == tw;
            const size_t at = (size_t)hkv * a.mass_ld + t2;
            float x = 0.f, y = 0.f;
            for (int g = 0; g < nv; ++g) {
                const float2 s = have ? s0 : get2(sp.scores + (size_t)(hkv * G + g) * sp.scores_ld + t2);
                x = fmaf(__builtin_amdgcn_exp2f(s.x - fin[0][g]), fin[1][g], x); y = fmaf(__builtin_amdgcn_exp2f(s.y - fin[0][g]), fin[1][g], y);
            }
            a.mass_out[at] = (have ? in0.x : a.mass_in[at]) + x;
            if (t2 + 1 < a.mass_n) a.mass_out[at + 1] = (have ? in0.y : a.mass_in[at + 1]) + y;
        }
}
// After a split that was not joined inside its launch.  The first M H workgroups join a row and head each: 256 / (D / 4) groups of threads take
// the splits in turn.  The others (one row, scores left behind) count the weights: 512 positions of a K/V head each, with maxima and sums of
// the group's heads from their parts, so that they need not wait for the join.  8 MB of scores and 8 MB of weights twice (65535 positions, 32
// heads): 9 us.
template <int D>
__global__ __launch_bounds__(256) void kv8_attn_finish_kernel(Kv8Attn a, Kv8Split sp) {
    constexpr int R = 256 / (D / 4);
    __shared__ f4 part[R][D / 4];
    __shared__ float fin[2][16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    auto stats = [&](size_t r, float& e) {                           // the row's maximum and sum; e: this lane's split's share
        const float2 ml = lane < sp.n ? sp.part_ml[r * sp.n + lane] : float2{-INFINITY, 0.f};
        const float m = wave_max(ml.x);
        e = __builtin_amdgcn_exp2f(ml.x - (m == -INFINITY ? 0.f : m));
        return float2{m, wave_sum(lane < sp.n ? ml.y * e : 0.f)};
    };
    if (blockIdx.x < (unsigned)(a.M * a.c.H)) {
        const size_t r = blockIdx.x;
        const int d = threadIdx.x % (D / 4), g = threadIdx.x / (D / 4);
        float e;
        const float2 ml = stats(r, e);
        f4 sum = f4{0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 < sp.n; i0 += R) {                           // all lanes in every round: a lane that has left can give nobody its share
            const int i = i0 + g;
            const float ei = __shfl(e, min(i, 63));
            if (i >= sp.n) continue;
            const f4 v = reinterpret_cast<const f4*>(sp.part_o + (r * sp.n + i) * D)[d];
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] = fmaf(v[k], ei, sum[k]);
        }
        part[g][d] = sum;
        __syncthreads();
        if (threadIdx.x < D / 4) {
            sum = part[0][d];
#pragma unroll
            for (int i = 1; i < R; ++i) sum += part[i][d];
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] = sum[k] / ml.y;
            reinterpret_cast<f4*>(a.out + r * D)[d] = sum;
        }
        if (threadIdx.x == 0 && a.ml) a.ml[r] = ml;
        return;
    }
    const int chunks = (a.mass_n + 511) / 512, b = blockIdx.x - a.M * a.c.H, hkv = b / chunks, t = (b % chunks) * 512 + threadIdx.x * 2, G = a.c.H / a.c.Hkv;
    float2 s[4];
    auto load = [&](int g0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = *reinterpret_cast<const float2*>(sp.scores + (size_t)(hkv * G + min(g0 + i, G - 1)) * sp.scores_ld + t);
    };
    if (t < a.mass_n) load(0);
    for (int g = w; g < G; g += 4) {
        float e;
        const float2 ml = stats((size_t)hkv * G + g, e);
        if (lane == 0) { fin[0][g] = ml.x; fin[1][g] = 1.f / ml.y; }
    }
    __syncthreads();
    if (t >= a.mass_n) return;
    const size_t at = (size_t)hkv * a.mass_ld + t;
    const float in0 = a.mass_in[at], in1 = a.mass_in[(size_t)hkv * a.mass_ld + min(t + 1, a.mass_n - 1)];
    float x = 0.f, y = 0.f;
    for (int g0 = 0; g0 < G; g0 += 4) {
        if (g0 > 0) load(g0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (g0 + i < G) {
                x = fmaf(__builtin_amdgcn_exp2f(s[i].x - fin[0][g0 + i]), fin[1][g0 + i], x);
                y = fmaf(__builtin_amdgcn_exp2f(s[i].y - fin[0][g0 + i]), fin[1][g0 + i], y);
            }
    }
    a.mass_out[at] = in0 + x;
    if (t + 1 < a.mass_n) a.mass_out[at + 1] = in1 + y;
}

// ---------------------------------------------------------------- attention of many rows: f16 matrix instructions, tiles shared through LDS
// Many rows make the products the bound, and the digits' i32 sums would have to be joined for every tile; here the f32 operand is two f16
// parts (hi + lo: 22 bits) on v_mfma_f32_16x16x32_f16 and the sums stay in f32 accumulators.  The codes become f16 exactly, once per workgroup
// and tile, on their way into LDS.  A workgroup of 4 waves takes 64 NC columns (row, head of the group), each wave 16 NC of them.
//   q       scaled by a power of two per column so that its largest entry is in [2^14, 2^15): both parts stay far from f16's ends
//   weights p * v_scale in units of 2^(ref - 15), ref >= the exponent of the largest weight the column has met (relative to its running
//           maximum): at most 2^15, and what the lo part cannot hold is below 2^-40 of that largest weight.  The accumulators are rescaled
//           only where the running maximum or ref moves, which a wave skips when none of its columns did.  For ref p counts
//           as 2^-113 at least, so that v_scale * 2^(15 - ref) is finite: what the lo part then loses, 2^-151 of the scale, f32's own p does not hold.
// Bound by the matrix instructions and, beside them, the softmax's vector ones (on f16 the two do not overlap): 2048 rows over 6144 positions, 32
// heads on 8, 424 - 430 us, 481 GFLOP of f16 products (the f32 work twice) at 1.13 PFLOP/s; a large f16 matrix product reaches 1.16.
// S = 2: a second group of four waves takes every other tile, and its sums join the first's through LDS: 512 rows on 32 heads 18.8 -> 16.2 us.
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef _Float16 hf2 __attribute__((ext_vector_type(2)));
struct HF8x2 { hf8 a, b; };
// 16 codes -> 16 f16: byte + 128 behind 0x64 is 1024 + byte + 128 exactly, less 1152
__device__ __forceinline__ HF8x2 codes_f16(i4 q) {
    unsigned o[8];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const unsigned u = (unsigned)q[w] ^ 0x80808080u;
        o[2 * w] = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
        o[2 * w + 1] = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(hf2, o[i]) - hf2{(_Float16)1152.f, (_Float16)1152.f});
    HF8x2 r;
    const uint4 lo = {o[0], o[1], o[2], o[3]}, hi = {o[4], o[5], o[6], o[7]};
    r.a = __builtin_bit_cast(hf8, lo); r.b = __builtin_bit_cast(hf8, hi);
    return r;
}
// hi and lo parts of x[i] * f: hi the product cut to 11 bits, lo the rest of the exact product, rounded: together good to 2^-22 of it
__device__ __forceinline__ void split_f16(const float* x, float f, hf8& hi, hf8& lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const hf2 h = __builtin_bit_cast(hf2, __builtin_amdgcn_cvt_pkrtz(x[i] * f, x[i + 1] * f));
        hi[i] = h[0]; hi[i + 1] = h[1];
        lo[i] = (_Float16)fmaf(x[i], f, -(float)h[0]); lo[i + 1] = (_Float16)fmaf(x[i + 1], f, -(float)h[1]);
    }
}
// The B operand of q for one column: parts of dimensions 64 (st / 2) + 16 (lane / 16) + 8 (st % 2) + j, st = 0 .. D/32 - 1.  Returns 1 / the power of two.
template <int D>
__device__ __forceinline__ float q_f16(const f4 (&x)[D / 16], hf8 (&hi)[D / 32], hf8 (&lo)[D / 32]) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) { const unsigned u = abs_bits(x[i][j]); m = u > m ? u : m; }
    m = chunks_max_bits(m);
    const float amax = as_f(m);
    const bool fine = amax >= 0x1p-100f && m < 0x7F800000u;
    const int e = fine ? __builtin_amdgcn_frexp_expf(amax) : 15;
    const float up = fine ? ldexpf(1.f, 15 - e) : 0.f;
#pragma unroll
    for (int st = 0; st < D / 32; ++st) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = fine ? x[2 * st + j / 4][j % 4] : 0.f;
        split_f16(y, up, hi[st], lo[st]);
    }
    return m >= 0x7F800000u ? as_f(0x7FC00000u) : ldexpf(1.f, e - 15);
}
// What turns the f16 sums of q and codes into scores.  Zero times a masked -inf would be NaN, so products below 2^-126 count as that: the sums
// are below 2^30, a score moves by 2^-96 at most.
__device__ __forceinline__ float score_factor(float qf, float ks) {
    const float f = qf * ks;
    return f < 0x1p-126f ? 0x1p-126f : f;
}
// consecutive logical indices on one XCD (workgroups are dealt to the 8 XCDs in turn): neighbours share a head's codes in that XCD's L2
__device__ __forceinline__ int xcd_order(int id, int n) {
    const int q = n / 8, r = n % 8, x = id % 8;
    return x * q + (x < r ? x : r) + id / 8;
}

static const int kRefLeast = -126;                          // p * v_scale below f32's normal numbers: zero or no more than 2^15 units
template <int D, int NC, int S>
__global__ __launch_bounds__(256 * S, 2) void kv8_attn_tile_kernel(Kv8Attn a, int blocks, float scale) {
    constexpr int ST = D / 32, NG = D / 16, KF = 4 * ST, VF = 2 * NG, PIECES = (D / 64 * 4 + NG) / 4;      // f16 fragments of a tile; 16-byte pieces a thread stages
    extern __shared__ __align__(16) char smem[];
    const Kv8View& c = a.c;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6 & 3, grp = S > 1 ? threadIdx.x >> 8 : 0, n = lane & 15, ch = lane >> 4;
    hf8* frag = reinterpret_cast<hf8*>(smem) + grp * (2 * (KF + VF) * 64);   // [2][KF + VF][64]: K fragments (group, step), V fragments (dimensions, half)
    const int id = xcd_order(blockIdx.x, gridDim.x), hkv = id / blocks, blk = blocks - 1 - id % blocks;       // longest rows first
    // S = 2: the columns are half a block from the front and half from the back, so that all workgroups have alike to do, and each SIMD has
    // a wave of either half
    const int G = c.H / c.Hkv, cols = a.M * G, set = (w + 2 * grp) & 3, half = set < 2 ? 2 * blocks - 1 - blk : blk;
    const int wcol0 = S > 1 ? half * 32 * NC + (set & 1) * 16 * NC : (blk * 4 + w) * 16 * NC, end = S > 1 ? (2 * blocks - blk) * 32 * NC : (blk + 1) * 64 * NC;
    const int T = a.n_past + (min(end, cols) - 1) / G + 1, tiles = (T + kKv8Tile - 1) / kKv8Tile;
    const int wrow0 = wcol0 / G, wrow1 = (min(wcol0 + 16 * NC, cols) - 1) / G;                             // rows this wave holds (none: wcol0 >= cols)
    const int8_t* kb = c.k + ((size_t)hkv * c.n_blk * kKv8Block + 16 * (n >> 2) + (n & 3)) * D + ch * 16;
    const int8_t* vb = c.v + (((size_t)hkv * c.n_blk + ch) * D + n) * 16;
    const float *ksb = c.ks + (size_t)hkv * c.n_blk + ch, *vsb = c.vs + (size_t)hkv * c.n_blk + ch;

    // piece p of a tile: K group p / (D/64), chunk p % (D/64), or V dimensions 16 (p - 4 D/64); wave w stages pieces w, w + 4, ...
    i4 st[PIECES];
    auto fetch = [&](int t) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int p = 4 * j + w;
            const int8_t* src = p < 4 * (D / 64) ? kb + (size_t)t * (kKv8Tile * D) + 4 * (p / (D / 64)) * D + (p % (D / 64)) * 64 : vb + (size_t)t * (kKv8Tile * D) + (p - 4 * (D / 64)) * 256;
            st[j] = *reinterpret_cast<const i4*>(src);
        }
    };
    auto stage = [&](int buf) {
        hf8* f = frag + (size_t)buf * (KF + VF) * 64 + lane;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int p = 4 * j + w;
            const HF8x2 h = codes_f16(st[j]);
            f[(2 * p) * 64] = h.a;                                         // K: fragment group * ST + 2 chunk (+ 1); V: KF + 2 dims (+ 1): both 2 p
            f[(2 * p + 1) * 64] = h.b;
        }
    };
    fetch(grp);                                                            // tiles to a multiple of S exist in the cache; those behind T are skipped
    hf8 qh[NC][ST], ql[NC][ST];
    float qf[NC], m[NC], l[NC];
    int ref[NC], lim[NC];
    f4 o[NC][NG];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        const int col = wcol0 + 16 * k + n;
        const bool valid = col < cols;
        lim[k] = valid ? a.n_past + col / G : T - 1;
        f4 x[D / 16];
        load_q<D>(a.q + (valid ? (size_t)(col / G) * c.H + hkv * G + col % G : 0) * D + ch * 16, valid, x);
        qf[k] = q_f16<D>(x, qh[k], ql[k]) * scale;
        m[k] = -INFINITY; l[k] = 0.f; ref[k] = kRefLeast;
#pragma unroll
        for (int g = 0; g < NG; ++g) o[k][g] = f4{0.f, 0.f, 0.f, 0.f};
    }
    stage(0);
    float ks = ksb[grp * 4], vs = vsb[grp * 4];
    asm("" : "+v"(ks), "+v"(vs));                                          // here, not in the loop, is where they are waited for
    __syncthreads();
    // One tile.  `more` is a constant in each of its two uses: with a branch around the loads the compiler would wait for all of them wherever
    // it waits for any.
    auto step = [&](int it, auto more_) {
        constexpr bool more = decltype(more_)::value;
        const int t = it * S + grp;
        float ksn = 0.f, vsn = 0.f;
        if (more) { fetch(t + S); ksn = ksb[(size_t)(t + S) * 4]; vsn = vsb[(size_t)(t + S) * 4]; }
        if (wcol0 < cols && t * kKv8Tile <= a.n_past + wrow1) {             // some row of this wave sees the tile
            const hf8* kf_ = frag + (size_t)(it & 1) * (KF + VF) * 64 + lane;
            const hf8* vf_ = kf_ + KF * 64;
            // both products: the fragments of the next step are read while the present one's matrix instructions run, and 2 NC sums
            // take turns, so that each finds its predecessor done
            f4 s[NC][4];
            hf8 fr[2][2][2];                                               // [turn][group of the pair][step of the pair]
            auto read_k = [&](int j) {                                     // pair j of groups x pair of steps
                const int g = j / (ST / 2) * 2, i = j % (ST / 2) * 2;
#pragma unroll
                for (int x = 0; x < 2; ++x) { fr[j & 1][0][x] = kf_[(g * ST + i + x) * 64]; fr[j & 1][1][x] = kf_[((g + 1) * ST + i + x) * 64]; }
            };
            read_k(0);
#pragma unroll
            for (int j = 0; j < ST; ++j) {
                const int g = j / (ST / 2) * 2, i = j % (ST / 2) * 2;
                if (j + 1 < ST) read_k(j + 1);
                if (i == 0) {
#pragma unroll
                    for (int k = 0; k < NC; ++k) s[k][g] = s[k][g + 1] = f4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
#pragma unroll
                    for (int k = 0; k < NC; ++k) {
                        s[k][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[j & 1][0][x], qh[k][i + x], s[k][g], 0, 0, 0);
                        s[k][g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[j & 1][1][x], qh[k][i + x], s[k][g + 1], 0, 0, 0);
                    }
#pragma unroll
                    for (int k = 0; k < NC; ++k) {
                        s[k][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[j & 1][0][x], ql[k][i + x], s[k][g], 0, 0, 0);
                        s[k][g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[j & 1][1][x], ql[k][i + x], s[k][g + 1], 0, 0, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            hf8 ph[NC][2], pl[NC][2];
            const int pos = t * kKv8Tile + ch * 16;
            const bool edge = t * kKv8Tile + kKv8Tile - 1 > a.n_past + wrow0;
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const float kf = pos > lim[k] ? 1.f : score_factor(qf[k], ks);      // a block nobody sees has only -inf: its own factor may be NaN
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[k][i >> 2][i & 3] = pos + i <= lim[k] ? s[k][i >> 2][i & 3] : -INFINITY;
                }
                float top = s[k][0][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, s[k][i >> 2][i & 3]);
                top = rounded_product(top, kf);
                const float mn = fmaxf(m[k], chunks_max(top)), mu = mn == -INFINITY ? 0.f : mn;
                float p[16], ls = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    p[i] = __builtin_amdgcn_exp2f(rounded_product(s[k][i >> 2][i & 3], kf) - mu);
                    ls += p[i];
                }
                const float vsu = pos <= lim[k] ? vs : 0.f;
                const unsigned wm = chunks_max_bits(as_u(fmaxf(__builtin_amdgcn_exp2f(top - mu), 0x1p-113f) * vsu));
                const int e = wm >= 0x7F800000u ? 1000 : wm == 0 ? -1000 : __builtin_amdgcn_frexp_expf(as_f(wm));
                if (__any(mn != m[k] || e > ref[k])) {                      // NaN maxima compare unequal: rescaled each time, harmless
                    const float al = __builtin_amdgcn_exp2f(m[k] - mu);
                    const int shrunk = ref[k] + (al > 0.f ? __builtin_amdgcn_frexp_expf(al) - 1 : -1000), rn = max(max(shrunk, e), kRefLeast);
                    const float f = ldexpf(al, max(min(ref[k] - rn, 2000), -2000));
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[k][g][i] *= f;
                    l[k] *= al; m[k] = mn; ref[k] = rn;
                }
                l[k] += ls;
                const float fac = ldexpf(vsu, 15 - ref[k]) + (as_f(wm) - as_f(wm));
#pragma unroll
                for (int h = 0; h < 2; ++h) split_f16(p + 8 * h, fac, ph[k][h], pl[k][h]);
            }
            auto read_v = [&](int j) {                                     // dimension pair j, both halves of the positions
#pragma unroll
                for (int h = 0; h < 2; ++h) { fr[j & 1][0][h] = vf_[(4 * j + h) * 64]; fr[j & 1][1][h] = vf_[(4 * j + 2 + h) * 64]; }
            };
            read_v(0);
#pragma unroll
            for (int j = 0; j < NG / 2; ++j) {
                if (j + 1 < NG / 2) read_v(j + 1);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int k = 0; k < NC; ++k) {
                        o[k][2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[j & 1][0][h], ph[k][h], o[k][2 * j], 0, 0, 0);
                        o[k][2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[j & 1][1][h], ph[k][h], o[k][2 * j + 1], 0, 0, 0);
                    }
#pragma unroll
                    for (int k = 0; k < NC; ++k) {
                        o[k][2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[j & 1][0][h], pl[k][h], o[k][2 * j], 0, 0, 0);
                        o[k][2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[j & 1][1][h], pl[k][h], o[k][2 * j + 1], 0, 0, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (more) { stage((it + 1) & 1); ks = ksn; vs = vsn; __syncthreads(); }
    };
    const int steps = (tiles + S - 1) / S;
    for (int it = 0; it + 1 < steps; ++it) step(it, std::true_type{});
    step(steps - 1, std::false_type{});
    if (S > 1) {                                                           // the second group's sums join the first's
        f4* so = reinterpret_cast<f4*>(smem);                              // [NC][NG + 1][256]
        const int tid = set * 64 + lane;
        __syncthreads();                                                   // the fragments have been read
        if (grp == 1) {
#pragma unroll
            for (int k = 0; k < NC; ++k) {
#pragma unroll
                for (int g = 0; g < NG; ++g) so[(k * (NG + 1) + g) * 256 + tid] = o[k][g];
                so[(k * (NG + 1) + NG) * 256 + tid] = f4{m[k], l[k], (float)ref[k], 0.f};
            }
        }
        __syncthreads();
        if (grp == 1) return;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const f4 st1 = so[(k * (NG + 1) + NG) * 256 + tid];
            const float mn = fmaxf(m[k], st1[0]), mu = mn == -INFINITY ? 0.f : mn, a0 = __builtin_amdgcn_exp2f(m[k] - mu), a1 = __builtin_amdgcn_exp2f(st1[0] - mu);
            const int r1 = (int)st1[2], rn = max(ref[k], r1);
            const float f0 = ldexpf(a0, max(ref[k] - rn, -2000)), f1 = ldexpf(a1, max(r1 - rn, -2000));
#pragma unroll
            for (int g = 0; g < NG; ++g) o[k][g] = o[k][g] * f0 + so[(k * (NG + 1) + g) * 256 + tid] * f1;
            l[k] = fmaf(st1[1], a1, l[k] * a0); m[k] = mn; ref[k] = rn;
        }
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        const int col = wcol0 + 16 * k + n;
        if (col >= cols) continue;
        const size_t r = (size_t)(col / G) * c.H + hkv * G + col % G;
        const float lt = chunks_sum(l[k]), inv = 1.f / lt;
#pragma unroll
        for (int g = 0; g < NG; ++g) {                                     // the unit last: with 1 / sum it may leave the normal numbers where the output does not
            f4 v = o[k][g] * inv;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = ldexpf(v[i], ref[k] - 15);
            *reinterpret_cast<f4*>(a.out + r * D + 16 * g + 4 * ch) = v;
        }
        if (a.ml && ch == 0) a.ml[r] = float2{m[k], lt};
    }
}

// ---------------------------------------------------------------- weight count of many rows
// mass_out = mass_in + sum over the columns of exp2(s - m) / l.  A workgroup takes 64 positions; its W waves share the columns, 16 at a time
// in turn, each with the K fragments of all 64 positions in registers and the next columns' q on the way; the waves' sums are added in a
// fixed order.  Scores anew instead of kept ones: [rows][heads][positions] would be hundreds of times the cache.  They are computed as the attention
// kernel computed them (F16: the one for many rows, its parts and order of products; else digits): m is one of them, and from any others large
// scores' weights would be off by the exponential of the difference.  512
// rows on 32 heads 13 us (15 in a trace), one workgroup a CU: its first tile's, with all rows' columns, has 1.8 times the mean to do and is what the
// launch takes.  The vector instructions are 4.1 us of it on even load; waves wait 45 % of their cycles.
template <int D, int W, bool F16>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void kv8_mass_tile_kernel(Kv8Attn a, float scale) {
    constexpr int KC = D / 64, ST = D / 32;
    __shared__ float part[W][64];
    const Kv8View& c = a.c;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 15, ch = lane >> 4, hkv = blockIdx.y, G = c.H / c.Hkv, cols = a.M * G;
    const int tile = blockIdx.x, pos = tile * kKv8Tile + ch * 16;          // lane chunk ch, score i: position pos + i
    const int row0 = max(tile * kKv8Tile - a.n_past, 0);                   // the first row that sees a position of this tile
    const int8_t* kb = c.k + ((size_t)hkv * c.n_blk * kKv8Block + (size_t)tile * kKv8Tile + 16 * (n >> 2) + (n & 3)) * D + ch * 16;
    i4 kr[4][KC];
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) kr[g][kc] = *reinterpret_cast<const i4*>(kb + 4 * g * D + kc * 64);
    const float ks = c.ks[(size_t)hkv * c.n_blk + (size_t)tile * 4 + ch];
    hf8 kh[4][ST];
    if (F16) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) { const HF8x2 h = codes_f16(kr[g][kc]); kh[g][2 * kc] = h.a; kh[g][2 * kc + 1] = h.b; }
    }
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.f;
    f4 x[D / 16];
    float2 ml;
    auto load = [&](int c0) {                                              // columns c0 + n; behind the last one the last one again
        const int col = min(c0 + n, cols - 1), row = col / G;
        const size_t r = (size_t)row * c.H + hkv * G + (col - row * G);
        load_q<D>(a.q + r * D + ch * 16, true, x);
        ml = a.ml[r];
    };
    int c0 = row0 * G / 16 * 16 + w * 16;
    if (c0 < cols) load(c0);
#pragma unroll 1
    for (; c0 < cols; c0 += 16 * W) {
        i4 qd[3][KC];
        hf8 qh[ST], ql[ST];
        const float qf = (F16 ? q_f16<D>(x, qh, ql) : q_digits<D>(x, qd)) * scale, top = ml.x, inv = 1.f / ml.y;
        load(min(c0 + 16 * W, cols - 1));                                      // without a branch: the next ones, or any
        const int row = min(c0 + n, cols - 1) / G, lim = c0 + n < cols ? a.n_past + row : -1;
        const bool edge = __any(tile * kKv8Tile + kKv8Tile - 1 > lim);
        const float kf = F16 ? score_factor(qf, ks) : qf * ks;             // NaN at most in a block this column does not see: left out below
        float p[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            f4 s;
            if (F16) {
                s = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < ST; ++st) {
                    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[g][st], qh[st], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[g][st], ql[st], s, 0, 0, 0);
                }
            } else {
                i4 acc[3];
#pragma unroll
                for (int d = 0; d < 3; ++d) {
                    acc[d] = i4{0, 0, 0, 0};
#pragma unroll
                    for (int kc = 0; kc < KC; ++kc) acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[g][kc], qd[d][kc], acc[d], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = join_digits(acc[2][i], acc[1][i], acc[0][i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) p[4 * g + i] = __builtin_amdgcn_exp2f(rounded_product(s[i], kf) - top);
        }
        if (edge) {                                                        // a row of NaN weights must not reach positions it does not see
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[i] += pos + i <= lim ? p[i] * inv : 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[i] = fmaf(p[i], inv, sum[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float t = row16_sum(sum[i]);
        if (n == i) part[w][ch * 16 + i] = t;
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int t = tile * kKv8Tile + threadIdx.x;
        const size_t at = (size_t)hkv * a.mass_ld + t;
        float all = part[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < W; ++i) all += part[i][threadIdx.x];
        if (t < a.n_past + a.M) a.mass_out[at] = a.mass_in[at] + all;
    }
}
// entries behind the slab's positions: carried over
__global__ __launch_bounds__(256) void kv8_mass_rest_kernel(Kv8Attn a) {
    const int t = a.n_past + a.M + blockIdx.x * 256 + threadIdx.x;
    if (t < a.mass_n) a.mass_out[(size_t)blockIdx.y * a.mass_ld + t] = a.mass_in[(size_t)blockIdx.y * a.mass_ld + t];
}

// ---------------------------------------------------------------- launchers
template <typename F> static hipError_t lds_opt_in(F kernel, size_t bytes) {
    return bytes > 32768 ? hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : hipSuccess;
}

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
                             unsigned* work, int64_t work_words, hipStream_t st) {
    const int64_t slices = std::min((T + 4095) / 4096, (int)std::min<int64_t>(work_words / (Hkv * kKv8SliceWords), 64));
    if (T > kKv8SliceFrom && slices >= 2) {
        const int n = (int)slices, slice = ((T + n - 1) / n + 3) & ~3;
        Slices s{work, work + (size_t)3 * Hkv * n * 2048, nullptr};
        s.picks = s.above + (size_t)2 * Hkv * n;
        auto part = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(n, Hkv), dim3(1024), 0, st, T, slice, n_keep, n_sink, n_recent, mass_in, ld_in, mass_out, ld_out, kept, s);
        };
        part(kv8_select_slice_kernel<0>); part(kv8_select_slice_kernel<1>); part(kv8_select_slice_kernel<2>); part(kv8_select_slice_kernel<3>);
        return hipGetLastError();
    }
#define KV8_SELECT(W, N, BITS)                                                                                                                       \
    do {                                                                                                                                           \
        const size_t lds = (size_t)N * 64 * W * 4;                                                                                                 \
        const hipError_t e = lds_opt_in(kv8_select_kernel<W, N, BITS>, lds);                                                                       \
        if (e != hipSuccess) return e;                                                                                                             \
        hipLaunchKernelGGL((kv8_select_kernel<W, N, BITS>), dim3(Hkv), dim3(64 * W), lds, st, T, n_keep, n_sink, n_recent, mass_in, ld_in, mass_out, \
                           ld_out, kept);                                                                                                          \
    } while (0)
    // 32 heads, with the move of 64 positions (4 us): T = 5000 14 us, 32768 27; 8 heads, T = 65536 67 us on one workgroup a head, 37 in slices,
    // 131072 125 and 44; in slices T = 32768 would take 30
    if (T <= 1024) KV8_SELECT(4, 4, 8);
    else if (T <= 4096) KV8_SELECT(16, 4, 11);
    else if (T <= 32768) KV8_SELECT(16, 32, 11);
    else KV8_SELECT(16, 0, 11);
#undef KV8_SELECT
    return hipGetLastError();
}
hipError_t launch_kv8_move(const Kv8View& src, const Kv8View& dst, int n_keep, const int32_t* kept, hipStream_t st) {
    const dim3 grid((unsigned)((n_keep + kKv8Block - 1) / kKv8Block), src.Hkv, 2);
    KV8_BY_DIM(src.D, hipLaunchKernelGGL(kv8_move_kernel<kD>, grid, dim3(256), 0, st, src, dst, n_keep, kept));
    return hipGetLastError();
}
template <int D, int NC, int S> static hipError_t attn_tile(const Kv8Attn& a, hipStream_t st) {
    constexpr size_t lds = (size_t)S * 2 * (4 * (D / 32) + 2 * (D / 16)) * 64 * 16;
    const int cols = a.M * (a.c.H / a.c.Hkv), blocks = (cols + 64 * NC - 1) / (64 * NC);
    const hipError_t e = lds_opt_in(kv8_attn_tile_kernel<D, NC, S>, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((kv8_attn_tile_kernel<D, NC, S>), dim3(blocks * a.c.Hkv), dim3(256 * S), lds, st, a, blocks, kLog2e / sqrtf((float)D));
    return hipGetLastError();
}
template <int D> static hipError_t attn_tile(const Kv8Attn& a, hipStream_t st) {
    // Wide: 32 columns a wave halve the LDS reads of 16.  Two groups of waves (S = 2) where there is at most one workgroup a CU: 512 rows on 32 heads
    // 18.8 -> 16.2 us narrow, 1024 rows over 8192 positions 316 -> 273 us wide instead of narrow.  With more, one group, and two workgroups a CU;
    // narrow ones until there are enough wide ones to share the CUs evenly: 800 rows on 40 heads (280 wide ones) 30 us narrow, 38 wide; 1500 rows
    // over 8192 positions, 32 heads on 8 (376) 495 and 472, but from the start 52 and 67.
    const int64_t cols = (int64_t)a.M * (a.c.H / a.c.Hkv), narrow = (cols + 63) / 64 * a.c.Hkv, wide = (cols + 127) / 128 * a.c.Hkv;
    if (narrow <= 256) return attn_tile<D, 1, 2>(a, st);
    if (wide <= 256) return attn_tile<D, 2, 2>(a, st);
    return wide < 384 ? attn_tile<D, 1, 1>(a, st) : attn_tile<D, 2, 1>(a, st);
}
hipError_t launch_kv8_attn_tile(const Kv8Attn& a, hipStream_t st) {
    switch (a.c.D) {
        case 64: return attn_tile<64>(a, st);
        case 128: return attn_tile<128>(a, st);
        case 256: return attn_tile<256, 1, 1>(a, st);                      // one group's tiles fill the LDS
        default: return hipErrorInvalidValue;
    }
}
template <int D> static hipError_t mass_tile(const Kv8Attn& a, hipStream_t st) {
    const int tiles = (a.n_past + a.M + kKv8Tile - 1) / kKv8Tile;
    constexpr int W = D == 256 ? 4 : 8;
    const dim3 grid(tiles, a.c.Hkv);
    const float scale = kLog2e / sqrtf((float)D);
    if (a.halves) hipLaunchKernelGGL((kv8_mass_tile_kernel<D, W, true>), grid, dim3(64 * W), 0, st, a, scale);
    else hipLaunchKernelGGL((kv8_mass_tile_kernel<D, W, false>), grid, dim3(64 * W), 0, st, a, scale);
    const int rest = a.mass_n - (a.n_past + a.M);
    if (rest > 0 && a.mass_in != a.mass_out) hipLaunchKernelGGL(kv8_mass_rest_kernel, dim3((rest + 255) / 256, a.c.Hkv), dim3(256), 0, st, a);
    return hipGetLastError();
}
hipError_t launch_kv8_attn_mass(const Kv8Attn& a, hipStream_t st) {
    KV8_BY_DIM(a.c.D, return mass_tile<kD>(a, st));
    return hipErrorInvalidValue;
}
template <int D, int W> static void attn_split(const Kv8Attn& a, const Kv8Split& sp, hipStream_t st) {
    const dim3 grid(sp.n, a.c.Hkv, (a.M * (a.c.H / a.c.Hkv) + 15) / 16);
    const float scale = kLog2e / sqrtf((float)D);
    if (sp.stream) hipLaunchKernelGGL((kv8_attn_split_kernel<D, W, true>), grid, dim3(64 * W), 0, st, a, sp, scale);
    else hipLaunchKernelGGL((kv8_attn_split_kernel<D, W, false>), grid, dim3(64 * W), 0, st, a, sp, scale);
}
hipError_t launch_kv8_attn_split(const Kv8Attn& a, const Kv8Split& sp, hipStream_t st) {
    switch (a.c.D) {
        case 64: attn_split<64, kv8_split_waves(64)>(a, sp, st); break;
        case 128: attn_split<128, kv8_split_waves(128)>(a, sp, st); break;
        case 256: attn_split<256, kv8_split_waves(256)>(a, sp, st); break;
        default: return hipErrorInvalidValue;
    }
    if (!sp.counters && sp.n > 1) {
        const unsigned mass = sp.scores ? (unsigned)((a.mass_n + 511) / 512 * a.c.Hkv) : 0u;
        KV8_BY_DIM(a.c.D, hipLaunchKernelGGL(kv8_attn_finish_kernel<kD>, dim3(a.M * a.c.H + mass), dim3(256), 0, st, a, sp));
    }
    return hipGetLastError();
}

}  // namespace thk
