// thk_kv8.hpp — the 8-bit K/V cache (thk_kv8_* of include/thk.h): device layout and launchers.  Internal.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace thk {

static const int kKv8Block = 16;      // positions that share one K scale and one V scale per K/V head
static const int kKv8Tile = 64;       // positions one step of the split attention kernel takes
static const int kKv8Pad = 128;       // a cache holds whole multiples of this many positions: no kernel's step reads behind it
static const int kKv8SplitRows = 4096; // rows x parts a launch has at most: 16 columns of 256 workgroups
static const int kKv8SliceFrom = 32768; // positions above which the selection may go in slices
static const int kKv8SliceRows = 8192; // rows of D words a cache that long keeps for the slices' counts: 5 slices at 32 heads of 128, 10 at 16
static const int kKv8Groups = 512;    // column groups x K/V heads up to which the positions are split (and counters there are)
static const int kKv8SliceWords = 3 * 2048 + 16; // what the selection of long sets keeps for a slice of a head, in words
static const int kKv8ScoredHeads = 16; // query heads of a K/V head up to which a single row's scores are kept for the weight count (else they are computed again)
static const int kKv8RowSlab = 2048;  // prompt rows one attention launch takes (sizes the per-row statistics)

// Device memory of one cache.  n_blk = blocks per head, a multiple of 8 (kKv8Pad).
//   k    int8 [Hkv][n_blk][16][D]    codes, row-major: a position's D codes are contiguous
//   v    int8 [Hkv][n_blk][D][16]    codes, transposed inside the block: the 16 positions of one dimension are contiguous, which is
//                                    the operand chunk of one lane when positions are the summed axis of a matrix instruction
//   ks, vs f32 [Hkv][n_blk]          scales
//   tail f32 [2][Hkv][16][D]         the rows of the block that was appended to last, unrounded (K, then V)
//   tail_at int2 [2][Hkv]            which block that is (-1: none) and how many of its rows tail holds
struct Kv8View {
    int8_t *k, *v;
    float *ks, *vs;
    float* tail;
    int2* tail_at;
    int n_blk, H, Hkv, D;
};

struct Kv8Attn {
    Kv8View c;
    const float* q;                   // [M][H][D]
    float* out;                       // [M][H][D]
    int n_past, M;                    // row i sees positions <= n_past + i
    float2* ml;                       // [M][H] running maximum (base-2 scores) and sum of every row, for the weight count; or null
    bool halves;                      // those are of scores from q in two f16 parts (the kernel for many rows), not from its digits
    const float* mass_in;             // [Hkv][mass_ld] or null (then no weights are counted)
    float* mass_out;
    int64_t mass_ld;
    int mass_n;                       // entries per head that are written: all positions of the call, also those this slab's rows do not see yet
};

// Few rows over a long axis: the positions are cut into n <= 64 parts of whole tiles.  With counters the last workgroup of a column group joins
// the parts (and counts the weights), otherwise a second launch does where n > 1.  Scores without counters need n > 1.
struct Kv8Split {
    int n;
    bool stream;                      // the codes are read past the caches
    float* part_o;                    // [M H][n][D]
    float2* part_ml;                  // [M H][n]
    float* scores;                    // [H][scores_ld] base-2 scores of a single row, for the weight count; or null
    int64_t scores_ld;
    unsigned* counters;               // one per column group and K/V head, zero between launches; or null
};
constexpr int kv8_split_waves(int D) { return D == 256 ? 4 : 8; }      // of a workgroup, a tile each in turn; one workgroup fills a CU's registers (two, D = 64)

hipError_t launch_kv8_append(const Kv8View& c, const float* k, const float* v, int64_t pos, int64_t n, hipStream_t st);
hipError_t launch_kv8_read(const Kv8View& c, int64_t pos, int64_t n, float* k_out, float* v_out, hipStream_t st);
hipError_t launch_kv8_select(int Hkv, int T, int n_keep, int n_sink, int n_recent, const float* mass_in, int64_t ld_in, float* mass_out, int64_t ld_out, int32_t* kept,
                             unsigned* work, int64_t work_words, hipStream_t st);
hipError_t launch_kv8_move(const Kv8View& src, const Kv8View& dst, int n_keep, const int32_t* kept, hipStream_t st);
hipError_t launch_kv8_attn_tile(const Kv8Attn& a, hipStream_t st);
hipError_t launch_kv8_attn_split(const Kv8Attn& a, const Kv8Split& sp, hipStream_t st);
hipError_t launch_kv8_attn_mass(const Kv8Attn& a, hipStream_t st);

}  // namespace thk
