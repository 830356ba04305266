// vrt_kv8.hpp -- the 8-bit key/value cache (vrt_kv8.hip): layout and launches.
//
// A cache is max_seqs regions x kv heads x nb blocks of 32 positions; position p of a region is in block
// (p / 32) % nb, so a region is a ring for windowed attention. A full ("closed") block holds int8 codes q and one
// scale each for its keys and values, the value being fl32(q s). The positions of the block that is not full (and
// of the block before it, so that a sequence can be taken back by a few positions) are kept in fp32, the "tail": two
// buffers per region and head, a block's is its number's parity. What a sequence was appended in does not matter to what
// the cache holds.
//
// Codes are kept in operand order of v_mfma_f32_16x16x32_f16 (lane l: row l % 16, k = 8 (l / 16) + e, e < 8), biased
// to unsigned bytes (q + 128), two tiles side by side, so that a lane's load is 16 bytes and a wave's 1 KB:
//   keys    [dim / 32][lane][token / 16][8]: row = token % 16, k = dim % 32
//   values  [dim / 32][lane][(dim / 16) % 2][8]: row = dim % 16, k = the token order in which a lane of the
//           transposed scores (rows: tokens 4 g + r of both halves, g = lane / 16) holds its eight weights:
//           token = 4 g + e for e < 4, 16 + 4 g + e - 4 after, so weights go from one product into the next in registers
// Dimensions past head_dim, up to a multiple of 32, hold zeros. The tail is kept twice: as fp32 rows, which a block's codes
// are made of, and as pairs of halves in the same operand order, each row scaled by a power of two, which the attention reads.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "vrt_hip.h"

namespace vrt {

constexpr uint32_t kKvBlock = VRT_KV8_BLOCK;
constexpr uint32_t kKvMaxSeqs = VRT_KV8_MAX_SEQS;

struct Kv8Dev {
    uint8_t* codes;    // [region][head][nb][K, V: 32 hdp each]
    float2* scales;    // [region][head][nb]: key and value scale
    float* tail;       // [region][head][parity][K, V][32][hdp]
    _Float16* pairs;   // [region][head][parity][K, V][high, low][32 hdp]: a row x as x 2^e = high + low
    float* factor;     // [region][head][parity][K, V][32]: 2^-e of the row; NaN: a value of it is not finite, its pair is 0
    uint32_t nb, kvh, hd, hdp;
};

// One sequence of a call.
struct Kv8Seq {
    uint32_t seq, pos, n, prefix;   // as vrt_kv8_rows
    uint32_t row0;                  // its first row of q / k / v / out
    uint32_t splits;                // splits of each of its (unit, head)s, and the first's place in the workspace
    uint32_t part0;
};

// Attention outputs: fp32 rows, or (gm not null) the activation buffer of a projection (vrt_gemm.hpp).
struct Kv8Out {
    float* rows;
    uint64_t stride;
    _Float16* gm;
    uint32_t gm_nkb;
    uint32_t* nonfinite;   // not null: a row whose sum of weights is not a positive number lowers it to code
    uint32_t code;
};

struct Kv8AttnArgs {
    Kv8Dev c;
    Kv8Out o;
    const float* q;
    uint64_t q_stride;
    float* part;          // [place][lines][hdp] unnormalised outputs, where a unit has several splits
    float2* part_ml;      // [place][lines]: reference maximum (log2 units) and sum
    float2* stats;        // [row][heads]: final maximum and 1 / sum (prompts, with weights)
    float* scores;        // single tokens, with weights: [place][lines][32 per] scores in log2 units
    const float* w_in;
    float* w_out;
    uint32_t heads, G, window, max_ctx;
    uint32_t unit;        // rows that run together: 16 (single tokens: a workgroup's waves share them), or a wave's own (prompt)
    uint32_t prompt, fold, lines;   // fold: all units run at once; lines: rows of a place in the workspace
    uint32_t per, splits; // blocks of a split; the most splits of a sequence
    uint32_t nseq, rows_most;   // rows_most: the most rows (queries times the heads of a group) of a sequence
    float scale, cap;
    Kv8Seq s[kKvMaxSeqs];
};

// A cache's memory: sizes of its parts, and the view of it.
struct Kv8Sizes {
    uint64_t codes, scales, tail, pairs, factor, total;
    uint32_t nb, hdp;
};
Kv8Sizes kv8_sizes(uint32_t max_seqs, uint32_t max_ctx, uint32_t kv_heads, uint32_t head_dim);
Kv8Dev kv8_view(const Kv8Sizes& z, void* data, uint32_t kv_heads, uint32_t head_dim);

// Launches on checked arguments. kv8_plan fills the split of A (heads, G, window and s[].seq .. row0 given) and says what the
// workspace has to hold; for one token a sequence at most kv8_workspace_most(...) bytes.
struct Kv8Plan {
    uint32_t units;    // the most of a sequence
    uint64_t part, ml, extra, total;
};
Kv8Plan kv8_plan(Kv8AttnArgs& A, uint32_t kvh, uint32_t hdp, uint32_t n, uint64_t rows, bool scored);
uint64_t kv8_workspace_most(uint32_t seqs, uint32_t max_ctx, uint32_t heads, uint32_t kvh, uint32_t hdp, bool scored);
int kv8_append(const Kv8Dev& c, const Kv8Seq* seqs, uint32_t n, const float* k, const float* v, uint64_t stride, hipStream_t s);
int kv8_attend(Kv8AttnArgs& A, const Kv8Plan& P, void* workspace, uint32_t n, hipStream_t s);
int kv8_evict(const Kv8Dev& c, const vrt_kv8_move* moves, uint32_t n, float* weights, uint32_t max_ctx, uint32_t* kept,
              uint64_t kept_stride, hipStream_t s);

}  // namespace vrt
