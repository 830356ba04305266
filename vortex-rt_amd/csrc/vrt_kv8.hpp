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
// Dimensions past head_dim, up to a multiple of 32, hold zeros.
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
    float* tmax;       // [region][head][parity][K, V][32]: max |x| of the tail's rows (not finite: a value of it is not)
    uint32_t nb, kvh, hd, hdp;
};

// One sequence of a call.
struct Kv8Seq {
    uint32_t seq, pos, n, prefix;   // as vrt_kv8_rows
    uint32_t row0;                  // its first row of q / k / v / out
    uint32_t item0;                 // its first (row tile, head) of the attention's workspace
};

}  // namespace vrt
