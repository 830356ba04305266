// vrt_kv8.hip -- the 8-bit key/value cache: append, read, attention, eviction (vrt_kv8_*).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "vrt_gemm.hpp"
#include "vrt_internal.hpp"
#include "vrt_kv8.hpp"
#include "vrt_q8_device.hpp"

namespace vrt {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kKvThreads = 256;
constexpr int kKvNoExp = -1000;   // no value scale yet

// ---- layout ---------------------------------------------------------------------------------

__device__ __forceinline__ uint64_t kv_block(const Kv8Dev& c, uint32_t seq, uint32_t head, uint32_t b) {
    return (static_cast<uint64_t>(seq) * c.kvh + head) * c.nb + (b < c.nb ? b : b % c.nb);
}
__device__ __forceinline__ uint8_t* kv_codes(const Kv8Dev& c, uint64_t block) { return c.codes + block * 64u * c.hdp; }
// The tail buffer of block b's keys or values, of 32 rows.
__device__ __forceinline__ uint64_t kv_tail_buf(const Kv8Dev& c, uint32_t seq, uint32_t head, uint32_t b, uint32_t z) {
    return ((static_cast<uint64_t>(seq) * c.kvh + head) * 2u + (b & 1u)) * 2u + z;
}
// Byte of a value inside its block's 32 hdp bytes.
__device__ __forceinline__ uint32_t kv_k_at(uint32_t t, uint32_t d) {
    return (d >> 5) * 1024u + (((d >> 3) & 3u) * 16u + (t & 15u)) * 16u + (t >> 4) * 8u + (d & 7u);
}
__device__ __forceinline__ uint32_t kv_v_at(uint32_t t, uint32_t d) {
    return (d >> 5) * 1024u + (((t >> 2) & 3u) * 16u + (d & 15u)) * 16u + ((d >> 4) & 1u) * 8u + (t & 3u) + (t >> 4) * 4u;
}

// A launch's arguments lie in memory that nothing has cached; read where they are used, they cost a latency for every line.
// These ask for the ones that a kernel uses all at once.
__device__ __forceinline__ void kv_ask(const Kv8Dev& c) {
    asm volatile("" ::"s"(c.codes), "s"(c.scales), "s"(c.tail), "s"(c.pairs), "s"(c.factor), "s"(c.nb), "s"(c.kvh), "s"(c.hd), "s"(c.hdp));
}
__device__ __forceinline__ void kv_ask(const Kv8Seq& s) {
    asm volatile("" ::"s"(s.seq), "s"(s.pos), "s"(s.n), "s"(s.prefix), "s"(s.row0), "s"(s.splits), "s"(s.part0));
}
__device__ __forceinline__ void kv_ask(const Kv8AttnArgs& A) {
    asm volatile("" ::"s"(A.c.codes), "s"(A.c.scales), "s"(A.c.pairs), "s"(A.c.factor), "s"(A.c.nb), "s"(A.c.kvh), "s"(A.c.hd), "s"(A.c.hdp),
                 "s"(A.o.rows), "s"(A.o.stride), "s"(A.o.gm), "s"(A.q), "s"(A.q_stride), "s"(A.part), "s"(A.part_ml), "s"(A.heads),
                 "s"(A.G), "s"(A.window), "s"(A.per), "s"(A.splits), "s"(A.nseq), "s"(A.scale));
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max_u32(uint32_t v) {   // lanes outside the row mask keep their own
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(v), static_cast<int>(v), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {   // wave-uniform (the steps of wave_red_max)
    v = dpp_max_u32<0xB1, 0xf>(v);
    v = dpp_max_u32<0x4E, 0xf>(v);
    v = dpp_max_u32<0x141, 0xf>(v);
    v = dpp_max_u32<0x140, 0xf>(v);
    v = dpp_max_u32<0x142, 0xa>(v);
    v = dpp_max_u32<0x143, 0xc>(v);
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

// Pairs of floats to pairs of halves, hi + lo = x (below 2^15 in magnitude; what is lost is below 2^-24). The barrier: see gm_split.
__device__ __forceinline__ void kv_split2(float x, float y, h2& hi, h2& lo) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    asm("" : "+v"(x), "+v"(y));
    hi = __builtin_convertvector((f2{x, y}), h2);
    lo = __builtin_convertvector((f2{x - static_cast<float>(hi[0]), y - static_cast<float>(hi[1])}), h2);
}

// The exponent e with m 2^e in [2^(to - 1), 2^to), at most 126 so that 2^-e is a number; 0 where m is 0 or not finite.
__device__ __forceinline__ int kv_exp(float m, int to) {
    return m > 0.0f && m < INFINITY ? min(to - __builtin_amdgcn_frexp_expf(m), 126) : 0;
}

// x / s to the nearest integer, ties to even, of the exact quotient: the remainder x - q s of the estimate is exact (q
// has 8 bits, and it is below s), and says whether the estimate is one off.
__device__ __forceinline__ float kv_round(float x, float s, float inv) {
#pragma clang fp contract(off)
    float q = rintf(x * inv);
    const float r = __builtin_fmaf(-q, s, x), half = 0.5f * s;
    const bool odd = static_cast<int>(q) & 1;
    if (r > half || (r == half && odd)) q += 1.0f;
    else if (r < -half || (r == -half && odd)) q -= 1.0f;
    return __builtin_amdgcn_fmed3f(q, -127.0f, 127.0f);
}

// ---- append ---------------------------------------------------------------------------------

// A workgroup's 32 rows of one head and block: KU float4 a thread (unit tid + TH k: token unit / (8 NT), dims 4 (unit % (8 NT)) ..;
// zeros past hd; the last unit again past the end), their largest magnitude, scale, codes, in operand order through an LDS
// image. Of 96 dims and more, 512 threads: with 256 a thread's share of 256 dims takes 217 registers, or spills; with 1024
// from 160 dims on an eviction's tiles take 137 us for 125 and a read's 65 for 52 (64 sequences, 2048 positions of 256 dims).
template <int NT>
struct KvTile {
    static constexpr uint32_t TH = NT >= 3 ? 512u : 256u, KU = (256u * NT + TH - 1u) / TH;
    f4 v[KU];
};
template <int NT>
__device__ __forceinline__ void kv_unit(uint32_t k, uint32_t& t, uint32_t& d) {
    const uint32_t u = min(threadIdx.x + KvTile<NT>::TH * k, 256u * NT - 1u);
    t = u / (8u * NT);
    d = (u - t * 8u * NT) * 4u;
}
__device__ __forceinline__ uint32_t f_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Largest magnitudes of the tile's rows, as integers: larger is larger, NaN above infinity above the rest. (Eight neighbouring
// lanes have the same row.)
template <int NT>
__device__ __forceinline__ void kv_row_max(const KvTile<NT>& x, uint32_t* rowmax) {
    if (threadIdx.x < 32u) rowmax[threadIdx.x] = 0u;
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
        uint32_t t, d, m = max(max(f_bits(x.v[k][0]), f_bits(x.v[k][1])), max(f_bits(x.v[k][2]), f_bits(x.v[k][3])));
        m = dpp_max_u32<0xB1, 0xf>(m);
        m = dpp_max_u32<0x4E, 0xf>(m);
        m = dpp_max_u32<0x141, 0xf>(m);
        kv_unit<NT>(k, t, d);
        if ((threadIdx.x & 7u) == 0u) atomicMax(&rowmax[t], m);
    }
    __syncthreads();
}

// Places (bytes) of operand-order images in LDS. A row's neighbouring values are 16 bytes apart, or 256: in order, all 64 lanes
// of a row meet in 4 or 8 of the 64 banks. Mixed, units of 16 bytes change places among the 16 of their 256 bytes, by the bits
// that tell a row's units apart; reads of units in order still have all banks. An eviction's gather, with an image more, takes
// 100 us for 125 (64 sequences, 2048 positions of 256 dims). Append, which waits for memory and needs the registers, leaves them in
// order: 4 fills of 8192 positions, 2 heads of 256, take 44 us, with mixed tails 62.
template <bool MIX>
__device__ __forceinline__ uint32_t kv_img(uint32_t z, uint32_t at) {
    return !MIX ? at : z ? at ^ (at >> 6 & 0x30u) : at ^ (at >> 4 & 0xf0u);
}
template <bool MIX>
__device__ __forceinline__ uint32_t kv_img_pairs(uint32_t z, uint32_t at) {   // of halves
    return !MIX ? at : z ? at ^ (at >> 6 & 0x30u) : at ^ (at >> 4 & 0x30u) ^ (at >> 5 & 0xc0u);
}

// A full block's codes and scale.
template <int NT, bool MIX>
__device__ __forceinline__ void kv_close_block(const Kv8Dev& c, const KvTile<NT>& x, const uint32_t* rowmax, uint64_t block, uint32_t z,
                                               uint8_t* img) {
    const uint32_t tid = threadIdx.x, m = wave_max_u32(rowmax[tid & 31u]);
    const float s = m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(m) / 127.0f;
    uint32_t w[KvTile<NT>::KU];
#pragma unroll
    for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) w[k] = 0x80808080u;
    if (s > 0.0f) {
        // the quotient's steps stay away from denormals: their halves and reciprocals are no numbers
        const float up = s < 0x1p-100f ? 0x1p60f : 1.0f, su = s * up, inv = 1.0f / su, half = 0.5f * su;
        bool near = false;   // a remainder of half a step or more: the quotient may be one off, or a tie
#pragma unroll
        for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
            w[k] = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y = x.v[k][e] * up, q = __builtin_amdgcn_fmed3f(rintf(y * inv), -127.0f, 127.0f);
                near |= fabsf(__builtin_fmaf(-q, su, y)) >= half;
                w[k] = __builtin_amdgcn_cvt_pk_u8_f32(q + 128.0f, e, w[k]);
            }
        }
        if (__any(near))   // seldom
#pragma unroll
            for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
                w[k] = 0u;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[k] = __builtin_amdgcn_cvt_pk_u8_f32(kv_round(x.v[k][e] * up, su, inv) + 128.0f, e, w[k]);
            }
    }
#pragma unroll
    for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
        uint32_t t, d;
        kv_unit<NT>(k, t, d);
        if (z == 0u) {
            *reinterpret_cast<uint32_t*>(img + kv_img<MIX>(0u, kv_k_at(t, d))) = w[k];
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) img[kv_img<MIX>(1u, kv_v_at(t, d + e))] = static_cast<uint8_t>(w[k] >> (8u * e));
        }
    }
    __syncthreads();
    uint4* dst = reinterpret_cast<uint4*>(kv_codes(c, block) + z * 32u * c.hdp);
    for (uint32_t i = tid; i < 64u * NT; i += KvTile<NT>::TH) dst[i] = *reinterpret_cast<const uint4*>(img + kv_img<MIX>(z, 16u * i));
    if (tid == 0u) reinterpret_cast<float*>(c.scales + block)[z] = s;
}

// Rows whose pairs are scattered: a step's one, as a buffer of 64 KB would be written for it; more go through LDS.
constexpr uint32_t kKvFew = 2;

// Halves of a row's pair in operand order: K by four dims, V by one.
__device__ __forceinline__ uint32_t kv_k_half(uint32_t t, uint32_t d) {
    return ((d >> 5) * 2u + (t >> 4)) * 512u + (((d >> 3) & 3u) * 16u + (t & 15u)) * 8u + (d & 7u);
}
__device__ __forceinline__ uint32_t kv_v_half(uint32_t t, uint32_t d) {
    return (d >> 4) * 512u + (((t >> 2) & 3u) * 16u + (d & 15u)) * 8u + (t & 3u) + (t >> 4) * 4u;
}

// Rows r0 .. r1 - 1 of the tile (which has all rows below r1) into a tail buffer: the fp32 rows, and pairs of halves in operand order.
// The halves of a row with a value that is not finite are zeros, so that what is masked adds nothing; its factor says so.
// A few rows' pairs are scattered (a value's halves are 2-byte stores, 16 bytes apart); of more, the whole buffer's go
// through LDS: scattered, 32 rows of 256 took a workgroup 7 us. img: 2048 NT bytes.
template <int NT, bool MIX>
__device__ __forceinline__ void kv_store_tail(const Kv8Dev& c, const KvTile<NT>& x, const uint32_t* rowmax, uint64_t buf, uint32_t z,
                                              uint32_t r0, uint32_t r1, uint8_t* img) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    _Float16* const dst = c.pairs + buf * 64u * c.hdp;
    const uint32_t tid = threadIdx.x;
    if (tid >= r0 && tid < r1) {
        const uint32_t m = rowmax[tid];
        c.factor[buf * 32u + tid] = m < 0x7f800000u ? ldexpf(1.0f, -kv_exp(__uint_as_float(m), 7)) : __uint_as_float(0x7fc00000u);
    }
    auto row = [&](uint32_t k, uint32_t t, h4 (&pair)[2]) {
        const uint32_t m = rowmax[t];
        const bool ok = m < 0x7f800000u && t < r1;
        const float up = ldexpf(1.0f, kv_exp(__uint_as_float(m), 7));
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            h2 a, b;
            kv_split2(ok ? x.v[k][e] * up : 0.0f, ok ? x.v[k][e + 1] * up : 0.0f, a, b);
            pair[0][e] = a[0], pair[0][e + 1] = a[1];
            pair[1][e] = b[0], pair[1][e + 1] = b[1];
        }
    };
    if (r1 - r0 <= kKvFew) {
#pragma unroll
        for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
            uint32_t t, d;
            kv_unit<NT>(k, t, d);
            if (t < r0 || t >= r1) continue;
            *reinterpret_cast<f4*>(c.tail + (buf * 32u + t) * c.hdp + d) = x.v[k];
            h4 pair[2];
            row(k, t, pair);
#pragma unroll
            for (uint32_t part = 0; part < 2u; ++part) {
                _Float16* const to = dst + part * 32u * c.hdp;
                if (z == 0u) *reinterpret_cast<h4*>(to + kv_k_half(t, d)) = pair[part];
                else
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e) to[kv_v_half(t, d + e)] = pair[part][e];
            }
        }
        return;
    }
#pragma unroll 1
    for (uint32_t part = 0; part < 2u; ++part) {
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
            uint32_t t, d;
            kv_unit<NT>(k, t, d);
            if (part == 0u && t >= r0 && t < r1) *reinterpret_cast<f4*>(c.tail + (buf * 32u + t) * c.hdp + d) = x.v[k];
            h4 pair[2];
            row(k, t, pair);
            const h4 v = part ? pair[1] : pair[0];
            if (z == 0u) *reinterpret_cast<h4*>(img + kv_img_pairs<MIX>(0u, 2u * kv_k_half(t, d))) = v;
            else
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) *reinterpret_cast<_Float16*>(img + kv_img_pairs<MIX>(1u, 2u * kv_v_half(t, d + e))) = v[e];
        }
        __syncthreads();
        uint4* const to = reinterpret_cast<uint4*>(dst + part * 32u * c.hdp);
        for (uint32_t i = tid; i < 128u * NT; i += KvTile<NT>::TH) to[i] = *reinterpret_cast<const uint4*>(img + kv_img_pairs<MIX>(z, 16u * i));
    }
}

struct Kv8AppendArgs {
    Kv8Dev c;
    const float* x[2];   // k, v
    uint64_t stride;
    Kv8Seq s[kKvMaxSeqs];
};

// One workgroup per (block the call touches, head and K or V, sequence): a full block's codes; of the last two blocks, the call's
// rows into the tail. The first block's earlier rows come from the tail, which a later block of the same parity overwrites:
// the first block's workgroup does that one too, after its own.
// Memory's time for long calls (2 sequences of 8192, 8 heads of 128: 55 us, 3.1 TB/s read and written); latency's for short ones
// (one position 3.5 us, 48 fills of up to 70 positions of 256 dims 12, most of it the tails).
template <int NT>
__global__ void __launch_bounds__((KvTile<NT>::TH)) k_kv8_append(const Kv8AppendArgs A) {
    __shared__ __align__(16) uint8_t img[2048 * NT];
    __shared__ uint32_t rowmax[32];
    const Kv8Dev& c = A.c;
    const Kv8Seq& S = A.s[blockIdx.z];
    const uint32_t head = blockIdx.y >> 1, z = blockIdx.y & 1u;
    kv_ask(c);
    kv_ask(S);
    asm volatile("" ::"s"(A.x[0]), "s"(A.x[1]), "s"(A.stride));
    if (S.n == 0u) return;
    const uint32_t end = S.pos + S.n, b0 = S.pos >> 5, bl = (end - 1u) >> 5;
    const float* x = A.x[z] + static_cast<uint64_t>(S.row0) * A.stride + head * c.hd;
    // the block of the last two that has the first one's tail, if the first one reads it
    const uint32_t other = (S.pos & 31u) && bl > b0 + 1u ? bl - ((bl ^ b0) & 1u) : b0;
    for (uint32_t b = b0 + blockIdx.x; b <= bl; b = other) {
        if (blockIdx.x && b == other) return;
        const uint32_t first = max(S.pos, 32u * b), last = min(end, 32u * b + 32u);   // the call's rows
        const uint64_t buf = kv_tail_buf(c, S.seq, head, b, z);
        const bool full = (b + 1u) * 32u <= end, tail = b + 1u >= bl;
        const uint32_t from = full || last - first > kKvFew ? 32u * b : first;   // rows that matter
        KvTile<NT> T;
        const float* old = c.tail + buf * 32u * c.hdp;
#pragma unroll
        for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
            uint32_t t, d;
            kv_unit<NT>(k, t, d);
            const uint32_t p = min(max(32u * b + t, from), last - 1u), dd = min(d, c.hd - 4u);
            T.v[k] = *reinterpret_cast<const f4*>(p < S.pos ? old + (p & 31u) * c.hdp + dd : x + static_cast<uint64_t>(p - S.pos) * A.stride + dd);
            if (d >= c.hd) T.v[k] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        kv_row_max<NT>(T, rowmax);   // (its barriers come after every read of the tail)
        if (full) kv_close_block<NT, false>(c, T, rowmax, kv_block(c, S.seq, head, b), z, img);
        if (tail) kv_store_tail<NT, false>(c, T, rowmax, buf, z, first & 31u, last - 32u * b, img);
        if (b != b0 || other == b0) return;
        __syncthreads();   // the next round's row maxima and image
    }
}

// ---- read -----------------------------------------------------------------------------------

struct Kv8ReadArgs {
    Kv8Dev c;
    float* x[2];
    uint64_t stride;
    Kv8Seq s[kKvMaxSeqs];   // prefix: the sequence's length
};

// One workgroup per (block, head and K or V, sequence): the block's codes in 16-byte units into LDS, rows out of it.
// Memory's time: 2 sequences of 8192, 8 heads of 128, 36 us, 4.7 TB/s.
template <int NT>
__global__ void __launch_bounds__((KvTile<NT>::TH)) k_kv8_read(const Kv8ReadArgs A) {
#pragma clang fp contract(off)
    __shared__ __align__(16) uint8_t img[1024 * NT];
    const Kv8Dev& c = A.c;
    const Kv8Seq& S = A.s[blockIdx.z];
    const uint32_t head = blockIdx.y >> 1, z = blockIdx.y & 1u, tid = threadIdx.x;
    const uint32_t b = (S.pos >> 5) + blockIdx.x;
    if (S.n == 0u || b > (S.pos + S.n - 1u) >> 5) return;
    const bool closed = (b + 1u) * 32u <= S.prefix;
    float s = 0.0f;
    if (closed) {
        const uint64_t blk = kv_block(c, S.seq, head, b);
        const uint4* src = reinterpret_cast<const uint4*>(kv_codes(c, blk) + z * 32u * c.hdp);
        s = reinterpret_cast<const float*>(c.scales + blk)[z];
        for (uint32_t i = tid; i < 64u * NT; i += KvTile<NT>::TH) reinterpret_cast<uint4*>(img)[i] = src[i];
        __syncthreads();
    }
    const float* old = c.tail + kv_tail_buf(c, S.seq, head, b, z) * 32u * c.hdp;
#pragma unroll
    for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
        uint32_t t, d;
        kv_unit<NT>(k, t, d);
        const uint32_t p = 32u * b + t;
        if (d >= c.hd || p < S.pos || p - S.pos >= S.n) continue;
        f4 v;
        if (closed) {
            uint32_t w;
            if (z == 0u) w = *reinterpret_cast<const uint32_t*>(img + kv_k_at(t, d));
            else w = img[kv_v_at(t, d)] | img[kv_v_at(t, d + 1u)] << 8 | img[kv_v_at(t, d + 2u)] << 16 | img[kv_v_at(t, d + 3u)] << 24;
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) v[e] = s * (static_cast<float>((w >> (8u * e)) & 255u) - 128.0f);
        } else {
            v = *reinterpret_cast<const f4*>(old + t * c.hdp + d);
        }
        *reinterpret_cast<f4*>(A.x[z] + (static_cast<uint64_t>(S.row0) + (p - S.pos)) * A.stride + head * c.hd + d) = v;
    }
}

// ---- attention ------------------------------------------------------------------------------

// The blocks that the rows of a tile (positions pmin .. pmax) see: virtual block i is i for i < n_pre, else lo + i - n_pre.
struct KvSpan {
    uint32_t n_pre, lo, n;
};
__device__ __forceinline__ KvSpan kv_span(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t pmin, uint32_t pmax) {
    const uint32_t len = S.pos + S.n, pre = min(S.prefix, len);
    const uint32_t first = A.window && pmin + 1u > A.window ? pmin + 1u - A.window : 0u;
    KvSpan r;
    r.lo = first >> 5;
    r.n_pre = min((pre + 31u) >> 5, r.lo);
    r.n = r.n_pre + ((max(pmax + 1u, pre) + 31u) >> 5) - r.lo;
    return r;
}

// Biased bytes to halves: the byte under 0x64 is 1024 + q + 128, exactly, and 1152 comes off. (As the half's low bits alone, (q + 128)
// 2^-24, a key takes no subtraction, but 128 times the sum of the queries has to come off the scores: five times the error.
// Signs and magnitudes kept so that they are subnormals right away lose digits: the matrix cores drop the product of two
// subnormals, and the low parts of small weights are such, 1.7e-4 of the outputs at 8192 positions.)
__device__ __forceinline__ h8 kv_halves(uint32_t w0, uint32_t w1) {
    const h2 off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)) + off;
    const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)) + off;
    const h2 c = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)) + off;
    const h2 d = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)) + off;
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// tanh(x). Up to 1/2 in magnitude its odd polynomial of degree 11 (a least-squares fit, relative error 4e-10); above, by
// e^(-2|x|), at 1 ulp each of exponential and reciprocal. `some`: whether a lane is above, wave-uniform, so that the scores of most
// blocks, well below the cap, cost no exponential here.
__device__ __forceinline__ float kv_tanh(float x, bool some) {
    const float y = x * x;
    float r = x + x * y * (-0.33333327f + y * (0.13332961f + y * (-0.05389886f + y * (0.02129668f + y * -0.0066456f))));
    if (some) {
        const float a = fabsf(x), e = __builtin_amdgcn_exp2f(a * -2.885390082f);
        const float big = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
        r = a <= 0.5f ? r : copysignf(big, x);
    }
    return r;
}

#define KV_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0)

__device__ __forceinline__ float max_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Queries are the B operand of the transposed scores (lane l: row l % 16, dims 32 s + 8 (l / 16) + e), each row scaled by a power
// of two to below 2^14 and split into halves: units (s, high or low) of 64 lanes x 16 bytes. One tile of 16 rows stays in
// registers; of more, which all waves of a workgroup share, they stay in LDS, so that the outputs' registers leave
// room for two waves a SIMD.
template <int NT>
struct KvQuery {
    h8 q[NT][2];
};
// Rows r0 .. r0 + 15 as they are; from them the queries and f, a score's factor but for its key's scale (log2 units without a cap).
template <int NT>
struct KvRows {
    f4 x[NT][2];
};
template <int NT>
__device__ __forceinline__ void kv_load_rows(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t kvh, uint32_t r0, KvRows<NT>& X) {
    const uint32_t lane = threadIdx.x & 63u, R = S.n * A.G, hd = A.c.hd;
    const uint32_t r = min(r0 + (lane & 15u), R - 1u), qi = r / A.G, h = kvh * A.G + (r - qi * A.G);
    const float* src = A.q + (static_cast<uint64_t>(S.row0) + qi) * A.q_stride + h * hd;
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j)
            X.x[s][j] = *reinterpret_cast<const f4*>(src + min(32u * s + 8u * (lane >> 4) + 4u * j, hd - 4u));
}
template <int NT, bool CAP>
__device__ __forceinline__ void kv_make_q(const Kv8AttnArgs& A, KvRows<NT>& X, KvQuery<NT>& Q, float& f) {
    const uint32_t lane = threadIdx.x & 63u;
    float m = 0.0f;
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j)
            if (32u * s + 8u * (lane >> 4) + 4u * j >= A.c.hd) X.x[s][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(X.x[s][j >> 2][j & 3]));
    m = max_xor32(max_xor16(m));
    const int ex = kv_exp(m, 14);
    const float sign = A.scale < 0.0f ? -1.0f : 1.0f;   // factors are not negative: the largest score is the largest product
    f = ldexpf(1.0f, -ex) * (fabsf(A.scale) * (CAP ? 1.0f : 1.4426950409f));
    const float up = ldexpf(sign, ex);
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            h2 a, b;
            kv_split2(X.x[s][j >> 2][j & 3] * up, X.x[s][j >> 2][(j & 3) + 1] * up, a, b);
            Q.q[s][0][j] = a[0], Q.q[s][0][j + 1] = a[1];
            Q.q[s][1][j] = b[0], Q.q[s][1][j + 1] = b[1];
        }
}
// What a wave holds of RT tiles of 16 rows (lane l: row l % 16 of each). The outputs are transposed too (dims 16 t + 4 (l / 16) + e), in
// units of 2^(eR - 9).
constexpr float kKvGrow = 6.0f;   // weights may pass 1 by 2^6 before the reference maximum follows
template <int NT, int RT>
struct KvWave {
    KvQuery<NT> q;    // RT == 1; else
    const h8* sq;     //   in LDS: [RT][NT][2][64], from this lane's place on
    f4 acc[RT][2 * NT];
    float f[RT];
    uint32_t p[RT];   // the rows' positions
    float m[RT], l[RT];
    int eR;           // 2^eR is above every value scale so far
    __device__ __forceinline__ h8 query(int k, int s, int part) const {
        if constexpr (RT == 1) return q.q[s][part];
        else return sq[((k * NT + s) * 2 + part) * 64];
    }
};
template <int NT, int RT>
__device__ __forceinline__ void kv_start(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t r0, KvWave<NT, RT>& W) {
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        W.p[k] = S.pos + min(r0 + 16u * k + (threadIdx.x & 15u), S.n * A.G - 1u) / A.G;
        W.m[k] = -INFINITY;
        W.l[k] = 0.0f;
#pragma unroll
        for (int t = 0; t < 2 * NT; ++t) W.acc[k][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    W.eR = kKvNoExp;
}

// A full block's codes in registers: lane l's 16 bytes of each 32 dims.
template <int NT>
struct KvRaw {
    uint4 w[NT];
};
template <int NT>
__device__ __forceinline__ void kv_load(const Kv8Dev& c, uint64_t blk, uint32_t z, KvRaw<NT>& r) {
    const uint4* src = reinterpret_cast<const uint4*>(kv_codes(c, blk) + z * 32u * c.hdp) + (threadIdx.x & 63u);
#pragma unroll
    for (int t = 0; t < NT; ++t) r.w[t] = src[64 * t];
}

// Products of 32 tokens' keys with the queries: s[k][half], lane l: row l % 16, tokens 16 half + 4 (l / 16) + e. Queries in
// LDS are read kAhead steps (a step: the high or low halves of 32 dims) before their products.
template <int NT, int RT>
__device__ __forceinline__ void kv_scores(const KvRaw<NT>& K, const KvWave<NT, RT>& W, f4 (&s)[RT][2]) {
    constexpr int kAhead = RT == 1 ? 0 : RT == 2 ? 2 : 1;
    h8 q[kAhead + 1][RT];
#pragma unroll
    for (int k = 0; k < RT; ++k) s[k][0] = s[k][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int k = 0; k < RT; ++k) q[i][k] = W.query(k, i >> 1, i & 1);
    h8 a0, a1;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
        const int j = i + kAhead;
        if (j < 2 * NT)
#pragma unroll
            for (int k = 0; k < RT; ++k) q[j % (kAhead + 1)][k] = W.query(k, j >> 1, j & 1);
        if (RT > 1) __builtin_amdgcn_sched_barrier(0);
        if ((i & 1) == 0) {
            a0 = kv_halves(K.w[i >> 1].x, K.w[i >> 1].y);
            a1 = kv_halves(K.w[i >> 1].z, K.w[i >> 1].w);
        }
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            s[k][0] = KV_MFMA(a0, q[i % (kAhead + 1)][k], s[k][0]);
            s[k][1] = KV_MFMA(a1, q[i % (kAhead + 1)][k], s[k][1]);
        }
    }
}
// The same of the open block, from the tail's pairs.
template <int NT, int RT>
__device__ __forceinline__ void kv_scores_open(const Kv8Dev& c, uint64_t buf, const KvWave<NT, RT>& W, f4 (&s)[RT][2]) {
    const h8* hi = reinterpret_cast<const h8*>(c.pairs + buf * 64u * c.hdp) + (threadIdx.x & 63u);
    const h8* lo = hi + 4u * c.hdp;
#pragma unroll
    for (int k = 0; k < RT; ++k) s[k][0] = s[k][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const h8 a = hi[64 * (2 * t + half)], b = lo[64 * (2 * t + half)];
#pragma unroll
            for (int k = 0; k < RT; ++k) {
                const h8 q = W.query(k, t, 0);
                s[k][half] = KV_MFMA(a, q, s[k][half]);
                s[k][half] = KV_MFMA(b, q, s[k][half]);
                s[k][half] = KV_MFMA(a, W.query(k, t, 1), s[k][half]);
            }
        }
}

// Tokens of a lane's eight scores.
__device__ __forceinline__ uint32_t kv_token(uint32_t e) { return 4u * ((threadIdx.x & 63u) >> 4) + (e & 3u) + 16u * (e >> 2); }

// One block's scores to weights: log2 units, running reference maximum and sum, the weights times the values' scale as
// pairs of halves. ks / vs: the block's scales, or (OPEN, always masked) those of the lane's tokens. dump: where the row's scores
// go. Nothing but short pieces is under a condition: what is not seen becomes -infinity, which a factor above zero
// leaves alone, and a weight of 0; a scale that is NaN becomes a NaN in the sums of the rows that see its block.
template <int NT, int RT, bool CAP, bool OPEN>
__device__ __forceinline__ void kv_soft(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t b, bool masked, f4 (&s)[RT][2],
                                        const float* ks, const float* vs, KvWave<NT, RT>& W, h8 (&ph)[RT], h8 (&pl)[RT], float* dump) {
    constexpr bool direct = CAP || OPEN;   // s becomes the score itself; else it is s F
    float F[RT];
#pragma unroll
    for (int k = 0; k < RT; ++k) F[k] = OPEN ? W.f[k] : fmaxf(W.f[k] * ks[0], 1e-36f);
    if constexpr (OPEN) {
#pragma unroll
        for (int k = 0; k < RT; ++k)
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) s[k][e >> 2][e & 3u] *= F[k] * ks[e];
    }
    if constexpr (CAP) {
        const float rc = 1.0f / A.cap;
        bool some = false;
#pragma unroll
        for (int k = 0; k < RT; ++k)
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                const float x = s[k][e >> 2][e & 3u] * (OPEN ? rc : F[k] * rc);
                s[k][e >> 2][e & 3u] = x;
                some |= fabsf(x) > 0.5f;
            }
        some = __any(some);
#pragma unroll
        for (int k = 0; k < RT; ++k)
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) s[k][e >> 2][e & 3u] = A.cap * 1.4426950409f * kv_tanh(s[k][e >> 2][e & 3u], some);
    }
    if (masked) {
        const uint32_t len = S.pos + S.n;
#pragma unroll
        for (int k = 0; k < RT; ++k)
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                const uint32_t j = 32u * b + kv_token(e);
                const bool y = j < len && (j < S.prefix || (j <= W.p[k] && (!A.window || W.p[k] - j < A.window)));
                s[k][e >> 2][e & 3u] = y ? s[k][e >> 2][e & 3u] : -INFINITY;
            }
    }
    float top[RT], v = OPEN ? 0.0f : vs[0];
    if constexpr (OPEN) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v = fmaxf(v, vs[e]);
        v = max_xor32(max_xor16(v));
    } else if (!(ks[0] < INFINITY) || !(v < INFINITY)) {   // the block stands for NaN
        v = 0.0f;
#pragma unroll
        for (int k = 0; k < RT; ++k)
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) W.l[k] = s[k][e >> 2][e & 3u] != -INFINITY ? __uint_as_float(0x7fc00000u) : W.l[k];
    }
    const int ev = v > 0.0f ? __builtin_amdgcn_frexp_expf(v) : kKvNoExp;
    bool grow = ev > W.eR;
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        float t = -INFINITY;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) t = fmaxf(t, s[k][e >> 2][e & 3u]);
        t = max_xor32(max_xor16(t));
        top[k] = direct ? t : t * F[k];
        grow |= top[k] > W.m[k] + kKvGrow;
    }
    if (__any(grow)) {
        const int eR = max(W.eR, ev);
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            const float m = top[k] > W.m[k] + kKvGrow ? top[k] : W.m[k];
            const float beta = m == W.m[k] ? 1.0f : __builtin_amdgcn_exp2f(W.m[k] - m);
            const float alpha = ldexpf(beta, W.eR - eR);
            W.m[k] = m;
            W.l[k] *= beta;
#pragma unroll
            for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) W.acc[k][t][e] *= alpha;
        }
        W.eR = eR;
    }
    const int up = W.eR == kKvNoExp ? 0 : 9 - W.eR;
    const float vf = ldexpf(v, up);
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        const float ref = W.m[k] == -INFINITY ? 0.0f : W.m[k];
        float p[8];
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
            const float x = s[k][e >> 2][e & 3u];
            p[e] = __builtin_amdgcn_exp2f(direct ? x - ref : __builtin_fmaf(x, F[k], -ref));
            W.l[k] += p[e];
            if constexpr (OPEN) p[e] = x == -INFINITY ? 0.0f : p[e] * ldexpf(vs[e], up);   // (0 times a factor that is NaN)
            else p[e] *= vf;
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            h2 a, d;
            kv_split2(p[e], p[e + 1], a, d);
            ph[k][e] = a[0], ph[k][e + 1] = a[1];
            pl[k][e] = d[0], pl[k][e + 1] = d[1];
        }
    }
    if (dump) {
        f4 x[2];
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) x[e >> 2][e & 3u] = s[0][e >> 2][e & 3u] * (direct ? 1.0f : F[0]);
        *reinterpret_cast<f4*>(dump) = x[0];
        *reinterpret_cast<f4*>(dump + 16) = x[1];
    }
}

template <int NT, int RT>
__device__ __forceinline__ void kv_values(const KvRaw<NT>& V, const h8 (&ph)[RT], const h8 (&pl)[RT], KvWave<NT, RT>& W) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const h8 a0 = kv_halves(V.w[t].x, V.w[t].y), a1 = kv_halves(V.w[t].z, V.w[t].w);
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            W.acc[k][2 * t] = KV_MFMA(a0, ph[k], W.acc[k][2 * t]);
            W.acc[k][2 * t + 1] = KV_MFMA(a1, ph[k], W.acc[k][2 * t + 1]);
        }
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            W.acc[k][2 * t] = KV_MFMA(a0, pl[k], W.acc[k][2 * t]);
            W.acc[k][2 * t + 1] = KV_MFMA(a1, pl[k], W.acc[k][2 * t + 1]);
        }
    }
}

// The open block of a sequence (its last): live rows of the tail; what lies past them is whatever the memory held.
template <int NT, int RT, bool CAP>
__device__ __forceinline__ void kv_open(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t kvh, uint32_t b, KvWave<NT, RT>& W, float* dump) {
    const Kv8Dev& c = A.c;
    const uint32_t lane = threadIdx.x & 63u, live = S.pos + S.n - 32u * b;
    const uint64_t kb = kv_tail_buf(c, S.seq, kvh, b, 0u), vb = kb + 1u;
    float ks[8], vs[8];
    uint32_t keep[4];   // of the values' operand: halves 2 i and 2 i + 1
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e) {
        const bool y = kv_token(e) < live;
        ks[e] = c.factor[kb * 32u + kv_token(e)];
        vs[e] = c.factor[vb * 32u + kv_token(e)];
        ks[e] = y ? ks[e] : 0.0f;
        vs[e] = y ? vs[e] : 0.0f;
        keep[e >> 1] = (e & 1u ? keep[e >> 1] : 0u) | (y ? 0xffffu << (16u * (e & 1u)) : 0u);
    }
    f4 s[RT][2];
    h8 ph[RT], pl[RT];
    kv_scores_open<NT, RT>(c, kb, W, s);
    kv_soft<NT, RT, CAP, true>(A, S, b, true, s, ks, vs, W, ph, pl, dump);
    const uint4* hi = reinterpret_cast<const uint4*>(c.pairs + vb * 64u * c.hdp) + lane;
    const uint4* lo = hi + 4u * c.hdp;
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t) {
        uint4 x = hi[64 * t], y = lo[64 * t];
        x.x &= keep[0], x.y &= keep[1], x.z &= keep[2], x.w &= keep[3];
        y.x &= keep[0], y.y &= keep[1], y.z &= keep[2], y.w &= keep[3];
        const h8 a = __builtin_bit_cast(h8, x), d = __builtin_bit_cast(h8, y);
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            W.acc[k][t] = KV_MFMA(a, ph[k], W.acc[k][t]);
            W.acc[k][t] = KV_MFMA(a, pl[k], W.acc[k][t]);
            W.acc[k][t] = KV_MFMA(d, ph[k], W.acc[k][t]);
        }
    }
}

// The same by a workgroup's four waves together (one tile of rows): a wave's quarter of the dims goes into its part of the
// scores, which meet in LDS (xch: [4][2][64] f4), and out of its quarter of the values, into its own sums; `owner` counts the weights.
// By one wave alone, with 64 KB to read, it was half of a step's time at short histories.
template <int NT, bool CAP>
__device__ __forceinline__ void kv_open_all(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t kvh, uint32_t b, KvWave<NT, 1>& W, bool owner,
                                            f4* xch, float* dump) {
    constexpr int NK = (NT + 3) / 4, NV = (2 * NT + 3) / 4;
    const Kv8Dev& c = A.c;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), live = S.pos + S.n - 32u * b;
    const uint64_t kb = kv_tail_buf(c, S.seq, kvh, b, 0u), vb = kb + 1u;
    const h8* kp = reinterpret_cast<const h8*>(c.pairs + kb * 64u * c.hdp) + lane;
    const uint4* vp = reinterpret_cast<const uint4*>(c.pairs + vb * 64u * c.hdp) + lane;
    h8 k[NK][2][2];
    uint4 v[NV][2];
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (uint32_t part = 0; part < 2u; ++part)
                k[i][half][part] = kp[64u * (2u * min(wave + 4u * i, NT - 1u) + half) + part * 4u * c.hdp];
    float ks[8], vs[8];
    uint32_t keep[4];   // of the values' operand: halves 2 i and 2 i + 1
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e) {
        const bool y = kv_token(e) < live;
        ks[e] = c.factor[kb * 32u + kv_token(e)];
        vs[e] = c.factor[vb * 32u + kv_token(e)];
        ks[e] = y ? ks[e] : 0.0f;
        vs[e] = y ? vs[e] : 0.0f;
        keep[e >> 1] = (e & 1u ? keep[e >> 1] : 0u) | (y ? 0xffffu << (16u * (e & 1u)) : 0u);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (uint32_t part = 0; part < 2u; ++part) v[i][part] = vp[64u * min(wave + 4u * i, 2u * NT - 1u) + part * 4u * c.hdp];
    __builtin_amdgcn_sched_barrier(0);
    f4 s[1][2] = {{{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}}};
#pragma unroll
    for (int t = 0; t < NT; ++t)
        if (static_cast<uint32_t>(t & 3) == wave)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                s[0][half] = KV_MFMA(k[t >> 2][half][0], W.query(0, t, 0), s[0][half]);
                s[0][half] = KV_MFMA(k[t >> 2][half][1], W.query(0, t, 0), s[0][half]);
                s[0][half] = KV_MFMA(k[t >> 2][half][0], W.query(0, t, 1), s[0][half]);
            }
#pragma unroll
    for (int half = 0; half < 2; ++half) xch[(wave * 2u + half) * 64u + lane] = s[0][half];
    __syncthreads();
#pragma unroll
    for (uint32_t half = 0; half < 2u; ++half)
        s[0][half] = (xch[half * 64u + lane] + xch[(2u + half) * 64u + lane]) + (xch[(4u + half) * 64u + lane] + xch[(6u + half) * 64u + lane]);
    h8 ph[1], pl[1];
    const float before = W.l[0];
    const float m0 = W.m[0];
    kv_soft<NT, 1, CAP, true>(A, S, b, true, s, ks, vs, W, ph, pl, owner ? dump : nullptr);
    if (!owner) W.l[0] = before * (W.m[0] == m0 ? 1.0f : __builtin_amdgcn_exp2f(m0 - W.m[0]));
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t)
        if (static_cast<uint32_t>(t & 3) == wave) {
            uint4 x = v[t >> 2][0], y = v[t >> 2][1];
            x.x &= keep[0], x.y &= keep[1], x.z &= keep[2], x.w &= keep[3];
            y.x &= keep[0], y.y &= keep[1], y.z &= keep[2], y.w &= keep[3];
            const h8 a = __builtin_bit_cast(h8, x), d = __builtin_bit_cast(h8, y);
            W.acc[0][t] = KV_MFMA(a, ph[0], W.acc[0][t]);
            W.acc[0][t] = KV_MFMA(a, pl[0], W.acc[0][t]);
            W.acc[0][t] = KV_MFMA(d, ph[0], W.acc[0][t]);
        }
    __syncthreads();   // xch is the waves' meeting place too
}

// Whether some row at positions pmin .. pmax does not see all of the full block b.
__device__ __forceinline__ bool kv_masked(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t b, uint32_t pmin, uint32_t pmax) {
    const uint32_t last = 32u * b + 31u;
    return last >= S.prefix && (last > pmin || (A.window && pmax - 32u * b >= A.window));
}

// Four outputs of (row, head), and what is left to say of it.
__device__ __forceinline__ void kv_give(const Kv8AttnArgs& A, uint32_t row, uint32_t h, uint32_t d, f4 v) {
    const uint32_t col = h * A.c.hd + d;
    if (!A.o.gm) {
        *reinterpret_cast<f4*>(A.o.rows + row * A.o.stride + col) = v;
        return;
    }
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const uint64_t o = gm_off(row, col, A.o.gm_nkb);
    h4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        _Float16 a, b;
        gm_split(v[e], a, b);
        hi[e] = a;
        lo[e] = b;
    }
    *reinterpret_cast<h4*>(A.o.gm + o) = hi;
    *reinterpret_cast<h4*>(A.o.gm + o + kGmLo) = lo;
}
__device__ __forceinline__ void kv_row_done(const Kv8AttnArgs& A, uint32_t row, uint32_t h, float M, float L) {
    if (A.stats) A.stats[static_cast<uint64_t>(row) * A.heads + h] = make_float2(M, 1.0f / L);
    if (A.o.nonfinite && (!(L > 0.0f) || !__builtin_isfinite(L))) atomicMin(A.o.nonfinite, A.o.code);
}

// The virtual blocks i0, i0 + 4, ... below i1 of a wave's rows (span sp). The keys of the next block are loaded while
// this one's weights are computed, its values while the next scores are (several tiles, whose blocks come out of L2: after the
// scores, which leaves those registers to the queries); the first block's before start() makes the queries.
template <int NT, int RT, bool CAP, class Start>
__device__ __forceinline__ void kv_run(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t kvh, const KvSpan& sp, uint32_t pmin, uint32_t pmax,
                                       uint32_t i0, uint32_t i1, KvWave<NT, RT>& W, f4* xch, float* dump, Start start) {
    const Kv8Dev& c = A.c;
    auto block = [&](uint32_t i) { return i < sp.n_pre ? i : sp.lo + (i - sp.n_pre); };
    const uint32_t last = block(sp.n - 1u);
    const bool open = (last + 1u) * 32u > S.pos + S.n;   // the last virtual block
    const uint32_t e1 = open ? min(i1, sp.n - 1u) : i1;
    KvRaw<NT> K, V;
    float2 sc = {0.0f, 0.0f};
    const bool any = i0 < e1;
    // (a wave without a full block loads one all the same, the first of the region, and uses nothing of it)
    uint64_t blk = kv_block(c, S.seq, kvh, any ? block(i0) : 0u);
    kv_load<NT>(c, blk, 0u, K);
    if (RT == 1) kv_load<NT>(c, blk, 1u, V);
    sc = c.scales[blk];
    __builtin_amdgcn_sched_barrier(0);
    start();
    uint32_t i = i0;
    for (; i < e1; i += 4u) {
        const uint32_t b = block(i);
        f4 s[RT][2];
        kv_scores<NT, RT>(K, W, s);
        if (RT > 1) kv_load<NT>(c, blk, 1u, V);
        // (the last block's "next" is itself, again in cache: with no branch, a wait counts the loads it is for alone)
        blk = kv_block(c, S.seq, kvh, block(i + 4u < e1 ? i + 4u : i));
        kv_load<NT>(c, blk, 0u, K);
        const float2 cur = sc;
        sc = c.scales[blk];
        __builtin_amdgcn_sched_barrier(0);   // the loads are issued here, and not next to their use
        h8 ph[RT], pl[RT];
        kv_soft<NT, RT, CAP, false>(A, S, b, kv_masked(A, S, b, pmin, pmax), s, &cur.x, &cur.y, W, ph, pl,
                                    dump ? dump + 32u * (i - i0) : nullptr);
        kv_values<NT, RT>(V, ph, pl, W);
        if (RT == 1) kv_load<NT>(c, blk, 1u, V);
        __builtin_amdgcn_sched_barrier(0);
    }
    const bool mine = open && i == sp.n - 1u && i < i1;
    float* const to = dump ? dump + 32u * (i - i0) : nullptr;
    if constexpr (RT == 1) {
        if (open && i1 == sp.n) kv_open_all<NT, CAP>(A, S, kvh, last, W, mine, xch, to);   // all waves of the workgroup
    } else if (mine) {
        kv_open<NT, RT, CAP>(A, S, kvh, last, W, to);
    }
}

// One workgroup per (split of a unit's blocks, head, sequence), its waves taking every fourth block and meeting in LDS, eight rows
// at a time. A unit is 16 RT rows: 16 for single tokens (memory's time: two workgroups a CU hold 16 KB a wave in
// flight); more for prompts, where a block's codes become halves once for all of a wave's rows. A sequence's units come the
// longest first, so that what is left at the end is short (or, where all run at once, so that a CU's two are as long
// together as any other's: a prompt of 4096 rows 95 us, in descending order 101, interleaved 113); the (head, sequence)s side by
// side: eight of them or a multiple have an XCD's L2 each.
// Measured: 64 sequences of up to 8 K, one head of 256: 39 us, 3.5 TB/s of codes; 2 of 128 K, 8 heads of 128: 105 us, 4.4 TB/s;
// a prompt of 4096 rows, 4 heads of 256: 95 us. Prompts are the vector unit's (exponentials, maxima, halves of the weights), tokens memory's.
template <int NT, int RT, bool CAP>
__global__ void __launch_bounds__(kKvThreads, 2) k_kv8_attn(const Kv8AttnArgs A) {
    constexpr uint32_t HDP = 32u * NT, C4 = HDP / 4u;
    // units of 16 bytes: the waves' outputs; the prompts' queries, or the waves' shares of the open block's scores
    constexpr uint32_t kMeet = 4u * 8u * C4, kOther = RT > 1 ? RT * NT * 128u : 4u * 2u * 64u;
    __shared__ __align__(16) f4 s_buf[kMeet > kOther ? kMeet : kOther];
    __shared__ float s_m[4][16 * RT], s_l[4][16 * RT], s_f[16 * RT];
    f4* const s_acc = s_buf;   // [4][8 C4], after the queries' last use
    kv_ask(A);
    const uint32_t pairs = A.nseq * A.c.kvh, pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
    const uint32_t kvh = pair % A.c.kvh, split = rest % A.splits;
    const Kv8Seq& S = A.s[pair / A.c.kvh];
    kv_ask(S);
    const uint32_t R = S.n * A.G, units = (R + 16u * RT - 1u) / (16u * RT), at = rest / A.splits;
    if (at >= units || split >= S.splits) return;
    const uint32_t unit = A.fold && at >= units / 2u ? at - units / 2u : units - 1u - at;
    const uint32_t r0 = 16u * RT * unit, rows = min(16u * RT, R - r0);
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, m16 = lane & 15u;
    const uint32_t pmin = S.pos + r0 / A.G, pmax = S.pos + (r0 + rows - 1u) / A.G;
    const KvSpan sp = kv_span(A, S, pmin, pmax);
    const uint32_t i0 = split * A.per, i1 = min(sp.n, i0 + A.per);
    if (i0 >= i1) return;
    const uint64_t place = static_cast<uint64_t>(S.part0) + (unit * A.c.kvh + kvh) * S.splits + split;
    float* dump = nullptr;   // this lane's row of the unit's scores
    if (RT == 1 && A.scores && m16 < rows) dump = A.scores + (place * A.lines + m16) * 32u * A.per + 32u * wave + 4u * g;
    KvWave<NT, RT> W;
    KvRows<NT> X;
    if (RT == 1 || wave < RT) kv_load_rows<NT>(A, S, kvh, r0 + (RT == 1 ? 0u : 16u * wave), X);   // (several tiles: one a wave)
    __builtin_amdgcn_sched_barrier(0);
    kv_run<NT, RT, CAP>(A, S, kvh, sp, pmin, pmax, i0 + wave, i1, W, s_buf, dump, [&]() {
        if constexpr (RT == 1) {
            kv_make_q<NT, CAP>(A, X, W.q, W.f[0]);
        } else {
            h8* sq = reinterpret_cast<h8*>(s_buf) + lane;
            if (wave < RT) {
                KvQuery<NT> Q;
                float f;
                kv_make_q<NT, CAP>(A, X, Q, f);
#pragma unroll
                for (int s = 0; s < NT; ++s)
#pragma unroll
                    for (int part = 0; part < 2; ++part) sq[((wave * NT + s) * 2u + part) * 64u] = Q.q[s][part];
                if (g == 0u) s_f[16u * wave + m16] = f;
            }
            __syncthreads();
            W.sq = sq;
#pragma unroll
            for (int k = 0; k < RT; ++k) W.f[k] = s_f[16 * k + m16];
        }
        kv_start<NT, RT>(A, S, r0, W);
    });
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        const float l = add_xor32(add_xor16(W.l[k]));
        if (g == 0u) {
            s_m[wave][16 * k + m16] = W.m[k];
            s_l[wave][16 * k + m16] = l;
        }
    }
    __syncthreads();
    const bool only = S.splits == 1u;
#pragma unroll
    for (int q = 0; q < 2 * RT; ++q) {   // rows 8 q .. 8 q + 7
        if (8u * q >= rows) break;
        if (q) __syncthreads();
        if (m16 >> 3 == (q & 1u)) {
            const uint32_t k = q >> 1, row = 16u * k + m16;
            const float M = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
            const float mine = __builtin_amdgcn_exp2f(W.m[k] - (M == -INFINITY ? 0.0f : M));
#pragma unroll
            for (int t = 0; t < 2 * NT; ++t) {
                f4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = ldexpf(W.acc[k][t][e], W.eR - 9) * mine;
                s_acc[(wave * 8u + (m16 & 7u)) * C4 + ((4u * t + g) ^ (m16 & 7u))] = v;   // (rows spread over the banks)
            }
        }
        __syncthreads();
        for (uint32_t u = threadIdx.x; u < min(8u, rows - 8u * q) * C4; u += kKvThreads) {
            const uint32_t rr = u / C4, c4 = u - rr * C4, row = 8u * q + rr, at4 = rr * C4 + (c4 ^ rr);
            const f4 v = (s_acc[at4] + s_acc[8u * C4 + at4]) + (s_acc[16u * C4 + at4] + s_acc[24u * C4 + at4]);
            const float m = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
            const float rf = m == -INFINITY ? 0.0f : m;
            float L = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) L += s_l[w][row] * __builtin_amdgcn_exp2f(s_m[w][row] - rf);
            if (only) {
                const uint32_t r = r0 + row, qi = r / A.G, h = kvh * A.G + (r - qi * A.G);
                if (4u * c4 < A.c.hd) kv_give(A, S.row0 + qi, h, 4u * c4, v * (1.0f / L));
                if (c4 == 0u) kv_row_done(A, S.row0 + qi, h, m, L);
            } else {
                *reinterpret_cast<f4*>(A.part + (place * A.lines + row) * HDP + 4u * c4) = v;
            }
            if (c4 == 0u && (!only || A.scores)) A.part_ml[place * A.lines + row] = make_float2(m, L);
        }
    }
}

// The splits of a row put together, one workgroup per (row, head, sequence): four-dim columns times groups of splits, which
// meet in LDS. With scores (single tokens): workgroups past the rows take 256 positions each, and add up their weights.
// 4 to 6 us, a launch's latencies.
__global__ void __launch_bounds__(kKvThreads) k_kv8_join(const Kv8AttnArgs A) {
    __shared__ f4 s_o[kKvThreads];
    __shared__ float s_l[kKvThreads];
    __shared__ float s_ref[64], s_inv[64];
    const Kv8Seq& S = A.s[blockIdx.z];
    const Kv8Dev& c = A.c;
    const uint32_t kvh = blockIdx.y, R = S.n * A.G, U = A.unit, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    kv_ask(A);
    kv_ask(S);
    const uint32_t join_rows = A.splits > 1u ? A.rows_most : 0u;
    if (blockIdx.x < join_rows) {
        const uint32_t r = blockIdx.x, unit = r / U, rr = r - unit * U;
        if (r >= R) return;
        const KvSpan sp = kv_span(A, S, S.pos + unit * U / A.G, S.pos + min(unit * U + U - 1u, R - 1u) / A.G);
        const uint32_t n = (sp.n + A.per - 1u) / A.per;
        if (S.splits == 1u) return;   // written by the only split
        const uint64_t p0 = static_cast<uint64_t>(S.part0) + (unit * c.kvh + kvh) * S.splits;
        float M = -INFINITY;
        for (uint32_t k = lane; k < n; k += 64u) M = fmaxf(M, A.part_ml[(p0 + k) * A.lines + rr].x);
        M = wave_red_max(M);
        const float ref = M == -INFINITY ? 0.0f : M;
        const uint32_t hd4 = c.hd >> 2, groups = kKvThreads / hd4, grp = tid / hd4, d = (tid - grp * hd4) * 4u;
        f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        float L = 0.0f;
        if (grp < groups)
            for (uint32_t k = grp; k < n; k += groups) {
                const float2 ml = A.part_ml[(p0 + k) * A.lines + rr];
                const float w = __builtin_amdgcn_exp2f(ml.x - ref);
                L += w * ml.y;
                o += w * *reinterpret_cast<const f4*>(A.part + ((p0 + k) * A.lines + rr) * c.hdp + d);
            }
        s_o[tid] = o;
        s_l[tid] = L;
        __syncthreads();
        if (tid >= hd4) return;
        for (uint32_t k = 1; k < groups; ++k) {
            o += s_o[tid + k * hd4];
            L += s_l[tid + k * hd4];
        }
        const uint32_t qi = r / A.G, h = kvh * A.G + (r - qi * A.G);
        kv_give(A, S.row0 + qi, h, d, o / L);
        if (tid == 0u) kv_row_done(A, S.row0 + qi, h, M, L);
        return;
    }
    const uint32_t j = (blockIdx.x - join_rows) * kKvThreads + tid, len = S.pos + S.n;
    if (S.n == 0u || j - tid >= len) return;
    float w = 0.0f;
    for (uint32_t r0 = 0; r0 < R; r0 += 16u) {
        const uint32_t unit = r0 / 16u, rows = min(16u, R - r0), pmin = S.pos + r0 / A.G, pmax = S.pos + (r0 + rows - 1u) / A.G;
        const KvSpan sp = kv_span(A, S, pmin, pmax);
        const uint64_t p0 = static_cast<uint64_t>(S.part0) + (unit * c.kvh + kvh) * S.splits;
        const uint32_t n = (sp.n + A.per - 1u) / A.per;
        __syncthreads();
        for (uint32_t rr = wave; rr < rows; rr += kKvThreads / 64u) {
            float M = -INFINITY, L = 0.0f;
            for (uint32_t k = lane; k < n; k += 64u) M = fmaxf(M, A.part_ml[(p0 + k) * A.lines + rr].x);
            M = wave_red_max(M);
            const float ref = M == -INFINITY ? 0.0f : M;
            for (uint32_t k = lane; k < n; k += 64u) {
                const float2 ml = A.part_ml[(p0 + k) * A.lines + rr];
                L += ml.y * __builtin_amdgcn_exp2f(ml.x - ref);
            }
            L = wave_sum(L);
            if (lane == 0u) {
                s_ref[rr] = ref;
                s_inv[rr] = 1.0f / L;
            }
        }
        __syncthreads();
        // position j's virtual block: in the prefix, or from lo on
        const uint32_t b = j >> 5, i = b < sp.n_pre ? b : b - sp.lo + sp.n_pre;
        if (j >= len || (b >= sp.n_pre && b < sp.lo) || i >= sp.n) continue;
        const uint32_t k = i / A.per;
        const float* src = A.scores + (p0 + k) * A.lines * 32u * A.per + 32u * (i - k * A.per) + (j & 31u);
        for (uint32_t rr = 0; rr < rows; ++rr) w += __builtin_amdgcn_exp2f(src[rr * 32u * A.per] - s_ref[rr]) * s_inv[rr];
    }
    if (j >= len) return;
    const uint64_t at = (static_cast<uint64_t>(S.seq) * c.kvh + kvh) * A.max_ctx + j;
    A.w_out[at] = (A.w_in && j < S.pos ? A.w_in[at] : 0.0f) + w;
}

// Prompts' accumulated weights: one workgroup per (block of positions, head, sequence), its waves taking every eighth of the 16-row
// tiles that see the block; the scores once more, against the rows' final maxima and sums. A tile's rows are loaded while the
// one before is worked on. The blocks that the most rows see come first, and every other 256 of the workgroups the other way
// round, so that the longest meets the shortest on its CU: 3 prompts of 2048 positions, 8 heads of 64, take 72 us, in the grid's
// own order 129 us. What remains is the vector unit's (a row's halves are made once for every block), not memory's.
constexpr uint32_t kKvWeightWaves = 8, kKvCus = 256;
template <int NT, bool CAP>
__global__ void __launch_bounds__(64 * kKvWeightWaves, 2) k_kv8_weights(const Kv8AttnArgs A) {
    __shared__ float s_w[kKvWeightWaves][32];
    const uint32_t pairs = gridDim.y * gridDim.z, id = (blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    const uint32_t in = id % kKvCus, first = id - in, left = min(pairs * gridDim.x - first, kKvCus);
    const uint32_t nth = first + (first & kKvCus ? left - 1u - in : in), pair = nth % pairs;
    const Kv8Seq& S = A.s[pair / A.c.kvh];
    const Kv8Dev& c = A.c;
    const uint32_t kvh = pair % A.c.kvh, m16 = threadIdx.x & 15u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t len = S.pos + S.n, R = S.n * A.G, b = nth / pairs, p0 = 32u * b, p1 = p0 + 31u;
    if (S.n == 0u || p0 >= len) return;
    const bool open = p1 >= len;
    float w[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    float ks[8];
    KvRaw<NT> K;
    const uint64_t kb = kv_tail_buf(c, S.seq, kvh, b, 0u);
    if (open) {
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) ks[e] = c.factor[kb * 32u + kv_token(e)];
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) ks[e] = p0 + kv_token(e) < len ? ks[e] : 0.0f;
    } else {
        const uint64_t blk = kv_block(c, S.seq, kvh, b);
        kv_load<NT>(c, blk, 0u, K);
#pragma unroll
        for (int e = 0; e < 8; ++e) ks[e] = c.scales[blk].x;
    }
    // the tiles that see the block: all of a prefix's, else from its first position's query to the last within the window
    uint32_t t0 = 0u, t1 = (R + 15u) / 16u;
    if (p0 >= S.prefix) {
        if (p0 > S.pos) t0 = (p0 - S.pos) * A.G / 16u;
        if (A.window && p1 + A.window > p1) {   // (query p1 + window - 1)
            const uint32_t q1 = p1 + A.window;
            t1 = q1 <= S.pos ? 0u : min(t1, static_cast<uint32_t>((static_cast<uint64_t>(q1 - S.pos) * A.G + 15u) / 16u));
        }
    }
    KvRows<NT> X;
    float2 st_next;
    auto fetch = [&](uint32_t t) {
        kv_load_rows<NT>(A, S, kvh, 16u * t, X);
        const uint32_t r = min(16u * t + m16, R - 1u), qi = r / A.G;
        st_next = A.stats[(static_cast<uint64_t>(S.row0) + qi) * A.heads + kvh * A.G + (r - qi * A.G)];
    };
    uint32_t t = t0 + wave;
    if (t < t1) fetch(t);
    for (; t < t1; t += kKvWeightWaves) {
        const uint32_t r0 = 16u * t, r = r0 + m16, p = S.pos + min(r, R - 1u) / A.G;
        const uint32_t pmin = S.pos + r0 / A.G, pmax = S.pos + min(r0 + 15u, R - 1u) / A.G;
        KvWave<NT, 1> W;
        kv_make_q<NT, CAP>(A, X, W.q, W.f[0]);
        const float2 st = st_next;
        fetch(min(t + kKvWeightWaves, t1 - 1u));
        __builtin_amdgcn_sched_barrier(0);
        f4 s[1][2];
        if (open) kv_scores_open<NT, 1>(c, kb, W, s);
        else kv_scores<NT, 1>(K, W, s);
        const bool masked = open || r0 + 15u >= R || kv_masked(A, S, b, pmin, pmax);
        float x[8];
        bool some = false;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
            x[e] = s[0][e >> 2][e & 3u] * (W.f[0] * ks[e]);
            if constexpr (CAP) {
                x[e] *= 1.0f / A.cap;
                some |= fabsf(x[e]) > 0.5f;
            }
        }
        if constexpr (CAP) {
            some = __any(some);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = A.cap * 1.4426950409f * kv_tanh(x[e], some);
        }
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) x[e] = __builtin_amdgcn_exp2f(x[e] - st.x) * st.y;
        if (masked)
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                const uint32_t j = p0 + kv_token(e);
                const bool y = r < R && j < len && (j < S.prefix || (j <= p && (!A.window || p - j < A.window)));
                x[e] = y ? x[e] : 0.0f;
            }
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] += x[e];
    }
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e) {
        const float y = slot_sum<16>(w[e]);
        if (m16 == 0u) s_w[wave][kv_token(e)] = y;
    }
    __syncthreads();
    const uint32_t j = p0 + threadIdx.x;
    if (threadIdx.x >= 32u || j >= len) return;
    float y = 0.0f;
#pragma unroll
    for (uint32_t v = 0; v < kKvWeightWaves; ++v) y += s_w[v][threadIdx.x];
    const uint64_t at = (static_cast<uint64_t>(S.seq) * c.kvh + kvh) * A.max_ctx + j;
    A.w_out[at] = (A.w_in && j < S.pos ? A.w_in[at] : 0.0f) + y;
}

// ---- eviction -------------------------------------------------------------------------------

struct Kv8EvictArgs {
    Kv8Dev c;
    float* w;
    uint32_t* kept;
    uint64_t kept_stride;
    uint32_t max_ctx;
    vrt_kv8_move m[kKvMaxSeqs];
};

// Larger is better: NaN last, then -infinity, ..., equal floats (also the two zeros) alike.
__device__ __forceinline__ uint32_t kv_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr uint32_t kKvSelThreads = 1024, kKvSelWaves = kKvSelThreads / 64u, kKvBins = 2048;

// One workgroup per (head, move). The key of the last weight that stays, by histograms of its upper 11, middle 11 and lower 10
// bits; then every wave counts what stays of its run of positions, and writes it, of those with that key the first ones.
// Its CU's vector time, 21 instructions a weight over the five passes: 64 K weights 61 us, 8 K 18.
__global__ void __launch_bounds__(kKvSelThreads) k_kv8_select(const Kv8EvictArgs A) {
    __shared__ uint32_t hist[kKvBins], s_bin, s_left, s_gt[kKvSelWaves], s_eq[kKvSelWaves], s_sum[kKvSelWaves];
    const vrt_kv8_move& V = A.m[blockIdx.y];
    const uint32_t head = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const float* src = A.w + (static_cast<uint64_t>(V.src) * A.c.kvh + head) * A.max_ctx;
    float* dst = A.w + (static_cast<uint64_t>(V.dst) * A.c.kvh + head) * A.max_ctx;
    uint32_t* kept = A.kept + (static_cast<uint64_t>(blockIdx.y) * A.c.kvh + head) * A.kept_stride;
    const uint32_t old = V.len - V.recent, want = V.keep - V.recent;
    for (uint32_t i = tid; i < V.recent; i += kKvSelThreads) {
        kept[want + i] = old + i;
        dst[want + i] = src[old + i];
    }
    if (want == 0u) return;
    uint32_t thr = 0u, need = want;   // keys above thr stay, and `need` of those equal to it
    constexpr uint32_t kShift[3] = {21u, 10u, 0u}, kBits[3] = {11u, 11u, 10u};
    constexpr uint32_t kAhead = 16u;   // loads in flight
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const uint32_t shift = kShift[pass], mask = (1u << kBits[pass]) - 1u, high = pass == 0 ? 0u : 0xffffffffu << (shift + kBits[pass]);
        for (uint32_t i = tid; i < kKvBins; i += kKvSelThreads) hist[i] = 0u;
        __syncthreads();
        for (uint32_t i0 = tid; i0 - lane < old; i0 += kKvSelThreads * kAhead) {
            float w[kAhead];
#pragma unroll
            for (uint32_t k = 0; k < kAhead; ++k) w[k] = src[min(i0 + kKvSelThreads * k, old - 1u)];
#pragma unroll
            for (uint32_t k = 0; k < kAhead; ++k) {
                const uint32_t key = kv_key(w[k]), bin = (key >> shift) & mask;
                const bool in = i0 + kKvSelThreads * k < old && (key & high) == thr;
                const uint64_t all = __ballot(in);
                if (!all) continue;
                // (lanes of one bin add one after the other: where all have the same, as where weights are 0, one adds for them)
                const uint32_t first = __builtin_amdgcn_readlane(static_cast<int>(bin), __builtin_ctzll(all));
                if (__ballot(in && bin == first) == all) {
                    if (lane == static_cast<uint32_t>(__builtin_ctzll(all))) atomicAdd(&hist[first], static_cast<uint32_t>(__popcll(all)));
                } else if (in) {
                    atomicAdd(&hist[bin], 1u);
                }
            }
        }
        __syncthreads();
        // bins from the top: thread t has bins kKvBins - 1 - 2 t and the one below
        const uint32_t hi = hist[kKvBins - 1u - 2u * tid], lo = hist[kKvBins - 2u - 2u * tid];
        uint32_t run = hi + lo;   // inclusive sums over the wave's threads
#pragma unroll
        for (uint32_t o = 1; o < 64u; o <<= 1) {
            const uint32_t up = __shfl_up(static_cast<int>(run), o);
            run += lane >= o ? up : 0u;
        }
        if (lane == 63u) s_sum[wave] = run;
        __syncthreads();
        for (uint32_t v = 0; v < wave; ++v) run += s_sum[v];
        const uint32_t before = run - hi - lo;
        if (before < need && need <= run) {   // one thread: the bin that the last one falls into
            s_bin = before + hi >= need ? kKvBins - 1u - 2u * tid : kKvBins - 2u - 2u * tid;
            s_left = before + hi >= need ? need - before : need - before - hi;
        }
        __syncthreads();
        thr |= s_bin << shift;
        need = s_left;
    }
    const uint32_t run = ((old + kKvSelWaves - 1u) / kKvSelWaves + 63u) & ~63u, j0 = min(old, run * wave), j1 = min(old, j0 + run);
    uint32_t n_gt = 0u, n_eq = 0u;
    for (uint32_t j = j0; j < j1; j += 64u * kAhead) {
        float w[kAhead];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) w[k] = src[min(j + 64u * k + lane, j1 - 1u)];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            const uint32_t key = kv_key(w[k]);
            const bool in = j + 64u * k + lane < j1;
            n_gt += __popcll(__ballot(in && key > thr));
            n_eq += __popcll(__ballot(in && key == thr));
        }
    }
    if (lane == 0u) {
        s_gt[wave] = n_gt;
        s_eq[wave] = n_eq;
    }
    __syncthreads();
    uint32_t gt = 0u, eq = 0u;   // before this wave's run
    for (uint32_t v = 0; v < wave; ++v) {
        gt += s_gt[v];
        eq += s_eq[v];
    }
    const uint64_t below = (1ull << lane) - 1ull;
    for (uint32_t j = j0; j < j1; j += 64u * kAhead) {
        float w[kAhead];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) w[k] = src[min(j + 64u * k + lane, j1 - 1u)];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            const uint32_t key = kv_key(w[k]), i = j + 64u * k + lane;
            const uint64_t bg = __ballot(i < j1 && key > thr), be = __ballot(i < j1 && key == thr);
            const uint32_t my_eq = eq + __popcll(be & below), at = gt + __popcll(bg & below) + min(my_eq, need);
            if (i < j1 && (key > thr || (key == thr && my_eq < need))) {
                kept[at] = i;
                dst[at] = w[k];
            }
            gt += __popcll(bg);
            eq += __popcll(be);
        }
    }
}

// One workgroup per (block of the destination, head and K or V, move): the kept values of the source, into a block as
// the append makes it, or into the tail. Their codes go through LDS as rows of biased bytes. A key's row is 8-byte pieces of its
// block, 16 bytes from its neighbours': lanes take the pieces of different tokens. A value's is a byte of every 8: lanes take
// neighbouring dims, 16 bytes (two dims of eight tokens) a load.
// 2 sequences of 64 K, 8 heads of 128, to 8190: 55 us, 5 TB/s; 64 of 8 K, one of 256, to 2048: 100 us, half of it vector time.
template <int NT>
__global__ void __launch_bounds__((KvTile<NT>::TH)) k_kv8_gather(const Kv8EvictArgs A) {
#pragma clang fp contract(off)
    constexpr uint32_t kRow = 32u * NT + 8u, TH = KvTile<NT>::TH;
    __shared__ __align__(16) uint8_t img[2048 * NT];
    __shared__ __align__(16) uint8_t raw[32 * kRow];
    __shared__ uint32_t rowmax[32], s_p[32];
    __shared__ float s_s[32];
    const Kv8Dev& c = A.c;
    const vrt_kv8_move& V = A.m[blockIdx.z];
    const uint32_t head = blockIdx.y >> 1, z = blockIdx.y & 1u, tid = threadIdx.x;
    const uint32_t b = (blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3);   // an XCD has neighbours, which read the same blocks
    if (32u * b >= V.keep) return;
    const uint32_t* kept = A.kept + (static_cast<uint64_t>(blockIdx.z) * c.kvh + head) * A.kept_stride;
    const uint32_t n = min(32u, V.keep - 32u * b), full = V.len >> 5;   // full blocks of the source
    const uint64_t src0 = (static_cast<uint64_t>(V.src) * c.kvh + head) * c.nb;   // (a source is no ring)
    if (tid < 32u) {
        const uint32_t p = kept[32u * b + min(tid, n - 1u)];
        s_p[tid] = p;
        s_s[tid] = reinterpret_cast<const float*>(c.scales + src0 + min(p >> 5, full ? full - 1u : 0u))[z];
    }
    __syncthreads();
    const uint32_t top = full ? full - 1u : 0u;
    // (every load issued, at a position that is there, before the first is put down)
    if (z == 0u) {
        constexpr uint32_t kPer = (128u * NT + TH - 1u) / TH;
        uint2 u[kPer];
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {   // (8 dims, token)
            const uint32_t i = min(tid + TH * k, 128u * NT - 1u), t = i & 31u, q = i >> 5, p = s_p[t];
            const uint8_t* blk = kv_codes(c, src0 + min(p >> 5, top));
            u[k] = *reinterpret_cast<const uint2*>(blk + kv_k_at(p & 31u, 8u * q));
        }
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {
            const uint32_t i = min(tid + TH * k, 128u * NT - 1u), t = i & 31u, q = i >> 5;
            *reinterpret_cast<uint2*>(raw + t * kRow + 8u * q) = u[k];
        }
    } else {
        constexpr uint32_t kPer = 512u * NT / TH;
        uint4 u[kPer];
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {   // (token, dims 32 jj + m and 16 on)
            const uint32_t i = tid + TH * k, m = i & 15u, jj = (i >> 4) % NT, t = (i >> 4) / NT, p = s_p[t];
            const uint8_t* blk = kv_codes(c, src0 + min(p >> 5, top)) + 32u * c.hdp;
            u[k] = *reinterpret_cast<const uint4*>(blk + jj * 1024u + (((p >> 2) & 3u) * 16u + m) * 16u);
        }
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k) {
            const uint32_t i = tid + TH * k, m = i & 15u, jj = (i >> 4) % NT, t = (i >> 4) / NT, tok = s_p[t] & 31u;
            const uint32_t sh = 8u * (tok & 3u) + 2u * (tok & 16u);   // its byte of the dim's eight
            const uint64_t lo = static_cast<uint64_t>(u[k].y) << 32 | u[k].x, hi = static_cast<uint64_t>(u[k].w) << 32 | u[k].z;
            raw[t * kRow + 32u * jj + m] = static_cast<uint8_t>(lo >> sh);
            raw[t * kRow + 32u * jj + 16u + m] = static_cast<uint8_t>(hi >> sh);
        }
    }
    __syncthreads();
    KvTile<NT> T;
#pragma unroll
    for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
        uint32_t t, d;
        kv_unit<NT>(k, t, d);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(raw + t * kRow + d);
        const float f = t < n && d < c.hd ? s_s[t] : 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) T.v[k][e] = f * (static_cast<float>((w >> (8u * e)) & 255u) - 128.0f);
    }
    if (s_p[n - 1u] >> 5 >= full)   // the source's open block has some of them: the last ones
#pragma unroll
        for (uint32_t k = 0; k < KvTile<NT>::KU; ++k) {
            uint32_t t, d;
            kv_unit<NT>(k, t, d);
            const uint32_t p = s_p[t];
            if (t < n && d < c.hd && p >> 5 >= full)
                T.v[k] = *reinterpret_cast<const f4*>(c.tail + (kv_tail_buf(c, V.src, head, p >> 5, z) * 32u + (p & 31u)) * c.hdp + d);
        }
    kv_row_max<NT>(T, rowmax);
    if (n == 32u) kv_close_block<NT, true>(c, T, rowmax, kv_block(c, V.dst, head, b), z, img);
    if (b + 1u >= (V.keep - 1u) >> 5)   // the last block and the one before
        kv_store_tail<NT, true>(c, T, rowmax, kv_tail_buf(c, V.dst, head, b, z), z, 0u, n, img);
}

// ---- host -----------------------------------------------------------------------------------

namespace {

// The context's device, for the length of a call.
struct OnDevice {
    int before = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

uint64_t up256(uint64_t x) { return (x + 255u) & ~uint64_t(255); }

int check_cache(const vrt_kv8_cache* c, const char* who, Kv8Sizes* z) {
    VRT_REQUIRE(c, "%s: null cache", who);
    VRT_REQUIRE(c->max_seqs >= 1u && c->max_seqs <= 65535u, "%s: max_seqs must be 1..65535", who);
    VRT_REQUIRE(c->max_ctx >= 1u && c->max_ctx <= VRT_KV8_MAX_CTX, "%s: max_ctx must be 1..%u", who, VRT_KV8_MAX_CTX);
    VRT_REQUIRE(c->kv_heads >= 1u && c->kv_heads <= 1024u, "%s: kv_heads must be 1..1024", who);
    VRT_REQUIRE(c->head_dim >= 4u && c->head_dim <= 256u && c->head_dim % 4u == 0u,
                "%s: head_dim must be a multiple of 4, 4..256", who);
    *z = kv8_sizes(c->max_seqs, c->max_ctx, c->kv_heads, c->head_dim);
    return VRT_OK;
}

int cache_view(const vrt_kv8_cache* c, const char* who, Kv8Dev* d) {
    Kv8Sizes z;
    if (int rc = check_cache(c, who, &z)) return rc;
    VRT_REQUIRE(c->data && (reinterpret_cast<uintptr_t>(c->data) & 255u) == 0u, "%s: cache memory must be 256-byte aligned", who);
    VRT_REQUIRE(c->bytes >= z.total, "%s: cache memory is too small (%llu of %llu bytes)", who,
                static_cast<unsigned long long>(c->bytes), static_cast<unsigned long long>(z.total));
    *d = kv8_view(z, c->data, c->kv_heads, c->head_dim);
    return VRT_OK;
}

int check_rows(const vrt_kv8_cache* c, const vrt_kv8_rows* rows, uint32_t n, const char* who, Kv8Seq* s, uint64_t* total) {
    VRT_REQUIRE(rows, "%s: null rows", who);
    VRT_REQUIRE(n >= 1u && n <= kKvMaxSeqs, "%s: n_seqs must be 1..%u", who, kKvMaxSeqs);
    uint64_t row = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const vrt_kv8_rows& r = rows[i];
        VRT_REQUIRE(r.seq < c->max_seqs, "%s: sequence %u out of range", who, r.seq);
        for (uint32_t j = 0; j < i; ++j) VRT_REQUIRE(rows[j].seq != r.seq, "%s: sequence %u appears twice", who, r.seq);
        VRT_REQUIRE(r.pos <= VRT_KV8_MAX_CTX && r.n <= VRT_KV8_MAX_CTX - r.pos, "%s: positions past %u", who, VRT_KV8_MAX_CTX);
        s[i] = Kv8Seq{r.seq, r.pos, r.n, r.prefix, static_cast<uint32_t>(row), 0u, 0u};
        row += r.n;
    }
    VRT_REQUIRE(row <= 0x7fffffffu, "%s: too many rows", who);
    *total = row;
    return VRT_OK;
}

// Rows of `width` floats, 16-byte aligned.
int check_array(const void* p, uint64_t* stride, uint64_t width, const char* who, const char* what) {
    if (*stride == 0u) *stride = width;
    VRT_REQUIRE(p && (reinterpret_cast<uintptr_t>(p) & 15u) == 0u, "%s: %s must be 16-byte aligned device memory", who, what);
    VRT_REQUIRE(*stride >= width && *stride % 4u == 0u && *stride <= (1ull << 32), "%s: %s row stride must be a multiple of 4, at least %llu",
                who, what, static_cast<unsigned long long>(width));
    return VRT_OK;
}

// Blocks that a span of positions touches.
uint32_t touched(const Kv8Seq& s) { return s.n ? ((s.pos + s.n - 1u) >> 5) - (s.pos >> 5) + 1u : 0u; }

// The most blocks that a unit's rows of a sequence see.
uint32_t most_blocks(const Kv8Seq& s, uint32_t window, uint32_t unit) {
    const uint32_t len = s.pos + s.n, pre = std::min(s.prefix, len), all = (len + 31u) / 32u;
    if (!window) return all;
    // (its rows span that many positions at most)
    const uint64_t w = static_cast<uint64_t>((pre + 31u) / 32u) + (static_cast<uint64_t>(window) + unit + 31u) / 32u + 1u;
    return static_cast<uint32_t>(std::min<uint64_t>(all, w));
}

int attn_plan(const vrt_kv8_cache* c, const vrt_kv8_attn* at, const vrt_kv8_rows* rows, uint32_t n, bool scored, const char* who,
              Kv8AttnArgs& A, Kv8Plan* P, uint64_t* total) {
    Kv8Sizes z;
    if (int rc = check_cache(c, who, &z)) return rc;
    VRT_REQUIRE(at, "%s: null attention", who);
    VRT_REQUIRE(at->heads >= 1u && at->heads <= 65535u && at->heads % c->kv_heads == 0u,
                "%s: heads must be a multiple of kv_heads, at most 65535", who);
    VRT_REQUIRE(std::isfinite(at->scale), "%s: scale is not finite", who);
    // (its reciprocal times a score's factor is to stay a number)
    VRT_REQUIRE(std::isfinite(at->softcap) && (at->softcap == 0.0f || at->softcap >= 1e-6f),
                "%s: softcap must be finite, 0 or at least 1e-6", who);
    if (int rc = check_rows(c, rows, n, who, A.s, total)) return rc;
    A.heads = at->heads;
    A.G = at->heads / c->kv_heads;
    A.window = at->window;
    A.scale = at->scale;
    A.cap = at->softcap;
    A.max_ctx = c->max_ctx;
    uint64_t items = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const Kv8Seq& s = A.s[i];
        if (s.n == 0u) continue;
        const uint32_t len = s.pos + s.n, pre = std::min(s.prefix, len);
        const uint32_t first = pre ? 0u : A.window && s.pos + 1u > A.window ? s.pos + 1u - A.window : 0u;   // that a query sees
        VRT_REQUIRE(static_cast<uint64_t>(first >> 5) + z.nb >= len / kKvBlock, "%s: sequence %u: the cache no longer holds position %u",
                    who, s.seq, first);
        VRT_REQUIRE(!scored || len <= c->max_ctx, "%s: weights need pos + n <= max_ctx", who);
        items += (static_cast<uint64_t>(s.n) * A.G + 15u) / 16u * c->kv_heads;
    }
    VRT_REQUIRE(*total * A.G <= 0x3fffffffu && items <= 0x3fffffu, "%s: too many rows", who);
    *P = kv8_plan(A, c->kv_heads, z.hdp, n, *total, scored);
    // a grid has fewer than 2^32 threads, and as many workgroups for every sequence as for the longest
    VRT_REQUIRE(static_cast<uint64_t>(P->units) * A.splits * c->kv_heads * n < (1ull << 32) / kKvThreads, "%s: too many rows", who);
    return VRT_OK;
}

// Tiles of 16 rows that a prompt's wave runs together: as many as leave two waves a SIMD.
constexpr int rows_of(int nt) { return nt <= 4 ? 4 : 2; }

uint32_t tile_threads(const Kv8Dev& c) { return c.hdp >= 96u ? 512u : 256u; }   // KvTile::TH

enum Kv8Kernel { kKvAppend, kKvRead, kKvToken, kKvPrompt, kKvWeights, kKvGather };
template <int NT>
const void* kernel_of(Kv8Kernel k, bool cap) {
    constexpr int RT = rows_of(NT);
    switch (k) {
        case kKvAppend: return reinterpret_cast<const void*>(&k_kv8_append<NT>);
        case kKvRead: return reinterpret_cast<const void*>(&k_kv8_read<NT>);
        case kKvGather: return reinterpret_cast<const void*>(&k_kv8_gather<NT>);
        case kKvToken: return cap ? reinterpret_cast<const void*>(&k_kv8_attn<NT, 1, true>) : reinterpret_cast<const void*>(&k_kv8_attn<NT, 1, false>);
        case kKvPrompt:
            return cap ? reinterpret_cast<const void*>(&k_kv8_attn<NT, RT, true>) : reinterpret_cast<const void*>(&k_kv8_attn<NT, RT, false>);
        default: return cap ? reinterpret_cast<const void*>(&k_kv8_weights<NT, true>) : reinterpret_cast<const void*>(&k_kv8_weights<NT, false>);
    }
}
const void* kernel_of(const Kv8Dev& c, Kv8Kernel k, bool cap = false) {
    switch (c.hdp / 32u) {
        case 1: return kernel_of<1>(k, cap);
        case 2: return kernel_of<2>(k, cap);
        case 3: return kernel_of<3>(k, cap);
        case 4: return kernel_of<4>(k, cap);
        case 5: return kernel_of<5>(k, cap);
        case 6: return kernel_of<6>(k, cap);
        case 7: return kernel_of<7>(k, cap);
        default: return kernel_of<8>(k, cap);
    }
}

template <class Args>
int launch(const void* fn, dim3 grid, uint32_t threads, Args& A, hipStream_t s) {
    void* args[] = {&A};
    VRT_HIP_CHECK(hipLaunchKernel(fn, grid, dim3(threads), args, 0, s));
    return VRT_OK;
}

}  // namespace

Kv8Sizes kv8_sizes(uint32_t max_seqs, uint32_t max_ctx, uint32_t kv_heads, uint32_t head_dim) {
    Kv8Sizes z;
    z.nb = (max_ctx + kKvBlock - 1u) / kKvBlock;
    z.hdp = (head_dim + 31u) / 32u * 32u;
    const uint64_t heads = static_cast<uint64_t>(max_seqs) * kv_heads, blocks = heads * z.nb;   // below 2^47
    z.codes = up256(blocks * 64u * z.hdp);
    z.scales = up256(blocks * sizeof(float2));
    z.tail = up256(heads * 128u * z.hdp * 4u);
    z.pairs = up256(heads * 256u * z.hdp * 2u);
    z.factor = up256(heads * 128u * 4u);
    z.total = z.codes + z.scales + z.tail + z.pairs + z.factor;
    return z;
}

Kv8Dev kv8_view(const Kv8Sizes& z, void* data, uint32_t kv_heads, uint32_t head_dim) {
    auto* p = static_cast<uint8_t*>(data);
    Kv8Dev d;
    d.codes = p;
    d.scales = reinterpret_cast<float2*>(p + z.codes);
    d.tail = reinterpret_cast<float*>(p + z.codes + z.scales);
    d.pairs = reinterpret_cast<_Float16*>(p + z.codes + z.scales + z.tail);
    d.factor = reinterpret_cast<float*>(p + z.codes + z.scales + z.tail + z.pairs);
    d.nb = z.nb;
    d.kvh = kv_heads;
    d.hd = head_dim;
    d.hdp = z.hdp;
    return d;
}

// A unit's blocks are split where there are too few units: into about 512 workgroups (two a CU), of four blocks (one a wave) at
// least. Into 512, 1024 and 2048: 64 sequences of 8 K, one head of 256, 43, 48 and 52 us; 2 of 128 K, 8 heads of 128, 109, 101 and 94
// but 5, 7 and 10 in the join. Prompts with a unit for every CU are not split: their outputs would be written and read once more.
constexpr uint64_t kKvSplits = 512;
// Units of this many blocks or fewer, six a wave, stay whole: 64 sequences in a window of 512 (17 blocks) take 15 to 18 us whole,
// and split by five 15 and 4 in the join.
constexpr uint32_t kKvWhole = 24;

Kv8Plan kv8_plan(Kv8AttnArgs& A, uint32_t kvh, uint32_t hdp, uint32_t n, uint64_t rows, bool scored) {
    Kv8Plan P{};
    uint32_t active = 0;
    A.rows_most = 0;
    for (uint32_t i = 0; i < n; ++i) {
        active += A.s[i].n != 0u;
        A.rows_most = std::max(A.rows_most, A.s[i].n * A.G);
    }
    A.nseq = n;
    A.prompt = rows * A.G > 32ull * active;   // from three of a token's tiles on; below, most of a prompt's tiles would be empty
    A.unit = A.prompt ? 16u * rows_of(static_cast<int>(hdp / 32u)) : 16u;
    A.lines = std::min(A.unit, std::max(1u, A.rows_most));
    uint64_t units_all = 0, blocks = 0;   // of all units and heads; a prompt's queries see half of its own on average
    uint32_t most = 1;                    // blocks of a unit
    for (uint32_t i = 0; i < n; ++i) {
        const Kv8Seq& s = A.s[i];
        const uint32_t nb = most_blocks(s, A.window, A.unit);
        most = std::max(most, nb);
        const uint64_t units = static_cast<uint64_t>((s.n * A.G + A.unit - 1u) / A.unit) * kvh;
        units_all += units;
        blocks += units * (s.prefix ? nb : std::min(nb, (s.pos + (s.n + 1u) / 2u + 31u) / 32u));
    }
    uint64_t per = std::max<uint64_t>(4u, (blocks + kKvSplits - 1u) / kKvSplits);
    if (A.prompt && units_all >= kKvSplits / 2u) per = VRT_KV8_MAX_CTX / 32u + 4u;
    else if (most <= kKvWhole) per = most;
    A.fold = A.prompt && units_all <= kKvSplits;
    A.per = static_cast<uint32_t>((per + 3u) & ~3ull);
    A.splits = 1u;
    const bool dump = scored && !A.prompt;
    uint64_t place = 0;
    for (uint32_t i = 0; i < n; ++i) {
        Kv8Seq& s = A.s[i];
        const uint32_t units = (s.n * A.G + A.unit - 1u) / A.unit;
        s.splits = std::max(1u, (most_blocks(s, A.window, A.unit) + A.per - 1u) / A.per);
        s.part0 = static_cast<uint32_t>(place);
        if (s.splits > 1u || dump) place += static_cast<uint64_t>(units) * kvh * s.splits;
        A.splits = std::max(A.splits, s.splits);
        P.units = std::max(P.units, units);
    }
    P.part = A.splits > 1u ? up256(place * A.lines * hdp * 4u) : 0u;
    P.ml = up256(place * A.lines * sizeof(float2));
    P.extra = !scored ? 0u : dump ? up256(place * A.lines * 32u * A.per * 4u) : up256(rows * A.heads * sizeof(float2));
    P.total = P.part + P.ml + P.extra;
    return P;
}

// Of calls with one row a sequence and at most 32 query heads a kv head. Blocks of a sequence's unit and head: at most
// ceil(max_ctx / 32); splits: at most blocks / per + 1, all blocks / per at most kKvSplits.
uint64_t kv8_workspace_most(uint32_t seqs, uint32_t max_ctx, uint32_t heads, uint32_t kvh, uint32_t hdp, bool scored) {
    const uint64_t items = static_cast<uint64_t>(seqs) * kvh * ((heads / kvh + 15u) / 16u), blocks = items * ((max_ctx + 31u) / 32u);
    const uint64_t per = (std::max<uint64_t>(4u, (blocks + kKvSplits - 1u) / kKvSplits) + 3u) & ~3ull;
    const uint64_t place = kKvSplits + items, lines = std::min(16u, heads / kvh);
    return up256(place * lines * hdp * 4u) + up256(place * lines * sizeof(float2)) +
           (scored ? up256((blocks + items * per) * lines * 32u * 4u) : 0u);
}

int kv8_append(const Kv8Dev& c, const Kv8Seq* seqs, uint32_t n, const float* k, const float* v, uint64_t stride, hipStream_t s) {
    Kv8AppendArgs A{};
    A.c = c;
    A.x[0] = k;
    A.x[1] = v;
    A.stride = stride;
    uint32_t blocks = 0;
    for (uint32_t i = 0; i < n; ++i) {
        A.s[i] = seqs[i];
        blocks = std::max(blocks, touched(seqs[i]));
    }
    if (blocks == 0u) return VRT_OK;
    return launch(kernel_of(c, kKvAppend), dim3(blocks, 2u * c.kvh, n), tile_threads(c), A, s);
}

int kv8_attend(Kv8AttnArgs& A, const Kv8Plan& P, void* workspace, uint32_t n, hipStream_t s) {
    auto* ws = static_cast<uint8_t*>(workspace);
    const bool scored = A.w_out != nullptr, cap = A.cap > 0.0f;
    A.part = reinterpret_cast<float*>(ws);
    A.part_ml = reinterpret_cast<float2*>(ws + P.part);
    auto* extra = reinterpret_cast<float*>(ws + P.part + P.ml);
    A.scores = scored && !A.prompt ? extra : nullptr;
    A.stats = scored && A.prompt ? reinterpret_cast<float2*>(extra) : nullptr;
    if (int rc = launch(kernel_of(A.c, A.prompt ? kKvPrompt : kKvToken, cap), dim3(P.units * A.splits * A.c.kvh * n), kKvThreads, A, s))
        return rc;
    uint32_t len = 0;
    for (uint32_t i = 0; i < n; ++i)
        if (A.s[i].n) len = std::max(len, A.s[i].pos + A.s[i].n);
    const uint32_t wgs = (A.splits > 1u ? A.rows_most : 0u) + (A.scores ? (len + kKvThreads - 1u) / kKvThreads : 0u);
    if (wgs)
        if (int rc = launch(reinterpret_cast<const void*>(&k_kv8_join), dim3(wgs, A.c.kvh, n), kKvThreads, A, s)) return rc;
    if (!scored || !A.prompt) return VRT_OK;
    return launch(kernel_of(A.c, kKvWeights, cap), dim3((len + 31u) / 32u, A.c.kvh, n), 64u * kKvWeightWaves, A, s);
}

int kv8_evict(const Kv8Dev& c, const vrt_kv8_move* moves, uint32_t n, float* weights, uint32_t max_ctx, uint32_t* kept,
              uint64_t kept_stride, hipStream_t s) {
    Kv8EvictArgs A{};
    A.c = c;
    A.w = weights;
    A.kept = kept;
    A.kept_stride = kept_stride;
    A.max_ctx = max_ctx;
    uint32_t keep = 0;
    for (uint32_t i = 0; i < n; ++i) {
        A.m[i] = moves[i];
        keep = std::max(keep, moves[i].keep);
    }
    if (keep == 0u) return VRT_OK;
    if (int rc = launch(reinterpret_cast<const void*>(&k_kv8_select), dim3(c.kvh, n), kKvSelThreads, A, s)) return rc;
    return launch(kernel_of(c, kKvGather), dim3(((keep + 31u) / 32u + 7u) & ~7u, 2u * c.kvh, n), tile_threads(c), A, s);
}

}  // namespace vrt

using namespace vrt;

extern "C" int vrt_kv8_cache_bytes(const vrt_kv8_cache* cache, uint64_t* bytes) {
    VRT_REQUIRE(bytes, "vrt_kv8_cache_bytes: null argument");
    Kv8Sizes z;
    if (int rc = check_cache(cache, "vrt_kv8_cache_bytes", &z)) return rc;
    *bytes = z.total;
    return VRT_OK;
}

extern "C" int vrt_kv8_append(vrt_ctx* ctx, const vrt_kv8_cache* cache, const vrt_kv8_rows* rows, uint32_t n_seqs,
                              const float* k, const float* v, uint64_t kv_stride) {
    const char* who = "vrt_kv8_append";
    VRT_REQUIRE(ctx, "%s: null context", who);
    Kv8Dev c;
    Kv8Seq s[kKvMaxSeqs];
    uint64_t total;
    if (int rc = cache_view(cache, who, &c)) return rc;
    if (int rc = check_rows(cache, rows, n_seqs, who, s, &total)) return rc;
    const uint64_t width = static_cast<uint64_t>(cache->kv_heads) * cache->head_dim;
    if (int rc = check_array(k, &kv_stride, width, who, "k")) return rc;
    if (int rc = check_array(v, &kv_stride, width, who, "v")) return rc;
    for (uint32_t i = 0; i < n_seqs; ++i)
        VRT_REQUIRE(touched(s[i]) <= c.nb, "%s: sequence %u: more blocks than a region of %u positions holds", who, s[i].seq,
                    cache->max_ctx);
    if (total == 0u) return VRT_OK;
    OnDevice on(ctx->device);
    VRT_HIP_CHECK(on.err);
    return kv8_append(c, s, n_seqs, k, v, kv_stride, ctx->stream);
}

extern "C" int vrt_kv8_read(vrt_ctx* ctx, const vrt_kv8_cache* cache, const vrt_kv8_rows* rows, uint32_t n_seqs,
                            const uint32_t* lens, float* k, float* v, uint64_t kv_stride) {
    const char* who = "vrt_kv8_read";
    VRT_REQUIRE(ctx, "%s: null context", who);
    Kv8ReadArgs A{};
    if (int rc = cache_view(cache, who, &A.c)) return rc;
    uint64_t total;
    if (int rc = check_rows(cache, rows, n_seqs, who, A.s, &total)) return rc;
    A.stride = kv_stride;
    const uint64_t width = static_cast<uint64_t>(cache->kv_heads) * cache->head_dim;
    if (int rc = check_array(k, &A.stride, width, who, "k")) return rc;
    if (int rc = check_array(v, &A.stride, width, who, "v")) return rc;
    A.x[0] = k;
    A.x[1] = v;
    uint32_t blocks = 0;
    for (uint32_t i = 0; i < n_seqs; ++i) {
        Kv8Seq& s = A.s[i];
        const uint32_t end = s.pos + s.n, len = lens ? lens[i] : end;
        VRT_REQUIRE(len >= end && len <= VRT_KV8_MAX_CTX, "%s: sequence %u: positions past its length", who, s.seq);
        VRT_REQUIRE(s.n == 0u || (s.pos >> 5) + A.c.nb >= len / kKvBlock, "%s: sequence %u: the cache no longer holds position %u", who,
                    s.seq, s.pos);
        s.prefix = len;
        blocks = std::max(blocks, touched(s));
    }
    if (blocks == 0u) return VRT_OK;
    OnDevice on(ctx->device);
    VRT_HIP_CHECK(on.err);
    return launch(kernel_of(A.c, kKvRead), dim3(blocks, 2u * A.c.kvh, n_seqs), tile_threads(A.c), A, ctx->stream);
}

extern "C" int vrt_kv8_attend_workspace(const vrt_kv8_cache* cache, const vrt_kv8_attn* attn, const vrt_kv8_rows* rows,
                                        uint32_t n_seqs, uint32_t scored, uint64_t* bytes) {
    const char* who = "vrt_kv8_attend_workspace";
    VRT_REQUIRE(bytes, "%s: null argument", who);
    Kv8AttnArgs A{};
    Kv8Plan P{};
    uint64_t total;
    if (int rc = attn_plan(cache, attn, rows, n_seqs, scored != 0u, who, A, &P, &total)) return rc;
    *bytes = P.total;
    return VRT_OK;
}

extern "C" int vrt_kv8_attend(vrt_ctx* ctx, const vrt_kv8_cache* cache, const vrt_kv8_attn* attn, const vrt_kv8_rows* rows,
                              uint32_t n_seqs, const float* q, uint64_t q_stride, float* out, uint64_t out_stride,
                              const float* weights_in, float* weights_out, void* workspace, uint64_t workspace_bytes) {
    const char* who = "vrt_kv8_attend";
    VRT_REQUIRE(ctx, "%s: null context", who);
    Kv8AttnArgs A{};
    Kv8Plan P{};
    uint64_t total;
    if (int rc = attn_plan(cache, attn, rows, n_seqs, weights_out != nullptr, who, A, &P, &total)) return rc;
    if (int rc = cache_view(cache, who, &A.c)) return rc;
    const uint64_t width = static_cast<uint64_t>(A.heads) * cache->head_dim;
    if (int rc = check_array(q, &q_stride, width, who, "q")) return rc;
    if (int rc = check_array(out, &out_stride, width, who, "out")) return rc;
    VRT_REQUIRE(weights_out || !weights_in, "%s: weights_in without weights_out", who);
    VRT_REQUIRE(((reinterpret_cast<uintptr_t>(weights_in) | reinterpret_cast<uintptr_t>(weights_out)) & 3u) == 0u,
                "%s: weights must be 4-byte aligned", who);
    VRT_REQUIRE(P.total == 0u || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0u && workspace_bytes >= P.total),
                "%s: workspace must be 256-byte aligned, at least %llu bytes", who, static_cast<unsigned long long>(P.total));
    if (total == 0u) return VRT_OK;
    A.q = q;
    A.q_stride = q_stride;
    A.o.rows = out;
    A.o.stride = out_stride;
    A.w_in = weights_in;
    A.w_out = weights_out;
    OnDevice on(ctx->device);
    VRT_HIP_CHECK(on.err);
    return kv8_attend(A, P, workspace, n_seqs, ctx->stream);
}

extern "C" int vrt_kv8_evict(vrt_ctx* ctx, const vrt_kv8_cache* cache, const vrt_kv8_move* moves, uint32_t n, float* weights,
                             uint32_t* kept, uint64_t kept_stride) {
    const char* who = "vrt_kv8_evict";
    VRT_REQUIRE(ctx && moves && weights && kept, "%s: null argument", who);
    Kv8Dev c;
    if (int rc = cache_view(cache, who, &c)) return rc;
    VRT_REQUIRE(n >= 1u && n <= kKvMaxSeqs, "%s: n must be 1..%u", who, kKvMaxSeqs);
    VRT_REQUIRE(((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(kept)) & 3u) == 0u,
                "%s: weights and kept must be 4-byte aligned", who);
    VRT_REQUIRE(kept_stride <= (1ull << 32), "%s: kept_stride is too large", who);
    for (uint32_t i = 0; i < n; ++i) {
        const vrt_kv8_move& m = moves[i];
        VRT_REQUIRE(m.src < cache->max_seqs && m.dst < cache->max_seqs, "%s: sequence out of range", who);
        VRT_REQUIRE(m.recent <= m.keep && m.keep <= m.len && m.len <= cache->max_ctx, "%s: needs recent <= keep <= len <= max_ctx", who);
        VRT_REQUIRE(m.keep <= kept_stride, "%s: kept_stride is smaller than keep", who);
        for (uint32_t j = 0; j < n; ++j) {
            VRT_REQUIRE(moves[j].src != m.dst, "%s: sequence %u is a source and a destination", who, m.dst);
            VRT_REQUIRE(j == i || moves[j].dst != m.dst, "%s: sequence %u is a destination twice", who, m.dst);
        }
    }
    OnDevice on(ctx->device);
    VRT_HIP_CHECK(on.err);
    return kv8_evict(c, moves, n, weights, cache->max_ctx, kept, kept_stride, ctx->stream);
}
