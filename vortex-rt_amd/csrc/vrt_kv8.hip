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
    return (static_cast<uint64_t>(seq) * c.kvh + head) * c.nb + b % c.nb;
}
__device__ __forceinline__ uint8_t* kv_codes(const Kv8Dev& c, uint64_t block) { return c.codes + block * 64u * c.hdp; }
// Row (parity, K or V, slot) of the tail.
__device__ __forceinline__ uint64_t kv_tail_row(const Kv8Dev& c, uint32_t seq, uint32_t head, uint32_t b, uint32_t z,
                                                uint32_t slot) {
    return (((static_cast<uint64_t>(seq) * c.kvh + head) * 2u + (b & 1u)) * 2u + z) * 32u + slot;
}
// Byte of a value inside its block's 32 hdp bytes.
__device__ __forceinline__ uint32_t kv_k_at(uint32_t t, uint32_t d) {
    return (d >> 5) * 1024u + (((d >> 3) & 3u) * 16u + (t & 15u)) * 16u + (t >> 4) * 8u + (d & 7u);
}
__device__ __forceinline__ uint32_t kv_v_at(uint32_t t, uint32_t d) {
    return (d >> 5) * 1024u + (((t >> 2) & 3u) * 16u + (d & 15u)) * 16u + ((d >> 4) & 1u) * 8u + (t & 3u) + (t >> 4) * 4u;
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    for (int o = 32; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o)));
    return v;
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
    return fminf(fmaxf(q, -127.0f), 127.0f);
}

// ---- append ---------------------------------------------------------------------------------

// A workgroup's 32 x hd values of one head and block, as up to 8 float4 per thread (unit tid + 256 k: token
// unit / (hd / 4), dims 4 (unit % (hd / 4)) ..): amax, scale, codes, in operand order through an LDS image.
struct KvTile {
    f4 v[8];
};
__device__ __forceinline__ void kv_unit(uint32_t u, uint32_t hd4, uint32_t& t, uint32_t& d) {
    t = u / hd4;
    d = (u - t * hd4) * 4u;
}
__device__ __forceinline__ uint32_t f_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ void kv_close_block(const Kv8Dev& c, const KvTile& x, uint64_t block, uint32_t z, uint8_t* img,
                                               uint32_t* red) {
    const uint32_t tid = threadIdx.x, hd4 = c.hd >> 2, units = 32u * hd4;
    uint32_t m = 0u;   // |x| as integers: larger is larger, NaN above infinity above the rest
#pragma unroll
    for (uint32_t k = 0; k < 8u; ++k)
        if (tid + kKvThreads * k < units)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = max(m, f_bits(x.v[k][e]));
    m = wave_max_u32(m);
    if ((tid & 63u) == 0u) red[tid >> 6] = m;
    if (c.hd != c.hdp)   // the padding dimensions' codes: zeros
        for (uint32_t i = tid; i < 8u * c.hdp; i += kKvThreads) reinterpret_cast<uint32_t*>(img)[i] = 0x80808080u;
    __syncthreads();
    m = max(max(red[0], red[1]), max(red[2], red[3]));
    const float s = m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(m) / 127.0f;
    const bool live = s > 0.0f;
    // the quotient's steps stay away from denormals: their halves and reciprocals are no numbers
    const float up = s < 0x1p-100f ? 0x1p60f : 1.0f, su = s * up;
    const float inv = live ? 1.0f / su : 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < 8u; ++k) {
        const uint32_t u = tid + kKvThreads * k;
        if (u >= units) break;
        uint32_t t, d, w = 0u;
        kv_unit(u, hd4, t, d);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float q = live ? kv_round(x.v[k][e] * up, su, inv) : 0.0f;
            w |= static_cast<uint32_t>(static_cast<int>(q) + 128) << (8 * e);
        }
        if (z == 0u) {
            *reinterpret_cast<uint32_t*>(img + kv_k_at(t, d)) = w;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) img[kv_v_at(t, d + e)] = static_cast<uint8_t>(w >> (8u * e));
        }
    }
    __syncthreads();
    uint4* dst = reinterpret_cast<uint4*>(kv_codes(c, block) + z * 32u * c.hdp);
    for (uint32_t i = tid; i < 2u * c.hdp; i += kKvThreads) dst[i] = reinterpret_cast<const uint4*>(img)[i];
    if (tid == 0u) reinterpret_cast<float*>(c.scales + block)[z] = s;
}

// Rows first .. last of block b (rows of x, which hold the call's positions from p0 on) into its tail: values and row maxima.
__device__ __forceinline__ void kv_to_tail(const Kv8Dev& c, uint32_t seq, uint32_t head, uint32_t b, uint32_t z, const float* x,
                                           uint64_t stride, uint32_t p0, uint32_t first, uint32_t last) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t p = first + wave; p <= last; p += kKvThreads / 64u) {
        const uint64_t row = kv_tail_row(c, seq, head, b, z, p & 31u);
        f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (4u * lane < c.hd) v = *reinterpret_cast<const f4*>(x + static_cast<uint64_t>(p - p0) * stride + 4u * lane);
        if (4u * lane < c.hdp) *reinterpret_cast<f4*>(c.tail + row * c.hdp + 4u * lane) = v;
        const uint32_t m = wave_max_u32(max(max(f_bits(v[0]), f_bits(v[1])), max(f_bits(v[2]), f_bits(v[3]))));
        if (lane == 0u) c.tmax[row] = __uint_as_float(m);
    }
}

struct Kv8AppendArgs {
    Kv8Dev c;
    const float* x[2];   // k, v
    uint64_t stride;
    Kv8Seq s[kKvMaxSeqs];
};

// One workgroup per (block the call touches, head and K or V, sequence). A full block's codes; the rows of the last two
// blocks also go to the tail. The first block's earlier rows come from the tail, which a later block of the same
// parity would overwrite: so the first block's workgroup writes all of the tail, after it has read it.
__global__ void __launch_bounds__(kKvThreads) k_kv8_append(const Kv8AppendArgs A) {
    __shared__ __align__(16) uint8_t img[32 * 256];
    __shared__ uint32_t red[4];
    const Kv8Dev& c = A.c;
    const Kv8Seq& S = A.s[blockIdx.z];
    const uint32_t head = blockIdx.y >> 1, z = blockIdx.y & 1u, tid = threadIdx.x;
    if (S.n == 0u) return;
    const uint32_t end = S.pos + S.n, b0 = S.pos >> 5, bl = (end - 1u) >> 5, b = b0 + blockIdx.x;
    if (b > bl) return;
    const bool closed = (b + 1u) * 32u <= end;
    const float* x = A.x[z] + static_cast<uint64_t>(S.row0) * A.stride + head * c.hd;
    if (closed) {
        KvTile T;
        const uint32_t hd4 = c.hd >> 2, units = 32u * hd4;
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) {
            const uint32_t u = tid + kKvThreads * k;
            T.v[k] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (u >= units) continue;
            uint32_t t, d;
            kv_unit(u, hd4, t, d);
            const uint32_t p = 32u * b + t;
            const float* src = p < S.pos ? c.tail + kv_tail_row(c, S.seq, head, b, z, t) * c.hdp + d
                                         : x + static_cast<uint64_t>(p - S.pos) * A.stride + d;
            T.v[k] = *reinterpret_cast<const f4*>(src);
        }
        kv_close_block(c, T, kv_block(c, S.seq, head, b), z, img, red);   // (its barriers come after every read of the tail)
    }
    if (b != b0) return;
    for (uint32_t t = bl > b0 ? bl - 1u : bl; t <= bl; ++t)
        kv_to_tail(c, S.seq, head, t, z, x, A.stride, S.pos, max(S.pos, 32u * t), min(end, 32u * t + 32u) - 1u);
}

// ---- read -----------------------------------------------------------------------------------

struct Kv8ReadArgs {
    Kv8Dev c;
    float* x[2];
    uint64_t stride;
    Kv8Seq s[kKvMaxSeqs];   // prefix: the sequence's length
};

__device__ __forceinline__ float kv_value(const Kv8Dev& c, uint32_t seq, uint32_t head, uint32_t z, uint32_t p, uint32_t d,
                                          uint32_t len) {
#pragma clang fp contract(off)
    const uint32_t b = p >> 5, t = p & 31u;
    if ((b + 1u) * 32u > len) return c.tail[kv_tail_row(c, seq, head, b, z, t) * c.hdp + d];
    const uint64_t blk = kv_block(c, seq, head, b);
    const uint8_t u = kv_codes(c, blk)[z * 32u * c.hdp + (z ? kv_v_at(t, d) : kv_k_at(t, d))];
    const float s = reinterpret_cast<const float*>(c.scales + blk)[z];
    return s * static_cast<float>(static_cast<int>(u) - 128);
}

__global__ void __launch_bounds__(kKvThreads) k_kv8_read(const Kv8ReadArgs A) {
    const Kv8Dev& c = A.c;
    const Kv8Seq& S = A.s[blockIdx.z];
    const uint32_t head = blockIdx.y >> 1, z = blockIdx.y & 1u;
    const uint32_t b = (S.pos >> 5) + blockIdx.x, hd4 = c.hd >> 2;
    for (uint32_t u = threadIdx.x; u < 32u * hd4; u += kKvThreads) {
        uint32_t t, d;
        kv_unit(u, hd4, t, d);
        const uint32_t p = 32u * b + t;
        if (p < S.pos || p - S.pos >= S.n) continue;
        f4 v;
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) v[e] = kv_value(c, S.seq, head, z, p, d + e, S.prefix);
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

// Four biased codes to f16: the byte under 0x64 is 1024 + u, exactly.
__device__ __forceinline__ void kv_cvt4(uint32_t w, h2& a, h2& b) {
    const h2 off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
    b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
}
__device__ __forceinline__ h8 kv_cvt8(uint32_t w0, uint32_t w1) {
    h2 a, b, c, d;
    kv_cvt4(w0, a, b);
    kv_cvt4(w1, c, d);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x = hi + lo in f16 (x below 2^15 in magnitude; what is lost is below 2^-24)
__device__ __forceinline__ void kv_split(float x, _Float16& hi, _Float16& lo) {
    asm("" : "+v"(x));
    hi = static_cast<_Float16>(x);
    lo = static_cast<_Float16>(x - static_cast<float>(hi));
}
// The exponent e with m 2^e in [2^(to - 1), 2^to), at most 126 so that 2^-e is a number; 0 where m is 0 or not finite.
__device__ __forceinline__ int kv_exp(float m, int to) {
    return m > 0.0f && m < INFINITY ? min(to - __builtin_amdgcn_frexp_expf(m), 126) : 0;
}

// tanh(x): below 1/4 its series (the next term is 9e-9 of it), above by e^(-2|x|), at 1 ulp each of exponential and
// reciprocal.
__device__ __forceinline__ float kv_tanh(float x) {
    const float a = fabsf(x), y = x * x;
    const float e = __builtin_amdgcn_exp2f(a * -2.885390082f);
    const float big = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
    const float small = x + x * y * (-0.3333333333f + y * (0.1333333333f + y * (-0.05396825397f + y * 0.02186948854f)));
    return a < 0.25f ? small : copysignf(big, x);
}

// A row tile's queries as the B operand of the transposed scores: lane l holds row r0 + l % 16 (query (r0 + l % 16) / G, head
// kvh G + (r0 + l % 16) % G), dims 32 s + 8 (l / 16) + e, scaled by a power of two to below 2^14 and split.
template <int NT>
struct KvQuery {
    h8 hi[NT], lo[NT];
    float back;    // the row's power of two, inverted
    uint32_t p;    // its position
};
template <int NT>
__device__ __forceinline__ void kv_load_q(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t kvh, uint32_t r0, KvQuery<NT>& Q) {
    const uint32_t lane = threadIdx.x & 63u, R = S.n * A.G, hd = A.c.hd;
    const uint32_t r = min(r0 + (lane & 15u), R - 1u), qi = r / A.G, h = kvh * A.G + (r - qi * A.G);
    const float* src = A.q + (static_cast<uint64_t>(S.row0) + qi) * A.q_stride + h * hd;
    f4 x[NT][2];
    float m = 0.0f;
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j) {
            const uint32_t d = 32u * s + 8u * (lane >> 4) + 4u * j;
            x[s][j] = d < hd ? *reinterpret_cast<const f4*>(src + d) : f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(x[s][j][e]));
        }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const int ex = kv_exp(m, 14);
    Q.back = ldexpf(1.0f, -ex);
    Q.p = S.pos + qi;
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            _Float16 a, b;
            kv_split(ldexpf(x[s][j >> 2][j & 3], ex), a, b);
            Q.hi[s][j] = a;
            Q.lo[s][j] = b;
        }
}

#define KV_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0)

// Block b's scores, in log2 units and masked: lane l holds row l % 16's of tokens 4 (l / 16) + e (e < 4) and 16 + 4 (l / 16) + e - 4.
// Of the sequence's open block the keys come from the tail, as f16 pairs; tmax names their largest and those not finite.
template <int NT, bool CAP>
__device__ __forceinline__ void kv_scores(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t kvh, uint32_t b, const KvQuery<NT>& Q,
                                          bool masked, float (&s)[8]) {
    const Kv8Dev& c = A.c;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, m16 = lane & 15u, len = S.pos + S.n;
    f4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
    float ks;
    if ((b + 1u) * 32u <= len) {
        const uint64_t blk = kv_block(c, S.seq, kvh, b);
        const uint4* src = reinterpret_cast<const uint4*>(kv_codes(c, blk)) + lane;
        ks = c.scales[blk].x;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint4 w = src[64 * t];
            const h8 a0 = kv_cvt8(w.x, w.y), a1 = kv_cvt8(w.z, w.w);
            acc[0] = KV_MFMA(a0, Q.hi[t], acc[0]);
            acc[1] = KV_MFMA(a1, Q.hi[t], acc[1]);
            acc[0] = KV_MFMA(a0, Q.lo[t], acc[0]);
            acc[1] = KV_MFMA(a1, Q.lo[t], acc[1]);
        }
    } else {
        const uint64_t row0 = kv_tail_row(c, S.seq, kvh, b, 0u, 0u);
        const uint32_t live = len - 32u * b;   // tokens of the block
        float m = (lane & 31u) < live ? c.tmax[row0 + (lane & 31u)] : 0.0f;
        m = wave_max(m < INFINITY ? m : 0.0f);
        const int ex = kv_exp(m, 7);
        ks = ldexpf(1.0f, -ex);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (uint32_t half = 0; half < 2u; ++half) {
                const uint32_t tok = 16u * half + m16;
                h8 hi, lo;
                f4 x[2];
#pragma unroll
                for (uint32_t j = 0; j < 2u; ++j)
                    x[j] = *reinterpret_cast<const f4*>(c.tail + (row0 + min(tok, live - 1u)) * c.hdp + 32u * t + 8u * g + 4u * j);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    _Float16 h, l;
                    kv_split(ldexpf(x[j >> 2][j & 3], ex), h, l);
                    hi[j] = h;
                    lo[j] = l;
                }
                acc[half] = KV_MFMA(hi, Q.hi[t], acc[half]);
                acc[half] = KV_MFMA(hi, Q.lo[t], acc[half]);
                acc[half] = KV_MFMA(lo, Q.hi[t], acc[half]);
            }
    }
    const float f = Q.back * (ks * A.scale);
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e) {
        float x = acc[e >> 2][e & 3u];
        if constexpr (CAP) x = A.cap * kv_tanh(x * f * (1.0f / A.cap)) * 1.4426950409f;
        else x = x * (f * 1.4426950409f);
        if (masked) {
            const uint32_t j = 32u * b + 4u * g + (e & 3u) + 16u * (e >> 2);
            const bool see = j < len && (j < S.prefix || (j <= Q.p && (!A.window || Q.p - j < A.window)));
            x = see ? x : -INFINITY;
        }
        s[e] = x;
    }
}

// Whether some row of a tile does not see all of block b.
__device__ __forceinline__ bool kv_masked(const Kv8AttnArgs& A, const Kv8Seq& S, uint32_t b, uint32_t pmin, uint32_t pmax) {
    const uint32_t last = 32u * b + 31u, len = S.pos + S.n;
    if (last < S.prefix && last < len) return false;
    return !(last <= pmin && (!A.window || pmax - 32u * b < A.window));
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

// One workgroup per (split of a row tile's blocks, head, sequence); wave w takes the split's blocks w, w + 4, ...: scores on
// the matrix cores with the tokens as rows, so that each lane holds eight weights of one query row in the order in
// which the values are kept; running maximum and sum per row; weights times the block's value scale, as f16 pairs, times
// the values' codes into the transposed output (rows: dims). The waves meet in LDS.
template <int NT, bool CAP>
__global__ void __launch_bounds__(kKvThreads) k_kv8_attn(const Kv8AttnArgs A) {
    constexpr uint32_t kRow = 32u * NT + 4u;
    __shared__ __align__(16) float s_acc[2][16 * kRow];
    __shared__ float s_m[4][16], s_l[4][16];
    const Kv8Seq& S = A.s[blockIdx.z];
    const uint32_t kvh = blockIdx.y, tile = blockIdx.x / A.splits, split = blockIdx.x - tile * A.splits;
    const uint32_t R = S.n * A.G, r0 = 16u * tile, len = S.pos + S.n;
    if (r0 >= R || split >= S.splits) return;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, m16 = lane & 15u;
    const uint32_t pmin = S.pos + r0 / A.G, pmax = S.pos + min(r0 + 15u, R - 1u) / A.G;
    const KvSpan sp = kv_span(A, S, pmin, pmax);
    const uint32_t i0 = split * A.per, i1 = min(sp.n, i0 + A.per);
    if (i0 >= i1) return;
    const Kv8Dev& c = A.c;
    KvQuery<NT> Q;
    kv_load_q<NT>(A, S, kvh, r0, Q);
    float m = -INFINITY, l = 0.0f;
    int eR = kKvNoExp;   // acc holds sum p v 2^(15 - eR), 2^eR above every value scale so far
    f4 acc[2 * NT];
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t) acc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i = i0 + wave; i < i1; i += 4u) {
        const uint32_t b = i < sp.n_pre ? i : sp.lo + (i - sp.n_pre);
        const bool open = (b + 1u) * 32u > len;
        float s[8];
        kv_scores<NT, CAP>(A, S, kvh, b, Q, open || kv_masked(A, S, b, pmin, pmax), s);
        // the block's value scale; of the open block: a power of two, and its tokens with a key or value that is not finite
        const uint64_t row0 = kv_tail_row(c, S.seq, kvh, b, 1u, 0u);
        const uint32_t live = min(32u, len - 32u * b);
        float vs;
        int tex = 0;
        uint32_t bad = 0u;
        if (!open) {
            vs = c.scales[kv_block(c, S.seq, kvh, b)].y;
        } else {
            const float tv = (lane & 31u) < live ? c.tmax[row0 + (lane & 31u)] : 0.0f;
            const float tk = (lane & 31u) < live ? c.tmax[kv_tail_row(c, S.seq, kvh, b, 0u, lane & 31u)] : 0.0f;
            bad = static_cast<uint32_t>(__ballot(!(tv < INFINITY) || !(tk < INFINITY)));
            tex = kv_exp(wave_max(tv < INFINITY ? tv : 0.0f), 7);
            vs = ldexpf(1.0f, -tex);
        }
        float mx = m;
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, s[e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float beta = __builtin_amdgcn_exp2f(m - ref);
        m = mx;
        const int ev = vs > 0.0f && vs < INFINITY ? __builtin_amdgcn_frexp_expf(vs) : kKvNoExp;
        const float alpha = ev > eR ? (eR == kKvNoExp ? 0.0f : ldexpf(beta, eR - ev)) : beta;
        const bool first = eR == kKvNoExp;
        eR = max(eR, ev);
        const float f = eR == kKvNoExp ? vs : ldexpf(vs, 15 - eR);
        h8 ph, pl;
        l *= beta;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
            const uint32_t tok = 4u * g + (e & 3u) + 16u * (e >> 2);
            const bool see = s[e] != -INFINITY;
            float p = __builtin_amdgcn_exp2f(s[e] - ref);
            if (see && ((bad >> tok) & 1u)) p = __uint_as_float(0x7fc00000u);
            l += p;
            _Float16 a, d;
            kv_split(see ? p * f : 0.0f, a, d);
            ph[e] = a;
            pl[e] = d;
        }
        if (!first)
#pragma unroll
            for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][e] *= alpha;
        if (!open) {
            const uint4* src = reinterpret_cast<const uint4*>(kv_codes(c, kv_block(c, S.seq, kvh, b)) + 32u * c.hdp) + lane;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint4 w = src[64 * t];
                const h8 a0 = kv_cvt8(w.x, w.y), a1 = kv_cvt8(w.z, w.w);
                acc[2 * t] = KV_MFMA(a0, ph, acc[2 * t]);
                acc[2 * t + 1] = KV_MFMA(a1, ph, acc[2 * t + 1]);
                acc[2 * t] = KV_MFMA(a0, pl, acc[2 * t]);
                acc[2 * t + 1] = KV_MFMA(a1, pl, acc[2 * t + 1]);
            }
        } else {
#pragma unroll
            for (int t = 0; t < 2 * NT; ++t) {
                h8 hi, lo;
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) {
                    const uint32_t tok = 4u * g + (e & 3u) + 16u * (e >> 2);
                    float x = c.tail[(row0 + min(tok, live - 1u)) * c.hdp + 16u * t + m16];
                    if (tok >= live || ((bad >> tok) & 1u)) x = 0.0f;   // 0 x NaN would be in every row's sum
                    _Float16 a, d;
                    kv_split(ldexpf(x, tex), a, d);
                    hi[e] = a;
                    lo[e] = d;
                }
                acc[t] = KV_MFMA(hi, ph, acc[t]);
                acc[t] = KV_MFMA(hi, pl, acc[t]);
                acc[t] = KV_MFMA(lo, ph, acc[t]);
            }
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0u) {
        s_m[wave][m16] = m;
        s_l[wave][m16] = l;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(s_m[0][m16], s_m[1][m16]), fmaxf(s_m[2][m16], s_m[3][m16]));
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) L += s_l[w][m16] * __builtin_amdgcn_exp2f(s_m[w][m16] - ref);
    const float mine = __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = ldexpf(acc[t][e], eR - 15) * mine;
    auto give = [&](uint32_t k) {
#pragma unroll
        for (int t = 0; t < 2 * NT; ++t) *reinterpret_cast<f4*>(&s_acc[k][m16 * kRow + 16u * t + 4u * g]) = acc[t];
    };
    auto take = [&](uint32_t k) {
#pragma unroll
        for (int t = 0; t < 2 * NT; ++t) acc[t] += *reinterpret_cast<const f4*>(&s_acc[k][m16 * kRow + 16u * t + 4u * g]);
    };
    if (wave >= 2u) give(wave - 2u);
    __syncthreads();
    if (wave < 2u) take(wave);
    __syncthreads();
    if (wave == 1u) give(0u);
    __syncthreads();
    if (wave != 0u) return;
    take(0u);
    const uint32_t r = r0 + m16;
    if (sp.n <= A.per) {   // the only split
        if (r >= R) return;
        const uint32_t qi = r / A.G, h = kvh * A.G + (r - qi * A.G);
#pragma unroll
        for (int t = 0; t < 2 * NT; ++t)
            if (16u * t + 4u * g < c.hd) kv_give(A, S.row0 + qi, h, 16u * t + 4u * g, acc[t] / L);
        if (g == 0u) kv_row_done(A, S.row0 + qi, h, M, L);
        return;
    }
    if (r >= R) return;
    const uint64_t pr = (static_cast<uint64_t>(S.part0) + (tile * c.kvh + kvh) * S.splits + split) * 16u + m16;
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t) *reinterpret_cast<f4*>(A.part + pr * c.hdp + 16u * t + 4u * g) = acc[t];
    if (g == 0u) A.part_ml[pr] = make_float2(M, L);
}

// The splits of a row tile put together: one workgroup per (row tile, head, sequence).
__global__ void __launch_bounds__(kKvThreads) k_kv8_merge(const Kv8AttnArgs A) {
    const Kv8Seq& S = A.s[blockIdx.z];
    const Kv8Dev& c = A.c;
    const uint32_t kvh = blockIdx.y, tile = blockIdx.x, R = S.n * A.G, r0 = 16u * tile;
    if (r0 >= R) return;
    const KvSpan sp = kv_span(A, S, S.pos + r0 / A.G, S.pos + min(r0 + 15u, R - 1u) / A.G);
    const uint32_t n = (sp.n + A.per - 1u) / A.per;
    if (n <= 1u) return;   // written by the only split
    const uint64_t p0 = (static_cast<uint64_t>(S.part0) + (tile * c.kvh + kvh) * S.splits) * 16u;
    const uint32_t hd4 = c.hd >> 2, rows = min(16u, R - r0);
    for (uint32_t u = threadIdx.x; u < rows * hd4; u += kKvThreads) {
        uint32_t rr, d;
        kv_unit(u, hd4, rr, d);
        float M = -INFINITY;
        for (uint32_t k = 0; k < n; ++k) M = fmaxf(M, A.part_ml[p0 + k * 16u + rr].x);
        const float ref = M == -INFINITY ? 0.0f : M;
        float L = 0.0f;
        f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t k = 0; k < n; ++k) {
            const float2 ml = A.part_ml[p0 + k * 16u + rr];
            const float w = __builtin_amdgcn_exp2f(ml.x - ref);
            L += w * ml.y;
            o += w * *reinterpret_cast<const f4*>(A.part + (p0 + k * 16u + rr) * c.hdp + d);
        }
        const uint32_t r = r0 + rr, qi = r / A.G, h = kvh * A.G + (r - qi * A.G);
        kv_give(A, S.row0 + qi, h, d, o / L);
        if (d == 0u) kv_row_done(A, S.row0 + qi, h, M, L);
    }
}

// Accumulated weights: one wave per block of positions; the scores once more, against the rows' final maxima and sums.
template <int NT, bool CAP>
__global__ void __launch_bounds__(kKvThreads) k_kv8_weights(const Kv8AttnArgs A) {
    const Kv8Seq& S = A.s[blockIdx.z];
    const Kv8Dev& c = A.c;
    const uint32_t kvh = blockIdx.y, lane = threadIdx.x & 63u, g = lane >> 4, m16 = lane & 15u;
    const uint32_t len = S.pos + S.n, R = S.n * A.G;
    const uint32_t b = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (S.n == 0u || 32u * b >= len) return;
    float w[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t r0 = 0; r0 < R; r0 += 16u) {
        const uint32_t pmin = S.pos + r0 / A.G, pmax = S.pos + min(r0 + 15u, R - 1u) / A.G;
        const bool in_pre = 32u * b < S.prefix;
        if (!in_pre && 32u * b > pmax) continue;
        if (!in_pre && A.window && pmin >= A.window && 32u * b + 31u <= pmin - A.window) break;   // and no later row sees it
        KvQuery<NT> Q;
        kv_load_q<NT>(A, S, kvh, r0, Q);
        float s[8];
        kv_scores<NT, CAP>(A, S, kvh, b, Q, true, s);
        const uint32_t r = r0 + m16;
        if (r < R) {
            const uint32_t qi = r / A.G, h = kvh * A.G + (r - qi * A.G);
            const float2 st = A.stats[(static_cast<uint64_t>(S.row0) + qi) * A.heads + h];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] += s[e] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s[e] - st.x) * st.y;
        }
    }
    const uint64_t base = (static_cast<uint64_t>(S.seq) * c.kvh + kvh) * A.max_ctx;
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e) {
        const float t = slot_sum<16>(w[e]);
        const uint32_t j = 32u * b + 4u * g + (e & 3u) + 16u * (e >> 2);
        if (m16 == 0u && j < len) A.w_out[base + j] = (A.w_in && j < S.pos ? A.w_in[base + j] : 0.0f) + t;
    }
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

constexpr uint32_t kKvSelThreads = 1024;

// One workgroup per (head, move): the key of the last weight that stays, by four passes of 8 bits, then the positions in
// order, of those with that key the first ones.
__global__ void __launch_bounds__(kKvSelThreads) k_kv8_select(const Kv8EvictArgs A) {
    __shared__ uint32_t hist[256], s_bin, s_left;
    __shared__ uint32_t wsum[2][kKvSelThreads / 64u];
    const vrt_kv8_move& V = A.m[blockIdx.y];
    const uint32_t head = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const float* src = A.w + (static_cast<uint64_t>(V.src) * A.c.kvh + head) * A.max_ctx;
    float* dst = A.w + (static_cast<uint64_t>(V.dst) * A.c.kvh + head) * A.max_ctx;
    uint32_t* kept = A.kept + (static_cast<uint64_t>(blockIdx.y) * A.c.kvh + head) * A.kept_stride;
    const uint32_t old = V.len - V.recent, want = V.keep - V.recent;
    uint32_t thr = 0u, need = want;   // keys above thr stay, and `need` of those equal to it
    if (want) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            const uint32_t high = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
            if (tid < 256u) hist[tid] = 0u;
            __syncthreads();
            for (uint32_t i = tid; i < old; i += kKvSelThreads) {
                const uint32_t k = kv_key(src[i]);
                if ((k & high) == thr) atomicAdd(&hist[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (tid == 0u) {
                uint32_t left = need, bin = 255u;
                while (hist[bin] < left) left -= hist[bin--];
                s_bin = bin;
                s_left = left;
            }
            __syncthreads();
            thr |= s_bin << shift;
            need = s_left;
            __syncthreads();
        }
        uint32_t n_kept = 0u, n_eq = 0u;   // so far
        for (uint32_t i0 = 0; i0 < old; i0 += kKvSelThreads) {
            const uint32_t i = i0 + tid;
            const float w = i < old ? src[i] : 0.0f;
            const uint32_t k = kv_key(w);
            const bool gt = i < old && k > thr, eq = i < old && k == thr;
            const uint64_t below = (1ull << lane) - 1ull, be = __ballot(eq);
            if (lane == 0u) wsum[0][wave] = __popcll(be);
            __syncthreads();
            uint32_t eq_at = n_eq + __popcll(be & below), eq_all = 0u;
            for (uint32_t v = 0; v < kKvSelThreads / 64u; ++v) {
                if (v < wave) eq_at += wsum[0][v];
                eq_all += wsum[0][v];
            }
            const bool stay = gt || (eq && eq_at < need);
            const uint64_t bs = __ballot(stay);
            if (lane == 0u) wsum[1][wave] = __popcll(bs);
            __syncthreads();
            uint32_t at = n_kept + __popcll(bs & below), all = 0u;
            for (uint32_t v = 0; v < kKvSelThreads / 64u; ++v) {
                if (v < wave) at += wsum[1][v];
                all += wsum[1][v];
            }
            if (stay) {
                kept[at] = i;
                dst[at] = w;
            }
            n_kept += all;
            n_eq += eq_all;
        }
    }
    for (uint32_t i = tid; i < V.recent; i += kKvSelThreads) {
        kept[want + i] = old + i;
        dst[want + i] = src[old + i];
    }
}

// One workgroup per (block of the destination, head and K or V, move): the kept values of the source, into a block as
// the append makes it, or into the tail.
__global__ void __launch_bounds__(kKvThreads) k_kv8_gather(const Kv8EvictArgs A) {
    __shared__ __align__(16) uint8_t img[32 * 256];
    __shared__ uint32_t red[4];
    const Kv8Dev& c = A.c;
    const vrt_kv8_move& V = A.m[blockIdx.z];
    const uint32_t head = blockIdx.y >> 1, z = blockIdx.y & 1u, b = blockIdx.x, tid = threadIdx.x;
    if (32u * b >= V.keep) return;
    const uint32_t* kept = A.kept + (static_cast<uint64_t>(blockIdx.z) * c.kvh + head) * A.kept_stride;
    const bool closed = (b + 1u) * 32u <= V.keep, tail = b + 1u >= (V.keep - 1u) >> 5;   // the last block and the one before
    KvTile T;
    const uint32_t hd4 = c.hd >> 2, units = 32u * hd4;
#pragma unroll
    for (uint32_t k = 0; k < 8u; ++k) {
        const uint32_t u = tid + kKvThreads * k;
        T.v[k] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (u >= units) continue;
        uint32_t t, d;
        kv_unit(u, hd4, t, d);
        if (32u * b + t >= V.keep) continue;
        const uint32_t p = kept[32u * b + t];
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) T.v[k][e] = kv_value(c, V.src, head, z, p, d + e, V.len);
        if (tail) *reinterpret_cast<f4*>(c.tail + kv_tail_row(c, V.dst, head, b, z, t) * c.hdp + d) = T.v[k];
    }
    if (closed) kv_close_block(c, T, kv_block(c, V.dst, head, b), z, img, red);
    if (!tail) return;
    __syncthreads();   // the tail rows are whole: their maxima, and zeros in the padding dimensions
    const uint32_t n = min(32u, V.keep - 32u * b), lane = tid & 63u;
    for (uint32_t t = tid >> 6; t < n; t += kKvThreads / 64u) {
        const uint64_t row = kv_tail_row(c, V.dst, head, b, z, t);
        f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (4u * lane < c.hd) v = *reinterpret_cast<const f4*>(c.tail + row * c.hdp + 4u * lane);
        else if (4u * lane < c.hdp) *reinterpret_cast<f4*>(c.tail + row * c.hdp + 4u * lane) = v;
        const uint32_t m = wave_max_u32(max(max(f_bits(v[0]), f_bits(v[1])), max(f_bits(v[2]), f_bits(v[3]))));
        if (lane == 0u) c.tmax[row] = __uint_as_float(m);
    }
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

// The most blocks that a row tile of a sequence sees.
uint32_t most_blocks(const Kv8Seq& s, uint32_t window) {
    const uint32_t len = s.pos + s.n, pre = std::min(s.prefix, len), all = (len + 31u) / 32u;
    if (!window) return all;
    // a tile's rows span 16 positions at most
    const uint64_t w = static_cast<uint64_t>((pre + 31u) / 32u) + (static_cast<uint64_t>(window) + 15u + 31u) / 32u + 1u;
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
    VRT_REQUIRE(std::isfinite(at->softcap) && at->softcap >= 0.0f, "%s: softcap must be finite, not negative", who);
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
    VRT_REQUIRE(*total * A.G <= 0x3fffffffu && items <= 0x3fffffffu, "%s: too many rows", who);
    *P = kv8_plan(A, c->kv_heads, z.hdp, n, *total, scored);
    return VRT_OK;
}

template <bool CAP>
const void* attn_kernel(uint32_t nt) {
    switch (nt) {
        case 1: return reinterpret_cast<const void*>(&k_kv8_attn<1, CAP>);
        case 2: return reinterpret_cast<const void*>(&k_kv8_attn<2, CAP>);
        case 3: return reinterpret_cast<const void*>(&k_kv8_attn<3, CAP>);
        case 4: return reinterpret_cast<const void*>(&k_kv8_attn<4, CAP>);
        case 5: return reinterpret_cast<const void*>(&k_kv8_attn<5, CAP>);
        case 6: return reinterpret_cast<const void*>(&k_kv8_attn<6, CAP>);
        case 7: return reinterpret_cast<const void*>(&k_kv8_attn<7, CAP>);
        default: return reinterpret_cast<const void*>(&k_kv8_attn<8, CAP>);
    }
}
template <bool CAP>
const void* weights_kernel(uint32_t nt) {
    switch (nt) {
        case 1: return reinterpret_cast<const void*>(&k_kv8_weights<1, CAP>);
        case 2: return reinterpret_cast<const void*>(&k_kv8_weights<2, CAP>);
        case 3: return reinterpret_cast<const void*>(&k_kv8_weights<3, CAP>);
        case 4: return reinterpret_cast<const void*>(&k_kv8_weights<4, CAP>);
        case 5: return reinterpret_cast<const void*>(&k_kv8_weights<5, CAP>);
        case 6: return reinterpret_cast<const void*>(&k_kv8_weights<6, CAP>);
        case 7: return reinterpret_cast<const void*>(&k_kv8_weights<7, CAP>);
        default: return reinterpret_cast<const void*>(&k_kv8_weights<8, CAP>);
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
    z.tmax = up256(heads * 128u * 4u);
    z.total = z.codes + z.scales + z.tail + z.tmax;
    return z;
}

Kv8Dev kv8_view(const Kv8Sizes& z, void* data, uint32_t kv_heads, uint32_t head_dim) {
    auto* p = static_cast<uint8_t*>(data);
    Kv8Dev d;
    d.codes = p;
    d.scales = reinterpret_cast<float2*>(p + z.codes);
    d.tail = reinterpret_cast<float*>(p + z.codes + z.scales);
    d.tmax = reinterpret_cast<float*>(p + z.codes + z.scales + z.tail);
    d.nb = z.nb;
    d.kvh = kv_heads;
    d.hd = head_dim;
    d.hdp = z.hdp;
    return d;
}

// About kKvSplits workgroups, of four blocks at least.
constexpr uint64_t kKvSplits = 1024;

Kv8Plan kv8_plan(Kv8AttnArgs& A, uint32_t kvh, uint32_t hdp, uint32_t n, uint64_t rows, bool scored) {
    Kv8Plan P{};
    uint64_t blocks = 0;   // of all row tiles and heads
    for (uint32_t i = 0; i < n; ++i)
        blocks += static_cast<uint64_t>((A.s[i].n * A.G + 15u) / 16u) * kvh * most_blocks(A.s[i], A.window);
    const uint64_t per = std::max<uint64_t>(4u, (blocks + kKvSplits - 1u) / kKvSplits);
    A.per = static_cast<uint32_t>((per + 3u) & ~3ull);
    A.splits = 1u;
    uint64_t place = 0;
    for (uint32_t i = 0; i < n; ++i) {
        Kv8Seq& s = A.s[i];
        const uint32_t tiles = (s.n * A.G + 15u) / 16u;
        s.splits = std::max(1u, (most_blocks(s, A.window) + A.per - 1u) / A.per);
        s.part0 = static_cast<uint32_t>(place);
        if (s.splits > 1u) place += static_cast<uint64_t>(tiles) * kvh * s.splits;
        A.splits = std::max(A.splits, s.splits);
        P.tiles = std::max(P.tiles, tiles);
    }
    P.part = up256(place * 16u * hdp * 4u);
    P.ml = up256(place * 16u * sizeof(float2));
    P.stats = scored ? up256(rows * A.heads * sizeof(float2)) : 0u;
    P.total = P.part + P.ml + P.stats;
    return P;
}

// (a sequence's splits are at most its blocks / per + 1, and all blocks / per at most kKvSplits)
uint64_t kv8_workspace_most(uint64_t items, uint32_t hdp, uint64_t rows, uint32_t heads) {
    const uint64_t place = kKvSplits + items;
    return up256(place * 16u * hdp * 4u) + up256(place * 16u * sizeof(float2)) + up256(rows * heads * sizeof(float2));
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
    return launch(reinterpret_cast<const void*>(&k_kv8_append), dim3(blocks, 2u * c.kvh, n), kKvThreads, A, s);
}

int kv8_attend(Kv8AttnArgs& A, const Kv8Plan& P, void* workspace, uint32_t n, hipStream_t s) {
    auto* ws = static_cast<uint8_t*>(workspace);
    A.part = reinterpret_cast<float*>(ws);
    A.part_ml = reinterpret_cast<float2*>(ws + P.part);
    A.stats = A.w_out ? reinterpret_cast<float2*>(ws + P.part + P.ml) : nullptr;
    const uint32_t nt = A.c.hdp / 32u;
    const bool cap = A.cap > 0.0f;
    if (int rc = launch(cap ? attn_kernel<true>(nt) : attn_kernel<false>(nt), dim3(P.tiles * A.splits, A.c.kvh, n), kKvThreads, A, s))
        return rc;
    if (A.splits > 1u)
        if (int rc = launch(reinterpret_cast<const void*>(&k_kv8_merge), dim3(P.tiles, A.c.kvh, n), kKvThreads, A, s)) return rc;
    if (!A.w_out) return VRT_OK;
    uint32_t len = 0;
    for (uint32_t i = 0; i < n; ++i)
        if (A.s[i].n) len = std::max(len, A.s[i].pos + A.s[i].n);
    return launch(cap ? weights_kernel<true>(nt) : weights_kernel<false>(nt), dim3((len + 127u) / 128u, A.c.kvh, n), kKvThreads, A, s);
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
    return launch(reinterpret_cast<const void*>(&k_kv8_gather), dim3((keep + 31u) / 32u, 2u * c.kvh, n), kKvThreads, A, s);
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
    return launch(reinterpret_cast<const void*>(&k_kv8_read), dim3(blocks, 2u * A.c.kvh, n_seqs), kKvThreads, A, ctx->stream);
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
