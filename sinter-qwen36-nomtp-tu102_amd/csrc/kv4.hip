// The 4-bit paged KV cache of a batch of sequences: q/k norm and rotation at
// the batch's positions, the quantising append, the read back and causal
// attention over the cache (sinter_kv4_*, include/sinter.h).
//
//   kv4_prep_kernel    RMSNorm + NEOX RoPE of q and k heads
//   kv4_append_kernel  k, v rows quantised into the cache's pages
//   kv4_read_kernel    cache rows back to f32 / f16 / bf16
//   kv4_split_kernel   attention of 16 (token, head) rows over a part of the cache rows
//   kv4_merge_kernel   the parts of a row joined
//   kv4_tile_kernel    attention of 128 or 256 rows of one sequence over a chunk
//   kv4_join_kernel    its chunks joined
//
// A page holds per kv head page_rows rows of codes (hd / 2 bytes; byte 16 b +
// i of a row holds elements 32 b + i and 32 b + 16 + i in its low and high
// four bits), then page_rows rows of hd / 32 f16 scales: both planes are whole
// 16-byte units, contiguous over a page, so that a wave streams them by
// LDS-DMA with nothing read twice.  Element = scale * (code - 8).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dev_common.h"
#include "internal.h"

namespace sinter {

// the first device error of this unit's kernels: [0] code, [1] aux (a sequence)
__device__ unsigned g_kv4_err[2];

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f16x2 pair_of(uint32_t w) { return __builtin_bit_cast(f16x2, w); }
typedef uint16_t __attribute__((may_alias)) u16a;   // (written as halves, read as wider words)
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float F16_MAX = 65504.0f;
constexpr float REF_NONE = -1e30f;   // the softmax reference of a row that has seen nothing

// ------------------------------------------------------------------ rows of any type

__device__ __forceinline__ float4 cvt4(u32x2 u, uint32_t type) {
    if (type == SINTER_BF16)
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xffff0000u));
    return make_float4(h2f((uint16_t)u.x), h2f((uint16_t)(u.x >> 16)), h2f((uint16_t)u.y), h2f((uint16_t)(u.y >> 16)));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, uint32_t type) {
    if (type == SINTER_BF16) {   // (one instruction, to nearest even)
        const bf16x2 v = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
    return (uint32_t)f2h(a) | ((uint32_t)f2h(b) << 16);
}
// four elements at element `e` (a multiple of 4) of a buffer of `type`
__device__ __forceinline__ float4 load4(const void *p, int64_t e, uint32_t type) {
    if (type == SINTER_F32) return *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + e);
    return cvt4(*reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(p) + e), type);
}
__device__ __forceinline__ void store4(void *p, int64_t e, uint32_t type, float4 v) {
    if (type == SINTER_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p) + e) = v;
        return;
    }
    const u32x2 u = {pack2(v.x, v.y, type), pack2(v.z, v.w, type)};
    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p) + e) = u;
}

// Four elements as they lie: loads are issued together, conversions come later
template <uint32_t T>
struct Raw4 {
    typename std::conditional<T == SINTER_F32, f32x4, u32x2>::type v;
    __device__ __forceinline__ void load(const void *p, int64_t e) {
        if constexpr (T == SINTER_F32) v = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + e);
        else v = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(p) + e);
    }
    __device__ __forceinline__ float4 get() const {
        if constexpr (T == SINTER_F32) return make_float4(v.x, v.y, v.z, v.w);
        else return cvt4(v, T);
    }
};

// ------------------------------------------------------------------ the batch

// The first of 64 sequences among which token t's is (wave-uniform), or any if
// it has none: 64 starts are compared at a time, so that of up to 4096
// sequences one load finds the 64 (the append of one row of 2048 sequences, 8
// heads of 128: 18 us, 31 with a look through all of them).
__device__ __forceinline__ uint32_t seq_base(const sinter_kv4_batch &b, uint32_t t) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t base = 0, span = b.n_seq;
    while (span > 64) {
        const uint32_t stride = (span + 63) / 64, i = base + lane * stride;
        const bool before = lane * stride < span && b.tok_start[min(i, b.n_seq)] <= (int)t;
        const uint32_t c = (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(before)), at = c ? (c - 1) * stride : 0u;
        base += at;
        span = min(stride, span - at);
    }
    return base;
}

// the sequence that token t belongs to (wave-uniform), or -1
__device__ __forceinline__ int seq_of(const sinter_kv4_batch &b, uint32_t t) {
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t base = seq_base(b, t); base < b.n_seq; base += 64) {
        const uint32_t i = min(base + lane, b.n_seq - 1u);
        const bool past = base + lane < b.n_seq && b.tok_start[i + 1] > (int)t;
        const uint64_t m = __builtin_amdgcn_ballot_w64(past);
        if (m != 0) {
            const uint32_t s = base + (uint32_t)__builtin_ctzll(m);
            return b.tok_start[s] <= (int)t ? (int)s : -1;
        }
    }
    return -1;
}

// Where tokens t0 .. t0 + n - 1 (n <= 64) stand: lane k gets token t0 + k's
// sequence and position (-1 where it has none: behind the last sequence, or
// before row 0 of its own).  Sixty-four sequences' bounds are loaded at once
// and the tokens found among them without further loads.
__device__ __forceinline__ void token_places(const sinter_kv4_batch &b, uint32_t t0, uint32_t n, int &seq, int &pos) {
    const uint32_t lane = threadIdx.x & 63u;
    seq = pos = -1;
    uint32_t k = 0;
    for (uint32_t base = seq_base(b, t0); base < b.n_seq && k < n; base += 64) {
        const uint32_t i = min(base + lane, b.n_seq - 1u);
        const int start = b.tok_start[i], stop = b.tok_start[i + 1], len = b.kv_len[i];
        for (; k < n; k++) {
            const int t = (int)(t0 + k);
            const uint64_t m = __builtin_amdgcn_ballot_w64(base + lane < b.n_seq && stop > t);
            if (m == 0) break;   // (in the next sequences, or behind all)
            const int l = __builtin_ctzll(m);
            if (__builtin_amdgcn_readlane(start, l) > t) continue;
            const int p = __builtin_amdgcn_readlane(len, l) - (__builtin_amdgcn_readlane(stop, l) - t);
            if (lane == k && p >= 0) {
                seq = (int)base + l;
                pos = p;
            }
        }
    }
}

// Tokens a workgroup of append and read takes at most: their places are found
// together (reading 20 sequences, F32: 4 tokens 68 us, 8 71 us, 16 83 us, one 98)
constexpr uint32_t TOKS = 4;

// The cache rows of tokens t0 .. t0 + n - 1 (n <= TOKS) for a workgroup: byte
// offset of their page (or -1: none, with the error raised where the table has
// no page for a row) and row in it.
struct TokRows {
    uint64_t page[TOKS];
    uint32_t row[TOKS];
};
__device__ __forceinline__ void token_rows(const sinter_kv4_batch &b, uint32_t t0, uint32_t n, size_t page_bytes, TokRows &rows) {
    if (threadIdx.x < 64) {
        int seq, pos;
        token_places(b, t0, n, seq, pos);
        if (threadIdx.x < n) {
            int page = -1;
            if (pos >= 0) {
                const uint32_t e = (uint32_t)pos / b.page_rows;
                page = e < b.max_pages ? b.pages[(size_t)seq * b.max_pages + e] : -1;
                if ((uint32_t)page >= b.n_pages) {
                    raise_error(g_kv4_err, SINTER_E_BAD_SHAPE, (unsigned)seq);
                    page = -1;
                }
            }
            rows.page[threadIdx.x] = page < 0 ? ~0ull : (uint64_t)(uint32_t)page * page_bytes;
            rows.row[threadIdx.x] = page < 0 ? 0u : (uint32_t)pos & (b.page_rows - 1u);
        }
    }
    __syncthreads();
}

// ------------------------------------------------------------------ prep

struct Prep {
    sinter_kv4_batch b;
    sinter_heads q, q_out, k, k_out;
    const float *q_norm, *k_norm;
    double rate;   // log2(base) / (rope_dims / 2)
    uint32_t nq, nk, half;
    float eps, inv_hd;
};

// y = x / sqrt(mean(x^2) + eps) * w, then the pairs (i, i + half) turned by
// pos * base^(-i / half).  The angle is held in turns in fp64 (at position
// 131072 an fp32 angle is off by thousandths of a radian), once a token and
// workgroup.  A head is hd / 8 lanes of two times four elements: those of a
// pair in one lane, so that nothing moves between lanes but the sum of
// squares.  A wave takes `per` heads of one kind at a time; blockIdx.y: a
// workgroup's share of them.
// The heads' loads are issued before the angles, whose fp64 the time is for
// few tokens (one token of 24 + 4 heads of 256: 4 us of the kernel, all
// latency).  Of many the rows' traffic: 2557 tokens of 28 heads of 256, bf16,
// 73 MB in and out in 16 us, 4.6 TB/s where a copy reaches 5.2 (with a pair's
// halves in two lanes and four elements a lane 26 us, bound by instructions;
// the weights read again for every head 8 % more).
template <uint32_t T>
__global__ __launch_bounds__(256) void kv4_prep_kernel(Prep a) {
    __shared__ float2 turn[128];
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 63u;
    const uint32_t hd = a.b.hd, lph = hd / 8, l = lane % lph, hl = lane / lph, per = 64 / lph;
    const uint32_t quarter = a.half / 4, step = gridDim.y * 4;
    const uint32_t first = blockIdx.y * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t uq = (a.nq + per - 1) / per, units = uq + (a.nk + per - 1) / per;
    const bool in = l < quarter;   // (its eight elements are four pairs)
    const uint32_t e0 = in ? 4 * l : 8 * l, e1 = in ? e0 + a.half : e0 + 4;
    struct X { Raw4<T> lo, hi; };
    auto fetch = [&](uint32_t u) {
        X x = {};
        const bool isq = u < uq;
        const uint32_t h = (isq ? u : u - uq) * per + hl;
        const sinter_heads &p = isq ? a.q : a.k;
        if (u < units && h < (isq ? a.nq : a.nk)) {
            const int64_t at = (int64_t)t * p.ld + (int64_t)h * p.hs;
            x.lo.load(p.p, at + e0);
            x.hi.load(p.p, at + e1);
        }
        return x;
    };
    // (a token that is nobody's has its row in the arrays too)
    X x0 = fetch(first), x1 = fetch(first + step);
    float4 w[2][2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float *n = k ? a.k_norm : a.q_norm;
        w[k][0] = w[k][1] = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (n) {
            w[k][0] = *reinterpret_cast<const float4 *>(n + e0);
            w[k][1] = *reinterpret_cast<const float4 *>(n + e1);
        }
    }
    int seq, pos;
    token_places(a.b, t, 1, seq, pos);
    pos = __builtin_amdgcn_readfirstlane(pos);
    if (pos < 0) return;   // (uniform)
    if (threadIdx.x < a.half) {
        const double f = exp2(-(double)threadIdx.x * a.rate) * 0.15915494309189533577;   // 1 / (2 pi)
        const double y = (double)pos * f, fr = y - rint(y);
        double s, c;
        sincospi(2.0 * fr, &s, &c);
        turn[threadIdx.x] = make_float2((float)c, (float)s);
    }
    __syncthreads();
    float2 cs[4];
#pragma unroll
    for (uint32_t c = 0; c < 4; c++) cs[c] = in ? turn[4 * l + c] : make_float2(1.0f, 0.0f);
    for (uint32_t u = first; u < units; u += step) {
        const float4 lo = x0.lo.get(), hi = x0.hi.get();
        x0 = x1;
        x1 = fetch(u + 2 * step);
        const float ss = lanes_sum_f32((lo.x * lo.x + lo.y * lo.y + (lo.z * lo.z + lo.w * lo.w)) + (hi.x * hi.x + hi.y * hi.y + (hi.z * hi.z + hi.w * hi.w)), lph);
        const float r = 1.0f / sqrtf(ss * a.inv_hd + a.eps);
        float y[8] = {lo.x * r, lo.y * r, lo.z * r, lo.w * r, hi.x * r, hi.y * r, hi.z * r, hi.w * r};
        const bool isq = u < uq;
        auto weigh = [&](const float4 &w0, const float4 &w1) {
            y[0] *= w0.x; y[1] *= w0.y; y[2] *= w0.z; y[3] *= w0.w;
            y[4] *= w1.x; y[5] *= w1.y; y[6] *= w1.z; y[7] *= w1.w;
        };
        if (isq) weigh(w[0][0], w[0][1]);
        else weigh(w[1][0], w[1][1]);
        if (in) {
#pragma unroll
            for (uint32_t c = 0; c < 4; c++) {
                const float p = y[c], o = y[c + 4];
                y[c] = p * cs[c].x - o * cs[c].y;
                y[c + 4] = o * cs[c].x + p * cs[c].y;
            }
        }
        const uint32_t h = (isq ? u : u - uq) * per + hl;
        if (h < (isq ? a.nq : a.nk)) {
            const sinter_heads &p = isq ? a.q_out : a.k_out;
            const int64_t at = (int64_t)t * p.ld + (int64_t)h * p.hs;
            store4(p.p, at + e0, T, make_float4(y[0], y[1], y[2], y[3]));
            store4(p.p, at + e1, T, make_float4(y[4], y[5], y[6], y[7]));
        }
    }
}

// ------------------------------------------------------------------ append

struct Rows {
    sinter_kv4_batch b;
    sinter_heads k, v;
    uint32_t toks, parts;   // tokens a workgroup; workgroups that share them
};

// Four lanes quantise one block of 32, eight elements each: m = the first
// element of the largest magnitude (saturated at the f16 maximum), d = m / -8,
// code = min(15, trunc(x / d + 8.5)) by the product with 1 / d, in fp32 with
// every product and sum rounded.  A block
// whose f16 scale is zero has every code 8; one with a NaN has a NaN scale.
// A workgroup takes several tokens, whose places are found together, and four
// blocks' loads at a time.  Bound by instructions (about 200 for a wave's 16
// blocks, ten of the time's microseconds) before the rows' traffic: 32 MB of
// bf16 rows of 8 heads of 128 into 9 MB of pages in 15 us, 2.7 TB/s (eight lanes a block, each with its own division and search: 20 us; a
// workgroup a token, one block's loads at a time, 24 us).
template <uint32_t T>
__global__ __launch_bounds__(256) void kv4_append_kernel(Rows a) {
    __shared__ TokRows tok;
    const uint32_t nb = a.b.hd / 32, nblk = a.b.nkv * nb, rows = a.b.page_rows, hb = a.b.hd / 2;
    const size_t head_bytes = (size_t)rows * (hb + hb / 8);
    const uint32_t grp = blockIdx.x / a.parts, part = blockIdx.x % a.parts, t0 = grp * a.toks, n = min(a.toks, a.b.n_tok - t0);
    token_rows(a.b, t0, n, head_bytes * a.b.nkv, tok);
    // block j of a token (K's, then V's) stays with its four lanes, token after token
    const uint32_t l4 = threadIdx.x & 3u, wide = min(2 * nblk, 64u), step = 64u / wide, k0 = threadIdx.x / 4u / wide;
    if (k0 >= step) return;
    for (uint32_t j0 = part * wide + threadIdx.x / 4u % wide; j0 < 2 * nblk; j0 += wide * a.parts) {
        const bool isv = j0 >= nblk;
        const uint32_t j = isv ? j0 - nblk : j0, g = j / nb, bl = j % nb;
        const int64_t ld = isv ? a.v.ld : a.k.ld, at0 = (int64_t)g * (isv ? a.v.hs : a.k.hs) + 32 * bl + 8 * l4;
        const void *src = isv ? a.v.p : a.k.p;
        unsigned char *plane = static_cast<unsigned char *>(isv ? a.b.vc : a.b.kc) + g * head_bytes;
        for (uint32_t kb = k0; kb < n; kb += 4 * step) {
            Raw4<T> in[4][2];
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) {
                const int64_t at = (int64_t)(t0 + min(kb + u * step, n - 1u)) * ld + at0;
                in[u][0].load(src, at);
                in[u][1].load(src, at + 4);
            }
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) {
                const uint32_t k = kb + u * step;
                if (k >= n || tok.page[k] == ~0ull) continue;   // (the same for a block's four lanes)
                const float4 f0 = in[u][0].get(), f1 = in[u][1].get();
                float x[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
                int nan = 0;
#pragma unroll
                for (int c = 0; c < 8; c += 2) nan |= __builtin_isunordered(x[c], x[c + 1]);
                float hi = -F16_MAX, lo = F16_MAX;   // (a NaN leaves them)
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    x[c] = __builtin_amdgcn_fmed3f(x[c], -F16_MAX, F16_MAX);
                    hi = fmaxf(hi, x[c]);
                    lo = fminf(lo, x[c]);
                }
                hi = fmaxf(hi, dpp_f<DPP_XOR1>(hi));
                lo = fminf(lo, dpp_f<DPP_XOR1>(lo));
                nan |= dpp_i<DPP_XOR1>(nan);
                hi = fmaxf(hi, dpp_f<DPP_XOR2>(hi));
                lo = fminf(lo, dpp_f<DPP_XOR2>(lo));
                nan |= dpp_i<DPP_XOR2>(nan);
                bool pos = hi > -lo;
                if (__builtin_amdgcn_ballot_w64(hi == -lo) != 0) {   // both signs have the largest magnitude: which comes first
                    int at = 64;
#pragma unroll
                    for (int c = 7; c >= 0; c--)
                        if (fabsf(x[c]) == hi) at = 2 * (int)(8 * l4 + c) + (x[c] > 0.0f ? 1 : 0);
                    at = min(at, dpp_i<DPP_XOR1>(at));
                    at = min(at, dpp_i<DPP_XOR2>(at));
                    if (hi == -lo) pos = at & 1;
                }
                const float d = (pos ? hi : lo) / -8.0f;
                uint16_t dh = f2h(d);
                const bool zero = (dh & 0x7fffu) == 0;
                if (zero) dh = 0;
                if (nan) dh = 0x7e00u;
                const float inv = zero ? 0.0f : 1.0f / d;
                uint32_t q[2];
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    q[p] = 0;
#pragma unroll
                    for (int c = 0; c < 4; c++) q[p] |= (uint32_t)(int)(x[4 * p + c] * inv + 8.5f) << (8 * c);
                    q[p] -= (q[p] >> 4) & 0x01010101u;   // (16 is 15)
                    if (nan) q[p] = 0x08080808u;
                    // lane l4 < 2 joins lane l4 + 2's codes (elements 16 further) above its own
                    q[p] |= (uint32_t)dpp_i<DPP_XOR2>((int)q[p]) << 4;
                }
                unsigned char *head = plane + tok.page[k];
                const uint32_t row = tok.row[k];
                if (l4 < 2) *reinterpret_cast<u32x2 *>(head + (size_t)row * hb + 16 * bl + 8 * l4) = u32x2{q[0], q[1]};
                if (l4 == 0) *reinterpret_cast<uint16_t *>(head + (size_t)rows * hb + (size_t)row * (hb / 8) + 2 * bl) = dh;
            }
        }
    }
}

// ------------------------------------------------------------------ read

// A thread gives back EL consecutive elements, 16 bytes of F32 (EL = 4) or of a
// 16-bit type (8): the low or the high four bits of EL code bytes, so that a
// wave's stores are consecutive (the two halves of a block read its bytes
// twice, the second time from the cache); four of them in flight.  Bound by the
// stores: 47 MB of pages and 240 MB of F32 rows in 55 us, 5.2 TB/s, a copy's
// rate (a workgroup a token, the two halves' stores apart: 85 us).
template <uint32_t T>
__global__ __launch_bounds__(256) void kv4_read_kernel(Rows a) {
    constexpr uint32_t EL = T == SINTER_F32 ? 4 : 8;
    __shared__ TokRows tok;
    const uint32_t rows = a.b.page_rows, hb = a.b.hd / 2, uh = a.b.hd / EL, half = a.b.nkv * uh;   // units a head, a token's K or V
    const size_t head_bytes = (size_t)rows * (hb + hb / 8);
    const uint32_t grp = blockIdx.x / a.parts, part = blockIdx.x % a.parts, t0 = grp * a.toks, n = min(a.toks, a.b.n_tok - t0);
    token_rows(a.b, t0, n, head_bytes * a.b.nkv, tok);
    // unit j of a token (K's, then V's) stays with its thread, token after token
    const uint32_t upt = (a.k.p && a.v.p ? 2u : 1u) * half, wide = min(upt, 256u), step = 256u / wide, k0 = threadIdx.x / wide;
    if (k0 >= step) return;
    for (uint32_t j0 = part * wide + threadIdx.x % wide; j0 < upt; j0 += wide * a.parts) {
        const bool isv = j0 >= half || !a.k.p;
        const uint32_t j = j0 >= half ? j0 - half : j0, g = j / uh, e = EL * (j % uh), sh = e & 16u ? 4u : 0u;
        const unsigned char *codes = static_cast<const unsigned char *>(isv ? a.b.vc : a.b.kc) + g * head_bytes + 16 * (e / 32) + e % 16;
        const unsigned char *scales = codes - 16 * (e / 32) - e % 16 + (size_t)rows * hb + 2 * (e / 32);
        const sinter_heads &dst = isv ? a.v : a.k;
        for (uint32_t kb = k0; kb < n; kb += 4 * step) {
            u32x2 w[4];
            uint16_t sc[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) {
                const uint32_t k = min(kb + u * step, n - 1u), row = tok.row[k];
                const uint64_t page = tok.page[k] == ~0ull ? 0 : tok.page[k];   // (a row without a page: page 0's, not kept)
                const unsigned char *c = codes + page + (size_t)row * hb;
                if constexpr (EL == 8) w[u] = *reinterpret_cast<const u32x2 *>(c);
                else w[u].x = *reinterpret_cast<const uint32_t *>(c);
                sc[u] = *reinterpret_cast<const uint16_t *>(scales + page + (size_t)row * (hb / 8));
            }
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) {
                const uint32_t k = kb + u * step;
                if (k >= n || tok.page[k] == ~0ull) continue;
                const int64_t to = (int64_t)(t0 + k) * dst.ld + (int64_t)g * dst.hs + e;
                const float d = h2f(sc[u]);
                float v[EL];
#pragma unroll
                for (uint32_t i = 0; i < EL; i++) v[i] = (float)((int)(((i < 4 ? w[u].x : w[u].y) >> (8 * (i & 3u) + sh)) & 15u) - 8) * d;
                if constexpr (EL == 4) {
                    *reinterpret_cast<float4 *>(static_cast<float *>(dst.p) + to) = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    const u32x4 o = {pack2(v[0], v[1], T), pack2(v[2], v[3], T), pack2(v[4], v[5], T), pack2(v[6], v[7], T)};
                    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(dst.p) + to) = o;
                }
            }
        }
    }
}

// ------------------------------------------------------------------ attention

constexpr uint32_t TILE = 32;   // cache rows a tile
// Of kv4_split_kernel (27B heads, F32): tiles a slot takes at least, one a wave
// (a reply behind 600 rows: 12.4 us, 8 tiles 14.2, 16 18.6); tiles up to which a
// segment is not divided (64 replies behind 400 rows: 23 us, up to 8 31; a reply
// behind 1000: 14, up to 32 24); and the tiles more a slot may get so that it has
// one segment only (4 to 16 measure alike)
constexpr uint32_t CT_MIN = 4, WHOLE = 16, OWN_MORE = 8;

struct Attn {
    sinter_kv4_batch b;
    sinter_heads q, gate, out;
    float *part;     // [slot][2][kv head][16][hd] unnormalised sums
    float2 *ml;      // [slot][2][kv head][16] reference and weight sum
    float *tpart;    // kv4_tile_kernel's: [tile][kv head][chunk][tile rows][hd]
    float2 *tml;
    uint32_t nq, gqa, max_q, max_kv, n_slots, type, page_shift;
    uint32_t n_tile, n_split, report;   // kv4_tile_kernel: row tiles and chunks; report the errors of lengths
    uint32_t split_rows;   // sequences of up to these rows are kv4_split_kernel's (0: it is not launched)
    uint32_t gqa_inv;   // ceil(2^32 / gqa), gqa > 1
    float qscale;    // scale * log2(e)
};

// The sequences of a call go two ways by their rows, (token, q head of a kv
// head) pairs: few to kv4_split_kernel, which streams the cache past 16 rows,
// many to kv4_tile_kernel, whose waves share a tile's codes once unpacked.
// SPLIT_ROWS: up to there the first is the faster one in any batch (8 sequences
// of 48 rows behind 5000, 27B heads, F32: 52 us, the other 139; 32 of 96 rows
// behind 2000, bf16: 124 and 143; of 192 rows 207 and 152).  SPLIT_MOST: where
// all of a batch is little work, which leaves the second's workgroups too few
// (one sequence of 252 rows behind 1000, F32: 24 us and 41).
constexpr uint32_t SPLIT_ROWS = 96, SPLIT_MOST = 256;

struct Work {
    int seq, len, tok0, n_new;   // the sequence: rows, first token, tokens (seq < 0: none)
    uint32_t item, first, count; // the item of it, the number of its item 0, its items
    uint32_t base, before;       // a sequence to look on from, the items before it
};

// the most rows of a sequence that the launch and the page table have room for
__device__ __forceinline__ uint32_t row_cap(const Attn &a) {
    return (uint32_t)min((uint64_t)a.max_kv, (uint64_t)a.b.max_pages << a.page_shift);
}

// sequence s: its rows, first token and tokens (0: none, or none of them within
// the arrays).  report: raise the error of lengths over the bounds
__device__ __forceinline__ void load_one(const Attn &a, uint32_t s, bool report, int &len, int &t0, int &n) {
    const uint32_t i = min(s, a.b.n_seq - 1u);
    t0 = a.b.tok_start[i];
    n = a.b.tok_start[i + 1] - t0;
    len = a.b.kv_len[i];
    if (s >= a.b.n_seq) n = 0;
    if (report && n > 0 && (len < 0 || (uint32_t)len > row_cap(a) || (uint32_t)n > a.max_q || t0 < 0 ||
                            (uint32_t)t0 + (uint32_t)n > a.b.n_tok))
        raise_error(g_kv4_err, SINTER_E_BAD_SHAPE, s);
    if (t0 < 0 || n <= 0 || (uint32_t)t0 >= a.b.n_tok) n = 0;
    else n = min(n, (int)(a.b.n_tok - (uint32_t)t0));
    len = max(0, len);
}

// sequence base + lane
__device__ __forceinline__ void load_seq(const Attn &a, uint32_t base, bool report, int &len, int &t0, int &n) {
    load_one(a, base + (threadIdx.x & 63u), report, len, t0, n);
}

// inclusive sum over the lanes (every lane active)
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
    auto step = [&](auto ctrl, auto rows) {
        v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    };
    using std::integral_constant;
    const integral_constant<int, 0xf> all;
    step(integral_constant<int, 0x111>{}, all);   // row_shr 1, 2, 4, 8
    step(integral_constant<int, 0x112>{}, all);
    step(integral_constant<int, 0x114>{}, all);
    step(integral_constant<int, 0x118>{}, all);
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});   // row_bcast 15 into rows 1 and 3
    step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});   // row_bcast 31 into rows 2 and 3
    return v;
}

__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(v), 63); }

// Of the 64 sequences from `base` on (a lane's: rows, first token, tokens, items
// c from number lo on), the one that has item `id`, or (by_seq) sequence `id`.
__device__ __forceinline__ bool pick(Work &w, uint32_t base, uint32_t id, bool by_seq, int len, int t0, int n, uint32_t c,
                                     uint32_t lo) {
    const bool mine = c > 0 && (by_seq ? base + (threadIdx.x & 63u) == id : id >= lo && id < lo + c);
    const uint64_t m = __builtin_amdgcn_ballot_w64(mine);
    if (m == 0) return false;
    const int l = __builtin_ctzll(m);
    w.seq = (int)base + l;
    w.len = __builtin_amdgcn_readlane(len, l);
    w.tok0 = __builtin_amdgcn_readlane(t0, l);
    w.n_new = __builtin_amdgcn_readlane(n, l);
    w.first = (uint32_t)__builtin_amdgcn_readlane((int)lo, l);
    w.count = (uint32_t)__builtin_amdgcn_readlane((int)c, l);
    w.item = by_seq ? 0u : id - w.first;
    return true;
}
// The sequences' items, count(len, n) each, numbered one sequence after the
// other: item `id`'s sequence, or (by_seq) sequence `id` with its item 0.
// from: an earlier result, whose place the search starts at.
template <class Count>
__device__ __forceinline__ Work locate(const Attn &a, uint32_t id, bool by_seq, Count count, const Work *from = nullptr) {
    Work w;
    w.seq = -1;
    w.base = from ? from->base : 0u;
    w.before = from ? from->before : 0u;
    for (; w.base < a.b.n_seq; w.base += 64) {
        int len, t0, n;
        load_seq(a, w.base, false, len, t0, n);
        const uint32_t c = n > 0 ? count(len, n) : 0u, sum = wave_scan_u32(c);
        if (pick(w, w.base, id, by_seq, len, t0, n, c, w.before + sum - c)) return w;
        w.before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    }
    return w;
}
// raise the error of lengths over the bounds
__device__ __forceinline__ void report_lengths(const Attn &a) {
    for (uint32_t base = 0; base < a.b.n_seq; base += 64) {
        int len, t0, n;
        load_seq(a, base, true, len, t0, n);
    }
}

__device__ __forceinline__ bool is_split(const Attn &a, int n) { return (uint32_t)n * a.gqa <= a.split_rows; }

// kv4_split_kernel's work is a list of segments, a segment being 16 rows of a
// sequence and its cache tiles (at least one), those of a sequence one after the
// other, counted in units of `tiles` tiles; a segment of up to WHOLE tiles is not
// divided.  Slot i takes units [i share, (i + 1) share), an undivided segment
// being the slot's that has its first.
struct Deal { uint32_t total, tiles, share; };
__device__ __forceinline__ uint32_t row_tiles(const Attn &a, int n) { return n > 0 && is_split(a, n) ? ((uint32_t)n * a.gqa + 15u) / 16u : 0u; }
__device__ __forceinline__ uint32_t seg_tiles(const Attn &a, int len) { return max(1u, (min((uint32_t)len, row_cap(a)) + TILE - 1u) / TILE); }
__device__ __forceinline__ uint32_t seg_units(uint32_t tiles, uint32_t per) {
    return per == 1u ? tiles : tiles <= WHOLE ? 1u : (tiles + per - 1u) / per;
}
// x / n rounded up, of uniform values (or a little more where x passes 2^22).
// Short: a call's first instructions are fetched as they are run, and a
// microsecond of a reply's 13 was this code's length
__device__ __forceinline__ uint32_t share_of(uint32_t x, uint32_t n) {
    uint32_t q = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)((float)x * __builtin_amdgcn_rcpf((float)n)));
    while (q * n < x) q++;
    return q;
}
// Where it makes the slots little longer a unit is a slot's share: none then has
// two segments, each with its start and end (8 replies of 4 tokens behind 5000
// rows, 27B heads, F32: 39.0 us, without 42.4).  Else a unit is a tile, in equal
// shares; of many segments at least their mean, so that the undivided start
// where a slot does (64 replies behind 400 rows: 18 us, without 23).
__device__ __forceinline__ Deal deal_of(const Attn &a, uint32_t total, uint32_t segs) {
    Deal d = {total, 1, 1};
    if (segs < a.n_slots) {
        // (segments' units are at most (total - segs) / tiles + segs)
        d.tiles = max(CT_MIN, share_of(total - segs, a.n_slots - segs));
        if (d.tiles <= OWN_MORE || (float)(d.tiles - OWN_MORE) * (float)a.n_slots <= (float)total) return d;
        d.tiles = 1;
    }
    d.share = max(1u, share_of(total, a.n_slots));
    if (segs * a.b.nkv >= 256u) d.share = max(d.share, min(WHOLE, share_of(total, segs)));
    return d;
}
__device__ __forceinline__ Work find_units(const Attn &a, const Deal &d, uint32_t id, bool by_seq, const Work *from = nullptr) {
    return locate(a, id, by_seq, [&](int len, int n) { return row_tiles(a, n) * seg_units(seg_tiles(a, len), d.tiles); }, from);
}
// The deal, and the work at slot `id`'s first unit or (by_seq) of sequence `id`.
__device__ __forceinline__ Work deal(const Attn &a, uint32_t id, bool by_seq, Deal &d) {
    int len, t0, n;
    if (a.b.n_seq <= 64) {   // (a lane holds every sequence)
        load_seq(a, 0, false, len, t0, n);
        const uint32_t mts = row_tiles(a, n), tiles = seg_tiles(a, len);
        d = deal_of(a, wave_sum_u32(mts * tiles), wave_sum_u32(mts));
        const uint32_t c = mts * seg_units(tiles, d.tiles), sum = wave_scan_u32(c);
        d.total = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        Work w;
        w.seq = -1;
        w.base = w.before = 0;
        pick(w, 0, by_seq ? id : id * d.share, by_seq, len, t0, n, c, sum - c);
        return w;
    }
    // More: a lane counts `per` sequences in a row (eight loads in flight), and
    // the search goes through one lane's (2048 replies behind 300 rows, 32 heads of
    // 128 over 8, bf16: 272 us, sixty-four at a time, one load after the other, 280)
    const uint32_t lane = threadIdx.x & 63u, per = (a.b.n_seq + 63u) / 64u;
    uint32_t mine = 0, segs = 0;
#pragma unroll 8
    for (uint32_t i = 0; i < per; i++) {
        load_one(a, lane * per + i, false, len, t0, n);
        const uint32_t mts = row_tiles(a, n);
        mine += mts * seg_tiles(a, len);
        segs += mts;
    }
    d = deal_of(a, wave_sum_u32(mine), wave_sum_u32(segs));
    if (d.tiles > 1u) {
        mine = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < per; i++) {
            load_one(a, lane * per + i, false, len, t0, n);
            mine += row_tiles(a, n) * seg_units(seg_tiles(a, len), d.tiles);
        }
    }
    const uint32_t sum = wave_scan_u32(mine), at = by_seq ? id : id * d.share;
    d.total = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    const uint64_t m = __builtin_amdgcn_ballot_w64(by_seq ? id >= lane * per && id < (lane + 1u) * per : at >= sum - mine && at < sum);
    Work from;
    from.base = a.b.n_seq;   // (none)
    from.before = 0;
    if (m != 0) {
        const int l = __builtin_ctzll(m);
        from.base = (uint32_t)l * per;
        from.before = (uint32_t)__builtin_amdgcn_readlane((int)(sum - mine), l);
    }
    return find_units(a, d, at, by_seq, &from);
}

// the gated, normalised output of four elements
__device__ __forceinline__ void store_out(const Attn &a, int64_t t, int64_t h, uint32_t e, f32x4 o, float l) {
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    float4 y = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    if (a.gate.p) {
        const float4 z = load4(a.gate.p, t * a.gate.ld + h * a.gate.hs + e, a.type);
        auto sig = [](float x) { return 1.0f / (1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f)); };
        y = make_float4(y.x * sig(z.x), y.y * sig(z.y), y.z * sig(z.z), y.w * sig(z.w));
    }
    store4(a.out.p, t * a.out.ld + h * a.out.hs + e, a.type, y);
}

// one LDS-DMA of 16 bytes a lane from per-lane addresses (lane l's land at lds_base + 16 l)
__device__ __forceinline__ void lds_dma16v(uint64_t addr, uint32_t lds_base) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, off\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(lds_base), "v"(addr)
        : "memory");
}

// Eight codes as f16 integers -8..7: the low (or high) four bits of two words'
// bytes, in the order bytes 0 2 1 3 of `x`, then of `y`.  0x6400 | q is 1024 +
// q; in the high bits 1024 + 16 q, brought down by an exact product and sum.
// (one v_and_or_b32, its constants in registers: the compiler's choice is an
// and and an or with a literal each)
__device__ __forceinline__ f16x2 and_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(bits));
    return pair_of(r);
}
__device__ __forceinline__ f16x2 code_pair_lo(uint32_t w) {
    return and_or(w, 0x000f000fu, 0x64006400u) + f16x2{(_Float16)-1032.0f, (_Float16)-1032.0f};
}
__device__ __forceinline__ f16x2 code_pair_hi(uint32_t w) {
    return __builtin_elementwise_fma(and_or(w, 0x00f000f0u, 0x64006400u), f16x2{(_Float16)0.0625f, (_Float16)0.0625f},
                                     f16x2{(_Float16)-72.0f, (_Float16)-72.0f});
}
// A branch around rare work, not selects beside the common: the compiler moves
// nothing past it
__device__ __forceinline__ void keep_branch() { asm volatile(""); }
// p in two f16 parts
__device__ __forceinline__ void split2(float p0, float p1, f16x2 &hi, f16x2 &lo) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    // (opaque: a product rounded to fp16 straight in one place and by way of
    // fp32 in the other, the parts would not add up)
    asm("" : "+v"(p0), "+v"(p1));
    hi = __builtin_convertvector((f32x2{p0, p1}), f16x2);
    lo = __builtin_convertvector((f32x2{fmaf(p0, 1.0f, -(float)hi.x), fmaf(p1, 1.0f, -(float)hi.y)}), f16x2);
}
__device__ __forceinline__ f16x8 join8(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The reference of a row's weights: p = exp2(s - ref), with s in log2 units.
// p * d enters the matrix cores as f16, so ref keeps p * |d| <= 2^TOP for the
// largest scale seen, 2^dlog; a new reference leaves the largest at 2^FRESH.
constexpr float TOP = 15.0f, FRESH = 6.0f;

// Work item: (slot, kv head), the slot's segments one after the other: 16 rows,
// a row being a (token, q head of the group) pair, token-major.  Each wave
// streams its own 32-row tiles of a segment (every fourth) through a private
// double buffer filled by LDS-DMA, so that no barrier stands between the first
// tile and the last.
//
// Scores S^T = K Q^T on 16x16x32 f16 MFMA, one per block of 32 dims: the codes
// are exact in f16, the block's scale multiplies the fp32 sum (one fma), and q
// is exact (f16, bf16 after a power-of-two scale of its row) or split into two
// f16 parts (f32: 22 bits; NS = 2).  D then holds key 4 g + v, row l % 16 in
// lane l (g = l / 16), which is the B operand's layout of P^T in O^T = V^T P^T
// with the keys in that order: P never leaves its lane.  V's operand comes
// from a transposing LDS read, eight keys' byte of one dim pair per lane; its
// scales multiply P (per block, in fp32, rounded once to f16, or to two parts).
//
// Bound by the cache's bytes and the codes' unpacking about alike: 64 replies
// with 8600 rows on average (24 heads over 4 of 256, bf16; 635 MB) in 135 us, 4.7
// TB/s; one behind 131,000 rows (F32; 151 MB) 42 us and 7 to join, where the
// start and end of the workgroups are a quarter of it.
template <int HD, int NS>
__global__ __launch_bounds__(256, 2) void kv4_split_kernel(Attn a) {
    constexpr uint32_t NB = HD / 32, HB = HD / 2, SB = HD / 16, NCH = HB / 16, KC = TILE * HB, SC = TILE * SB;
    constexpr uint32_t STAGE = 2 * KC + 2 * SC, NI = TILE * NCH / 64, SH = HD == 256 ? 1 : HD == 128 ? 2 : 3;
    constexpr uint32_t OST = HD + 4, RING = 4 * 2 * STAGE, COMB = 4 * 16 * OST * 4;
    __shared__ __attribute__((aligned(16))) unsigned char sm[RING > COMB ? RING : COMB];
    __shared__ float red[2][4][16];
    const uint32_t lane = threadIdx.x & 63u, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r16 = lane & 15u, g4 = lane >> 4, NKV = a.b.nkv;
    const uint32_t g = blockIdx.x, slot = blockIdx.y;
    uint32_t mt = 0;   // the segment's rows: 16 mt ..
    // (a row's token: rows <= SPLIT_MOST and gqa <= SPLIT_MOST, so the product with ceil(2^32 / gqa) has the quotient)
    auto tok_of = [&](uint32_t r) { return a.gqa == 1 ? 16 * mt + r : __umulhi(16 * mt + r, a.gqa_inv); };
    Deal d;
    Work wk = deal(a, slot, false, d);
    const uint32_t x0 = slot * d.share, x1 = min(x0 + d.share, d.total);
    bool again = false;
    for (uint32_t x = x0; x < x1;) {
    if (x > x0) {
        const Work last = wk;
        wk = find_units(a, d, x, false, &last);
    }
    if (wk.seq < 0) break;   // (never: x < total)
    const uint32_t tiles = seg_tiles(a, wk.len), units = seg_units(tiles, d.tiles);
    mt = wk.count == units ? 0u : (x - wk.first) / units;
    const uint32_t begin = wk.first + mt * units, stop = tiles <= WHOLE ? units : min(x1 - begin, units);
    const uint32_t t0 = (x - begin) * d.tiles, t1 = tiles <= WHOLE ? tiles : min(stop * d.tiles, tiles);   // the segment's tiles here
    const bool ours = t0 == 0 || tiles > WHOLE, whole = t0 == 0 && t1 == tiles;
    const uint32_t rec0 = slot * 2 + (x > x0 ? 1u : 0u);
    x = begin + stop;
    const uint32_t M = (uint32_t)wk.n_new * a.gqa;
    if (!ours) continue;
    if (again) __syncthreads();   // (the last segment's sums have been read)
    again = true;
    const uint32_t rows = min(16u, M - 16 * mt);
    const int p0 = wk.len - wk.n_new;   // the first token's position
    auto row_pos = [&](uint32_t r) { return p0 + (int)tok_of(r); };
    const int pmin = row_pos(0), pmax = row_pos(rows - 1), c0 = (int)(t0 * TILE), cap = (int)row_cap(a);
    const int end = min(min((int)(t1 * TILE), pmax + 1), cap);            // rows [c0, end)
    const int my_vis = r16 < rows ? min(row_pos(r16) + 1, end) : end;     // of them this lane's row sees [c0, my_vis)
    const int n_tile = end > c0 ? (end - c0 + (int)TILE - 1) / (int)TILE : 0;

    LDS unsigned char *L = (LDS unsigned char *)sm + w * 2 * STAGE;
    const uint32_t lbase = (uint32_t)(uintptr_t)(LDS unsigned char *)sm + w * 2 * STAGE;
    const size_t head_bytes = ((size_t)HB + SB) << a.page_shift, page_bytes = head_bytes * NKV;
    const uint64_t kc = (uint64_t)a.b.kc + g * head_bytes, vc = (uint64_t)a.b.vc + g * head_bytes;
    const uint32_t pmask = (1u << a.page_shift) - 1u;
    // 16-byte unit c of row r lies in slot c ^ swz(r): the 16 rows of one unit,
    // and the 8 rows of one transposing read, on different banks
    auto swz = [](uint32_t r) { return ((r >> SH) ^ ((r >> 4) * (NCH / 2))) & (NCH - 1); };
    const int32_t *table = a.b.pages + (size_t)wk.seq * a.b.max_pages;
    uint32_t win = 0x80000000u;   // entries [win, win + 64) of the page table, one a lane
    int ids = 0;
    uint32_t holes = 0;   // bits of the half tiles without a page, of the tile issued last
    auto page_at = [&](int row, uint32_t half) -> uint32_t {
        const uint32_t e = (uint32_t)row >> a.page_shift;
        if (e - win >= 64u) {
            win = e;
            ids = table[min(e + lane, a.b.max_pages - 1u)];
        }
        const uint32_t p = (uint32_t)__builtin_amdgcn_readlane(ids, (int)(e - win));
        if (p < a.b.n_pages) return p;
        if (lane == 0) raise_error(g_kv4_err, SINTER_E_BAD_SHAPE, (unsigned)wk.seq);
        holes |= half;
        return 0;
    };
    auto issue = [&](int j, uint32_t st) {
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));   // (opaque: addresses made of it would be kept through the loop)
        const int row = c0 + j * (int)TILE;
        holes = 0;
        const uint64_t o0 = page_at(row, 1u) * page_bytes;
        const uint32_t in0 = (uint32_t)row & pmask;
        uint64_t o1 = o0;   // (rows past the end: the first half's again, masked)
        uint32_t in1 = in0;
        if (row + 16 < end) {
            o1 = page_at(row + 16, 2u) * page_bytes;
            in1 = (uint32_t)(row + 16) & pmask;
        }
        const uint32_t to = lbase + st * STAGE;
        const uint64_t c_0 = o0 + (size_t)in0 * HB, c_1 = o1 + (size_t)in1 * HB;
#pragma unroll
        for (uint32_t i = 0; i < NI; i++) {
            const uint32_t u = 64 * i + ln, r = u / NCH, s = u % NCH;
            const uint32_t off = (r & 15u) * HB + 16 * (s ^ swz(r));
            const uint64_t at = (r < 16 ? c_0 : c_1) + off;
            lds_dma16v(kc + at, to + 1024 * i);
            lds_dma16v(vc + at, to + KC + 1024 * i);
        }
        // the scales: K's 32 rows, then V's
        constexpr uint32_t NU = SC / 16;   // lanes a tensor
        const size_t plane = (size_t)HB << a.page_shift;
        if (ln < 2 * NU) {
            const uint32_t u = ln % NU, h = u / (NU / 2), off = 16 * (u % (NU / 2));
            const uint64_t at = (h ? o1 + (size_t)in1 * SB : o0 + (size_t)in0 * SB) + plane + off;
            lds_dma16v((ln < NU ? kc : vc) + at, to + 2 * KC);
        }
    };

    const int nt = (n_tile - (int)w + 3) / 4;
    if (nt > 0) issue((int)w, 0);
    // the row's q, while the first tile is on its way: dims 32 b + {4 g, .., 4 g + 3} and 16 further, in the codes' order
    f16x8 Q[NS][NB];
    float qs;
    {
        const uint32_t r = min(r16, rows - 1), tk = tok_of(r);
        const int64_t e0 = (int64_t)(wk.tok0 + (int)tk) * a.q.ld + (int64_t)((g - tk) * a.gqa + 16 * mt + r) * a.q.hs + 4 * g4;
        float4 x[2 * NB];
        float am = 0.0f;
        // (all loads in flight before the first is used: no branch on the type between them)
        if constexpr (NS == 2) {
#pragma unroll
            for (uint32_t b = 0; b < 2 * NB; b++)
                x[b] = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q.p) + e0 + 16 * b);
        } else {
            u32x2 u[2 * NB];
#pragma unroll
            for (uint32_t b = 0; b < 2 * NB; b++)
                u[b] = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(a.q.p) + e0 + 16 * b);
            const bool bf = a.type == SINTER_BF16;
#pragma unroll
            for (uint32_t b = 0; b < 2 * NB; b++) {
                const float4 m = cvt4(u[b], SINTER_BF16), n = cvt4(u[b], SINTER_F16);
                x[b] = make_float4(bf ? m.x : n.x, bf ? m.y : n.y, bf ? m.z : n.z, bf ? m.w : n.w);
            }
        }
#pragma unroll
        for (uint32_t b = 0; b < 2 * NB; b++)
            am = fmaxf(am, fmaxf(fmaxf(fabsf(x[b].x), fabsf(x[b].y)), fmaxf(fabsf(x[b].z), fabsf(x[b].w))));
        am = fmaxf(am, __shfl_xor(am, 16, 64));
        am = fmaxf(am, __shfl_xor(am, 32, 64));
        // the row's largest element to [2^13, 2^14): its scale is a power of two
        int ex = am > 0.0f && am < INFINITY ? 14 - (int)((__float_as_uint(fmaxf(am, 1e-30f)) >> 23) - 126u) : 0;
        const float up = r16 < rows ? ldexpf(1.0f, ex) : 0.0f;
        qs = a.qscale * ldexpf(1.0f, -ex);
#pragma unroll
        for (uint32_t b = 0; b < NB; b++) {
            const float4 l = x[2 * b], h = x[2 * b + 1];
            float f[8] = {l.x * up, l.z * up, l.y * up, l.w * up, h.x * up, h.z * up, h.y * up, h.w * up};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if constexpr (NS == 2) asm volatile("" : "+v"(f[i]));   // (as for the weights below)
                const _Float16 hi = (_Float16)f[i];
                Q[0][b][i] = hi;
                if constexpr (NS == 2) Q[NS - 1][b][i] = (_Float16)(f[i] - (float)hi);
            }
        }
    }

    f32x4 O[2 * NB];
#pragma unroll
    for (uint32_t i = 0; i < 2 * NB; i++) O[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float ref = REF_NONE, lim = REF_NONE, lsum = 0.0f;
    float dtop = 0.0f, dlog = -24.0f;   // every V scale so far is at most dtop = 2^dlog (dtop 0: none yet)
    for (int i = 0; i < nt; i++) {
        const uint32_t st = i & 1;
        // (opaque, as in issue)
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));
        const uint32_t r16 = ln & 15u, g4 = ln >> 4;
        const uint32_t hole = holes;   // (this tile's)
        // the reads of the buffer that is filled next have landed
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + 1 < nt) {
            issue((int)w + 4 * (i + 1), st ^ 1u);
            if constexpr (NI == 4) asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
            else if constexpr (NI == 2) asm volatile("s_waitcnt vmcnt(5)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(3)" ::: "memory");
        } else {
            dma_wait();
        }
        const int row0 = c0 + ((int)w + 4 * i) * (int)TILE;
        const LDS unsigned char *kt = L + st * STAGE, *vt = kt + KC, *ks = kt + 2 * KC, *vs = ks + SC;
        // Scores, step by step kept in this order: a block's codes are taken
        // apart while the block before it is on the matrix core, whose sums are
        // scaled a step later (left to the scheduler each step waits for its
        // read, its MFMA and its sums in turn: 7000 cycles a tile of F32 rows)
        float s[2][4] = {};
        uint32_t kx[2][NB], d[2][4][NB / 2];   // codes; scales of keys 4 g + v, two blocks a word
#pragma unroll
        for (uint32_t h = 0; h < 2; h++) {
            const uint32_t r = 16 * h + r16;
#pragma unroll
            for (uint32_t b = 0; b < NB; b++)
                kx[h][b] = *reinterpret_cast<const LDS uint32_t *>(kt + r * HB + 16 * (b ^ swz(r)) + 4 * g4);
#pragma unroll
            for (uint32_t v = 0; v < 4; v++)
#pragma unroll
                for (uint32_t b = 0; b < NB / 2; b++)
                    d[h][v][b] = reinterpret_cast<const LDS uint32_t *>(ks + (16 * h + 4 * g4 + v) * SB)[b];
        }
        auto k_operand = [&](uint32_t u) {
            const uint32_t x = kx[u / NB][u % NB];
            return join8(code_pair_lo(x), code_pair_lo(x >> 8), code_pair_hi(x), code_pair_hi(x >> 8));
        };
        f16x8 A = k_operand(0);
        f32x4 t[2];
        auto scaled = [&](uint32_t u) {
            const uint32_t h = u / NB, b = u % NB;
#pragma unroll
            for (uint32_t v = 0; v < 4; v++) {
                const f16x2 dd = pair_of(d[h][v][b / 2]);
                s[h][v] = fmaf(t[u & 1][v], (float)(b & 1 ? dd.y : dd.x), s[h][v]);
            }
        };
#pragma unroll
        for (uint32_t u = 0; u < 2 * NB; u++) {
            sched_fence();
            const f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
            t[u & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, Q[0][u % NB], z, 0, 0, 0);
            if constexpr (NS == 2) t[u & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, Q[NS - 1][u % NB], t[u & 1], 0, 0, 0);
            if (u + 1 < 2 * NB) A = k_operand(u + 1);
            if (u > 0) scaled(u - 1);
        }
        sched_fence();
        // V's codes and scales, on their way while the weights are made
        const uint32_t kr = (r16 >> 1), vr = 16 * (kr >> 2) + 4 * g4 + (kr & 3);
        auto v_codes = [&](uint32_t b) {
            // (lane i of a group of 16 reads half i % 2 of row key(i / 2) and
            // gets byte i of the block for the group's eight keys)
            return __builtin_amdgcn_ds_read_tr8_b64_v2i32((LDS i32x2 *)(vt + vr * HB + 16 * (b ^ swz(vr)) + 8 * (r16 & 1u)));
        };
        i32x2 vx[NB];
        constexpr uint32_t AHEAD = NS == 2 && NB == 8 ? 4 : NB;
#pragma unroll
        for (uint32_t b = 0; b < AHEAD; b++) vx[b] = v_codes(b);
        scaled(2 * NB - 1);
        uint32_t dv[8][NB / 2];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++)
#pragma unroll
            for (uint32_t b = 0; b < NB / 2; b++)
                dv[k][b] = reinterpret_cast<const LDS uint32_t *>(vs + (16 * (k >> 2) + 4 * g4 + (k & 3)) * SB)[b];
        // the largest finite V scale of the lane's share of the tile
        float dm = 0.0f;
        {
            constexpr uint32_t PER = SC / 64;   // bytes a lane
            const uint32_t r = lane * PER / SB;
            const bool real = row0 + (int)r < end && !(hole >> (r >> 4) & 1u);
#pragma unroll
            for (uint32_t k = 0; k < PER / 2; k++) {
                const float x = fabsf(h2f(reinterpret_cast<const LDS uint16_t *>(vs + lane * PER)[k]));
                dm = real && x < INFINITY ? fmaxf(dm, x) : dm;
            }
        }
        // a tile with rows that some row here does not see
        const bool masked = __builtin_amdgcn_readfirstlane(row0 + (int)TILE > min(end, pmin + 1) || hole != 0 ? 1 : 0) != 0;
        float p[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) p[k] = s[k >> 2][k & 3];
        if (masked) {
            keep_branch();
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) {
                const bool ok = row0 + (int)(16 * (k >> 2) + 4 * g4 + (k & 3)) < my_vis && !(hole >> (k >> 2) & 1u);
                p[k] = ok ? p[k] : -INFINITY;
                // (a masked row's scale may be anything: 0 keeps it out)
#pragma unroll
                for (uint32_t b = 0; b < NB / 2; b++) dv[k][b] = ok ? dv[k][b] : 0u;
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
        mx = mx * qs;
        if (__builtin_amdgcn_ballot_w64(mx > lim || dm > dtop) != 0) {
            dm = wave_max_f32(dm);
            if (dm > dtop) {   // (uniform) to twice the largest, a power of two
                dlog = fminf(fmaxf((float)((int)(__float_as_uint(dm) >> 23) - 125), -23.0f), 17.0f);
                dtop = ldexpf(1.0f, (int)dlog);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float nr = fmaxf(ref, mx + dlog - FRESH);
            if (nr != ref) {
                const float c = __builtin_amdgcn_exp2f(ref - nr);
                lsum *= c;
#pragma unroll
                for (uint32_t k = 0; k < 2 * NB; k++) O[k] = O[k] * c;
                ref = nr;
            }
            lim = ref + TOP - dlog;
        }
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            p[k] = __builtin_amdgcn_exp2f(fmaf(p[k], qs, -ref));   // (0 where masked)
            lsum += p[k];
        }
        // The sums, in the same way
        f16x8 Al, Ah, P, Pl;
        auto v_operands = [&](uint32_t b) {
            const uint32_t x0 = (uint32_t)vx[b].x, x1 = (uint32_t)vx[b].y;
            Al = join8(code_pair_lo(x0), code_pair_lo(x0 >> 8), code_pair_lo(x1), code_pair_lo(x1 >> 8));
            Ah = join8(code_pair_hi(x0), code_pair_hi(x0 >> 8), code_pair_hi(x1), code_pair_hi(x1 >> 8));
#pragma unroll
            for (uint32_t k = 0; k < 8; k += 2) {   // keys 0 2, 1 3, 4 6, 5 7
                const uint32_t k0 = (k & 4) | ((k >> 1) & 1), k1 = k0 + 2;
                const f16x2 d0 = pair_of(dv[k0][b / 2]), d1 = pair_of(dv[k1][b / 2]);
                const float s0 = (float)(b & 1 ? d0.y : d0.x), s1 = (float)(b & 1 ? d1.y : d1.x);
                if constexpr (NS == 1) {
                    P[k] = (_Float16)fmaf(p[k0], s0, 0.0f);
                    P[k + 1] = (_Float16)fmaf(p[k1], s1, 0.0f);
                } else {
                    f16x2 hi, lo;
                    split2(fmaf(p[k0], s0, 0.0f), fmaf(p[k1], s1, 0.0f), hi, lo);
                    P[k] = hi.x; P[k + 1] = hi.y;
                    Pl[k] = lo.x; Pl[k + 1] = lo.y;
                }
            }
        };
        v_operands(0);
#pragma unroll
        for (uint32_t b = 0; b < NB; b++) {
            sched_fence();
            O[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Al, P, O[2 * b], 0, 0, 0);
            O[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Ah, P, O[2 * b + 1], 0, 0, 0);
            if constexpr (NS == 2) {
                O[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Al, Pl, O[2 * b], 0, 0, 0);
                O[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Ah, Pl, O[2 * b + 1], 0, 0, 0);
            }
            if (b + AHEAD < NB) vx[b + AHEAD] = v_codes(b + AHEAD);
            if (b + 1 < NB) v_operands(b + 1);
        }
        sched_fence();
    }
    // the four waves' sums joined through LDS
    lsum += __shfl_xor(lsum, 16, 64);
    lsum += __shfl_xor(lsum, 32, 64);
    if (lane < 16) {
        red[0][w][lane] = ref;
        red[1][w][lane] = lsum;
    }
    __syncthreads();   // (every wave is past its last tile: its buffers are free)
    LDS float *comb = (LDS float *)(LDS unsigned char *)sm;
#pragma unroll
    for (uint32_t i = 0; i < 2 * NB; i++)
        *reinterpret_cast<LDS f32x4 *>(comb + (w * 16 + r16) * OST + 16 * i + 4 * g4) = O[i];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < rows * (HD / 4); i += 256) {
        const uint32_t r = i / (HD / 4), e = 4 * (i % (HD / 4));
        const float m = fmaxf(fmaxf(red[0][0][r], red[0][1][r]), fmaxf(red[0][2][r], red[0][3][r]));
        float l = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const float c = __builtin_amdgcn_exp2f(red[0][k][r] - m);
            l = fmaf(red[1][k][r], c, l);
            const f32x4 x = *reinterpret_cast<const LDS f32x4 *>(comb + (k * 16 + r) * OST + e);
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = fmaf(x[j], c, o[j]);
        }
        if (whole) {
            const uint32_t tk = tok_of(r);
            store_out(a, wk.tok0 + (int)tk, (g - tk) * a.gqa + 16 * mt + r, e, o, l);
        } else {
            const size_t rec = ((size_t)rec0 * NKV + g) * 16 + r;
            *reinterpret_cast<f32x4 *>(a.part + rec * HD + e) = o;
            if (e == 0) a.ml[rec] = make_float2(m, l);
        }
    }
    }
    if ((g | slot) == 0 && w == 0) report_lengths(a);
}

// A segment divided over slots: out = sum c_i O_i / sum c_i l_i with c_i =
// exp2(ref_i - max ref) over its parts.  One workgroup per (sequence, kv head,
// row); wave w takes every NW-th part, all of its loads in flight for up to 8
// NW.  Latency: 3 us of a few parts, 7 of 128.
template <int NW>
__global__ __launch_bounds__(64 * NW) void kv4_merge_kernel(Attn a, uint32_t rows) {
    __shared__ float2 red[NW];   // a wave's reference and weight sum
    __shared__ __attribute__((aligned(16))) float comb[NW][256];
    const uint32_t r = blockIdx.x % rows, sg = blockIdx.x / rows, g = sg % a.b.nkv, lane = threadIdx.x & 63u, HD = a.b.hd;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Most of a mixed batch's workgroups have no such row: they leave at once
    const uint32_t seq = sg / a.b.nkv;
    const int rows_of = (a.b.tok_start[seq + 1] - a.b.tok_start[seq]) * (int)a.gqa;
    if ((int)r >= rows_of || rows_of > (int)a.split_rows || a.b.kv_len[seq] <= (int)(WHOLE * TILE)) return;
    // (one wave looks the parts up: sixteen at it would take turns)
    __shared__ uint32_t place[4];   // parts, the first one's slot, whether that is the slot's second record, first token
    if (w == 0) {
        Deal d;
        const Work wk = deal(a, seq, true, d);
        uint32_t n = 0, i0 = 0, second = 0;
        if (wk.seq >= 0 && r < (uint32_t)wk.n_new * a.gqa) {
            const uint32_t tiles = seg_tiles(a, wk.len), units = seg_units(tiles, d.tiles), begin = wk.first + r / 16 * units;
            i0 = begin;
            n = begin + units - 1u;
            if (d.share > 1u) {
                i0 /= d.share;
                n /= d.share;
            }
            n = tiles > WHOLE ? n - i0 + 1u : 0u;
            second = begin > i0 * d.share ? 1u : 0u;
        }
        if (lane == 0) {
            place[0] = n;
            place[1] = i0;
            place[2] = second;
            place[3] = (uint32_t)wk.tok0;
        }
    }
    __syncthreads();
    const uint32_t n = (uint32_t)__builtin_amdgcn_readfirstlane((int)place[0]), i0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)place[1]);
    const uint32_t head1 = (uint32_t)__builtin_amdgcn_readfirstlane((int)place[2]);
    if (n < 2) return;
    auto rec = [&](uint32_t c) {
        return (((size_t)(i0 + c) * 2 + (c == 0 ? head1 : 0u)) * a.b.nkv + g) * 16 + r % 16;
    };
    float m = REF_NONE, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t e = 4 * lane;
    for (uint32_t c0 = w; c0 < n; c0 += 8 * NW) {
        f32x4 x[8];
        float2 ml[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            const size_t at = rec(min(c0 + NW * k, n - 1u));
            ml[k] = a.ml[at];
            x[k] = *reinterpret_cast<const f32x4 *>(a.part + at * HD + (e < HD ? e : 0u));
        }
        float mn = m;
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) mn = fmaxf(mn, ml[k].x);
        const float f = __builtin_amdgcn_exp2f(m - mn);
        l *= f;
        o = o * f;
        m = mn;
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            if (c0 + NW * k >= n) break;
            const float c = __builtin_amdgcn_exp2f(ml[k].x - m);
            l = fmaf(ml[k].y, c, l);
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = fmaf(x[k][j], c, o[j]);
        }
    }
    if (lane == 0) red[w] = make_float2(m, l);
    *reinterpret_cast<f32x4 *>(&comb[w][e]) = o;
    __syncthreads();
    if (w != 0 || e >= HD) return;
#pragma unroll
    for (uint32_t k = 0; k < NW; k++) m = fmaxf(m, red[k].x);
    l = 0.0f;
    o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t k = 0; k < NW; k++) {
        const float c = __builtin_amdgcn_exp2f(red[k].x - m);
        const f32x4 x = *reinterpret_cast<const f32x4 *>(&comb[k][e]);
        l = fmaf(red[k].y, c, l);
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = fmaf(x[j], c, o[j]);
    }
    store_out(a, (int64_t)place[3] + r / a.gqa, g * a.gqa + r % a.gqa, e, o, l);
}

// ------------------------------------------------------------------ many rows

typedef float f32x16 __attribute__((ext_vector_type(16)));

// the tiles of ROWS rows of sequences that kv4_split_kernel leaves out
__device__ __forceinline__ Work find_tile(const Attn &a, uint32_t rows, uint32_t id, bool by_seq) {
    return locate(a, id, by_seq, [&](int len, int n) {
        return is_split(a, n) ? 0u : ((uint32_t)n * a.gqa + rows - 1u) / rows;
    });
}
// The id-th tile from the one with the most cache rows down, so that the
// longest start first (two prompts of 2000 tokens, bf16, 27B heads: sequence
// after sequence 377 us, so 205).  A sequence with p0 rows before its tokens
// has one tile in each of the levels p0 gqa / rows + 0, 1, ..: the level is
// found by bisection over the count of tiles at or above it, a lane a
// sequence.  More than 64 sequences are taken in their order.
__device__ __forceinline__ Work find_ranked_tile(const Attn &a, uint32_t rows, uint32_t id) {
    if (a.b.n_seq > 64) return find_tile(a, rows, id, false);
    int len, t0, n;
    load_seq(a, 0, false, len, t0, n);
    const uint32_t c = n > 0 && !is_split(a, n) ? ((uint32_t)n * a.gqa + rows - 1u) / rows : 0u;
    const uint32_t base = (uint32_t)((uint64_t)(uint32_t)max(0, len - n) * a.gqa / rows), top = c ? base + c : 0u;
    // (no branch on c: every lane takes part in the sums)
    auto above = [&](uint32_t y) { return wave_sum_u32(min(c, max(top, y) - y)); };
    Work w;
    w.seq = -1;
    if (above(0) <= id) return w;
    // above(lo) > id >= above(hi)
    // (the largest top, exact in fp32 by parts of 24 bits at most)
    const float m8 = wave_max_f32((float)(top >> 8)), m0 = wave_max_f32((float)(top >> 8) == m8 ? (float)(top & 255u) : 0.0f);
    uint32_t lo = 0, hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)((((uint32_t)m8 << 8) | (uint32_t)m0) + 1u));
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (above(mid) > id) lo = mid;
        else hi = mid;
    }
    const bool in = lo >= base && lo < top;
    const uint64_t all = __builtin_amdgcn_ballot_w64(in);
    const uint32_t before = __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0u));
    const uint32_t rank = id - above(hi);
    const uint64_t m = __builtin_amdgcn_ballot_w64(in && before == rank);
    if (m == 0) return w;
    const int l = __builtin_ctzll(m);
    w.seq = l;
    w.len = __builtin_amdgcn_readlane(len, l);
    w.tok0 = __builtin_amdgcn_readlane(t0, l);
    w.n_new = __builtin_amdgcn_readlane(n, l);
    w.item = lo - (uint32_t)__builtin_amdgcn_readlane((int)base, l);
    // (the tiles of the sequences before it)
    w.first = wave_sum_u32((threadIdx.x & 63u) < (uint32_t)l ? c : 0u);
    return w;
}
// The cache rows a chunk of a tile that sees `seen` rows takes: 128 at least (128
// rows behind 1000, 27B heads, bf16: 28 us, 512 at least 72, 64 27)
constexpr uint32_t CHUNK_MIN = 128;
__device__ __forceinline__ uint32_t chunk_rows(uint32_t seen, uint32_t n_split) {
    return max(CHUNK_MIN, ((seen + n_split - 1u) / n_split + TILE - 1u) / TILE * TILE);
}

// Work item: (tile of 32 NW rows, kv head, chunk of the cache rows the tile
// sees); wave w has rows 32 w .. 32 w + 31.  The waves unpack each 32-row cache
// tile into LDS together, a tile ahead of its use, so that its codes are taken
// apart once for 32 NW rows:
//   K  fragments [16-dim slice][half][32 keys] of 8 dims: the exact codes, the
//      scales multiplying each block's fp32 sum (KX), or, for BF16 rows,
//      f16(scale * code): 2^-12 of an element, well under the output's 2^-9
//   V  fragments [32-dim block][8-key group][32 dims] of 8 keys, transposed by
//      the LDS read of the raw codes: f16(scale * code), for F32 a second
//      fragment holds the rest of it (scale * code has 15 bits: exact in two)
// The weights are one f16 for BF16 rows and two (NP) for F16 and F32: with the
// rounded V one f16 would put F16 results at 1.6 times the error that rounding
// them once has, two at 1.26.
// Every operand read is 1 KiB of consecutive LDS.  Scores S^T = K Q^T and sums
// O^T = V^T P^T run on 32x32x16 f16 MFMA: D holds key 8 i + 4 (l / 32) + j of
// row l % 32 in lane l, the B operand's layout of P^T with the keys of a group
// in that order, so P stays in its lane.  The weights' reference moves as in
// kv4_split_kernel (with no scale in it: p <= 2^TOP).
//
// A V scale that is not finite would reach rows that do not see its key (0
// times it): it is 0 in the fragments and named in `odd`, and makes NaN of the
// block's sums of the rows that do.
//
// Bound by a wave's instructions and waits beside the matrix core, which is busy
// a quarter (bf16) to a third (F32) of the time: 500 tokens of 24 heads of 256 over 4 behind 32,000 rows,
// F32: 1344 us, 295 TF/s and with each product in three parts 885 TF/s of f16 (a
// large f16 product: 1166); bf16: 530 us, 750 TF/s.  Two prompts of 2000 tokens,
// bf16: 163 us, 640 TF/s.
template <int HD, int T, int NW>
__global__ __launch_bounds__(64 * NW, T == SINTER_F32 ? 1 : 2) void kv4_tile_kernel(Attn a) {
    constexpr uint32_t NS = T == SINTER_F32 ? 2 : 1, NP = T == SINTER_BF16 ? 1 : 2;   // f16 parts of q (and V), of the weights
    constexpr bool KX = T == SINTER_F16;   // exact codes of K in the fragments
    constexpr uint32_t NB = HD / 32, HB = HD / 2, SB = HD / 16, NCH = HB / 16, KC = TILE * HB, ROWS = 32 * NW;
    constexpr uint32_t SH = HD == 256 ? 1 : HD == 128 ? 2 : 3, BPW = NB > NW ? NB / NW : 1, ACT = NB / BPW;
    constexpr uint32_t KF = NS * NB * 2048, VF = NB * 2048, KS = KX ? NB * 64 : 0, BUF = KF + NS * VF + KS;
    // (the output's passes: blocks of 32 dims a pass, 16-byte units a row, bytes a wave)
    constexpr uint32_t FIT = 2 * BUF / (NW * 4096), PB = FIT >= 4 && NB >= 4 ? 4 : FIT >= 2 ? 2 : 1, UN = PB * 8, PASS = PB * 4096;
    __shared__ __attribute__((aligned(16))) unsigned char frag[2 * BUF > NW * PASS ? 2 * BUF : NW * PASS];
    __shared__ __attribute__((aligned(16))) unsigned char raw[2 * KC];
    __shared__ __attribute__((aligned(16))) _Float16 vsc[NB][32];
    __shared__ __attribute__((aligned(16))) uint32_t odd[2][8];
    // (Heads of 256: the sums and q leave too few registers for fragments read
    // ahead, and for F16 a block's own sums: the last QL slices of q are read
    // from LDS)
    constexpr uint32_t QL = HD != 256 || NS == 2 ? 0 : KX ? 4 : 2, QR = 2 * NB - QL;
    __shared__ __attribute__((aligned(16))) f16x8 qx[QL ? NW * QL * 64 : 1];
    const uint32_t lane = threadIdx.x & 63u, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t l32 = lane & 31u, hf = lane >> 5, NKV = a.b.nkv;
    uint32_t id = blockIdx.x;
    const uint32_t g = id % NKV;
    id /= NKV;
    const uint32_t ck = id / a.n_tile;
    if (a.report && blockIdx.x == 0 && w == 0) report_lengths(a);
    const Work wk = find_ranked_tile(a, ROWS, id % a.n_tile);
    if (wk.seq < 0) return;
    const uint32_t gt = wk.first + wk.item;
    if (gt >= a.n_tile) return;   // (sequences that overlap: no room for the chunks' sums)
    const uint32_t M = (uint32_t)wk.n_new * a.gqa, r0 = wk.item * ROWS;
    const int p0 = wk.len - wk.n_new, cap = (int)row_cap(a);
    auto row_pos = [&](uint32_t r) { return p0 + (int)(min(r, M - 1u) / a.gqa); };
    const int seen = max(0, min(row_pos(r0 + ROWS - 1u) + 1, cap));   // rows the tile's last row sees
    const uint32_t per = chunk_rows((uint32_t)seen, a.n_split);
    const int c0 = (int)(ck * per), end = min(seen, c0 + (int)per);   // rows [c0, end)
    if (ck > 0 && c0 >= seen) return;
    const bool whole = (uint32_t)seen <= per;   // one chunk
    const int n_tile = end > c0 ? (end - c0 + (int)TILE - 1) / (int)TILE : 0;
    const uint32_t row = r0 + 32 * w + l32;
    const bool live = row < M;
    const int my_vis = live ? min(row_pos(row) + 1, end) : end;
    const int wmin = __builtin_amdgcn_readfirstlane(min(row_pos(r0 + 32 * w) + 1, end));        // the wave's first row's
    const int wmax = r0 + 32 * w < M ? __builtin_amdgcn_readfirstlane(min(row_pos(r0 + 32 * w + 31u) + 1, end)) : 0;   // and last row's end

    // q: slice m = 2 b + half holds dims 32 b + 16 half + 8 hf + {0 2 1 3 4 6 5 7} (the codes' order)
    f16x8 Q[NS][2 * NB];
    float qs;
    {
        const int64_t tok = wk.tok0 + (int)(min(row, M - 1u) / a.gqa), head = g * a.gqa + min(row, M - 1u) % a.gqa;
        const int64_t e0 = tok * a.q.ld + head * a.q.hs + 8 * hf;
        float am = 0.0f;
        auto scale_of = [&](float m) {
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            return m > 0.0f && m < INFINITY ? 14 - (int)((__float_as_uint(fmaxf(m, 1e-30f)) >> 23) - 126u) : 0;
        };
        if constexpr (NS == 2) {
            const float *src = static_cast<const float *>(a.q.p) + e0;
#pragma unroll
            for (uint32_t m = 0; m < 2 * NB; m++)
#pragma unroll
                for (uint32_t k = 0; k < 8; k++) am = fmaxf(am, fabsf(src[16 * m + k]));
            const int ex = scale_of(am);
            const float up = live ? ldexpf(1.0f, ex) : 0.0f;
            qs = a.qscale * ldexpf(1.0f, -ex);
#pragma unroll
            for (uint32_t m = 0; m < 2 * NB; m++) {
                const float4 x = reinterpret_cast<const float4 *>(src + 16 * m)[0], y = reinterpret_cast<const float4 *>(src + 16 * m)[1];
                float f[8] = {x.x * up, x.z * up, x.y * up, x.w * up, y.x * up, y.z * up, y.y * up, y.w * up};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    asm volatile("" : "+v"(f[i]));   // (as for the weights in kv4_split_kernel)
                    const _Float16 hi = (_Float16)f[i];
                    Q[0][m][i] = hi;
                    Q[NS - 1][m][i] = (_Float16)(f[i] - (float)hi);
                }
            }
        } else {
            u32x4 u[2 * NB];
#pragma unroll
            for (uint32_t m = 0; m < 2 * NB; m++)
                u[m] = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.q.p) + e0 + 16 * m);
            const bool bf = a.type == SINTER_BF16;
            auto val = [&](uint32_t m, int k) {
                const uint32_t x = u[m][k >> 1];
                const float b = __uint_as_float(k & 1 ? x & 0xffff0000u : x << 16);
                const float h = h2f((uint16_t)(k & 1 ? x >> 16 : x));
                return bf ? b : h;
            };
#pragma unroll
            for (uint32_t m = 0; m < 2 * NB; m++)
#pragma unroll
                for (int k = 0; k < 8; k++) am = fmaxf(am, fabsf(val(m, k)));
            const int ex = scale_of(am);
            const float up = live ? ldexpf(1.0f, ex) : 0.0f;
            qs = a.qscale * ldexpf(1.0f, -ex);
#pragma unroll
            for (uint32_t m = 0; m < 2 * NB; m++)
#pragma unroll
                for (int i = 0; i < 8; i++) Q[0][m][i] = (_Float16)(val(m, (i & 4) | ((i & 1) << 1) | ((i >> 1) & 1)) * up);
        }
    }

    if constexpr (QL > 0) {
#pragma unroll
        for (uint32_t m = QR; m < 2 * NB; m++) qx[(w * QL + m - QR) * 64 + lane] = Q[0][m];
    }

    // --- a cache tile's way in: loads (two tiles ahead), unpacking (one ahead)
    const size_t head_bytes = ((size_t)HB + SB) << a.page_shift, page_bytes = head_bytes * NKV;
    const uint64_t kc = (uint64_t)a.b.kc + g * head_bytes, vc = (uint64_t)a.b.vc + g * head_bytes;
    const uint32_t pmask = (1u << a.page_shift) - 1u;
    auto swz = [](uint32_t r) { return ((r >> SH) ^ ((r >> 4) * (NCH / 2))) & (NCH - 1); };
    const int32_t *table = a.b.pages + (size_t)wk.seq * a.b.max_pages;
    uint32_t win = 0x80000000u;
    int ids = 0;
    auto page_at = [&](int r, uint32_t &holes, uint32_t half) -> uint32_t {
        const uint32_t e = (uint32_t)r >> a.page_shift;
        if (e - win >= 64u) {
            win = e;
            ids = table[min(e + lane, a.b.max_pages - 1u)];
        }
        const uint32_t p = (uint32_t)__builtin_amdgcn_readlane(ids, (int)(e - win));
        if (p < a.b.n_pages) return p;
        if (lane == 0) raise_error(g_kv4_err, SINTER_E_BAD_SHAPE, (unsigned)wk.seq);
        holes |= half;
        return 0;
    };
    const LDS unsigned char *R = (const LDS unsigned char *)raw;
    const uint32_t rbase = (uint32_t)(uintptr_t)(LDS unsigned char *)raw;
    LDS unsigned char *F = (LDS unsigned char *)frag;
    struct In { u32x2 k[BPW]; uint32_t sc[BPW], holes; };   // (sc: K's scale, V's above it)
    auto issue = [&](int j, In &in) {
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));   // (opaque: addresses made of it would be kept through the loop)
        const uint32_t l32 = ln & 31u, hf = ln >> 5;
        const int r = c0 + j * (int)TILE;
        in.holes = 0;
        const uint32_t in0 = (uint32_t)r & pmask, to = rbase + (j & 1) * KC;
        const uint64_t o0 = page_at(r, in.holes, 1u) * page_bytes;
        // V's codes to LDS, 1 KiB a wave; K's codes of the wave's blocks, both scales: key l32
        auto load = [&](auto codes, auto scales) {
            for (uint32_t i = w; i < KC / 1024; i += NW) {
                const uint32_t u = 64 * i + ln, rr = u / NCH;
                lds_dma16v((uint64_t)codes(vc, rr, 16 * ((u % NCH) ^ swz(rr))), to + 1024 * i);
            }
            if (ACT < NW && w >= ACT) return;
            const GLB unsigned char *kp = codes(kc, l32, 16 * BPW * w + 8 * hf);
            const GLB uint16_t *ksp = (const GLB uint16_t *)scales(kc, l32, 2 * BPW * w);
            const GLB uint16_t *vsp = (const GLB uint16_t *)scales(vc, l32, 2 * BPW * w);
#pragma unroll
            for (uint32_t i = 0; i < BPW; i++) {
                in.k[i] = *reinterpret_cast<const GLB u32x2 *>(kp + 16 * i);
                in.sc[i] = (uint32_t)ksp[i] | ((uint32_t)vsp[i] << 16);
            }
        };
        const uint64_t plane = (uint64_t)HB << a.page_shift;
        if (a.page_shift >= 5) {   // a tile lies in one page: one address and a lane's offset
            const uint64_t co = o0 + (uint64_t)in0 * HB, so = o0 + plane + (uint64_t)in0 * SB;
            in.holes |= in.holes << 1;
            load([&](uint64_t c, uint32_t rr, uint32_t off) { return (const GLB unsigned char *)(c + co) + (rr * HB + off); },
                 [&](uint64_t c, uint32_t rr, uint32_t off) { return (const GLB unsigned char *)(c + so) + (rr * SB + off); });
        } else {
            uint64_t o1 = o0;   // (rows past the end: the first half's again, masked)
            if (r + 16 < end) o1 = page_at(r + 16, in.holes, 2u) * page_bytes;
            load([&](uint64_t c, uint32_t rr, uint32_t off) { return (const GLB unsigned char *)(c + (rr < 16 ? o0 : o1)) + ((rr & 15u) * HB + off); },
                 [&](uint64_t c, uint32_t rr, uint32_t off) {
                     return (const GLB unsigned char *)(c + (rr < 16 ? o0 : o1) + plane) + ((rr & 15u) * SB + off);
                 });
        }
    };
    // Tile j's unpacking by the wave, in PIECES pieces.  MIX: F32's one wave a
    // SIMD puts them between the matrix instructions of the tile before (500
    // tokens behind 32,000 rows, heads of 256 and 128: 1344 and 1031 us, before
    // them 1390 and 1163).  The two waves a SIMD of 16-bit types take turns
    // instead, one unpacking before, one behind its tile's work (two prompts of
    // 2000 tokens, bf16: 163 us, MIX 171).
    constexpr uint32_t PIECES = 6 * BPW;
    constexpr bool MIX = NS == 2;
    constexpr uint32_t PD = NS == 2 && HD < 256 ? 3 : 2;   // slices read ahead of the matrix core (F32, heads of 128: 2 % faster with 3, of 256 no more)
    struct Half { i32x2 x; u32x4 d; } half;   // (V's codes and scales, from piece to piece)
    auto unpack = [&](int j, In &in, uint32_t piece, uint32_t ln) {
        if (ACT < NW && w >= ACT) return;
        const uint32_t l32 = ln & 31u, hf = ln >> 5, r16 = ln & 15u, g4 = ln >> 4, i = piece / 6, b = BPW * w + i;
        // (V's read on its way while K is taken apart)
        const uint32_t part = piece % 6 == 1 ? 3 : piece % 6 == 2 ? 1 : piece % 6 == 3 ? 2 : piece % 6;
        LDS unsigned char *B = F + (j & 1) * BUF;
        const LDS unsigned char *V = R + (j & 1) * KC;
        auto codes = [&](uint32_t x0, uint32_t x1, bool hi, f16x2(&o)[4]) {
            o[0] = hi ? code_pair_hi(x0) : code_pair_lo(x0);
            o[1] = hi ? code_pair_hi(x0 >> 8) : code_pair_lo(x0 >> 8);
            o[2] = hi ? code_pair_hi(x1) : code_pair_lo(x1);
            o[3] = hi ? code_pair_hi(x1 >> 8) : code_pair_lo(x1 >> 8);
        };
        // codes times scales to `to` and, for F32, what the rounding leaves to `rest`
        auto put = [&](const f16x2(&c)[4], const f16x2(&d)[4], LDS unsigned char *to, LDS unsigned char *rest) {
            f16x2 p[4], r[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                p[k] = c[k] * d[k];
                if constexpr (NS == 2) r[k] = __builtin_elementwise_fma(c[k], d[k], -p[k]);
            }
            *reinterpret_cast<LDS f16x8 *>(to) = join8(p[0], p[1], p[2], p[3]);
            if constexpr (NS == 2) *reinterpret_cast<LDS f16x8 *>(rest) = join8(r[0], r[1], r[2], r[3]);
        };
        f16x2 c[4];
        if (part == 0) {
            // V scales in the operand's key order (read back below by this wave alone): key 16 s + 4 h + x (x < 4), 8 + x (x >= 4) of group 2 s + h
            if (c0 + j * (int)TILE + (int)l32 >= end || (in.holes >> (l32 >> 4) & 1u)) in.sc[i] = 0;   // (no such row)
            const uint32_t vb = in.sc[i] >> 16;
            const bool fin = (vb & 0x7c00u) != 0x7c00u;
            const uint64_t bad = __builtin_amdgcn_ballot_w64(!fin);
            if (ln == 0) odd[j & 1][b] = (uint32_t)bad;
            const uint32_t grp = 2 * (l32 >> 4) + ((l32 >> 2) & 1u), x = (l32 & 3u) + ((l32 >> 1) & 4u);
            const uint32_t at = (x & 4) | ((x & 1) << 1) | ((x >> 1) & 1);   // 0 2 1 3 4 6 5 7
            ((LDS u16a *)vsc)[b * 32 + grp * 8 + at] = (uint16_t)(fin ? vb : 0u);
            if (KX && hf == 0) ((LDS u16a *)(B + KF + NS * VF))[b * 32 + l32] = (uint16_t)in.sc[i];
        } else if (part < 3) {   // K's elements 0..15 of the block, 16..31
            LDS unsigned char *to = B + (2 * b + part - 1) * 1024 + 16 * ln;
            codes(in.k[i].x, in.k[i].y, part == 2, c);
            if constexpr (KX) {
                *reinterpret_cast<LDS f16x8 *>(to) = join8(c[0], c[1], c[2], c[3]);
            } else {
                const _Float16 d = __builtin_bit_cast(_Float16, (uint16_t)in.sc[i]);
                const f16x2 dd[4] = {{d, d}, {d, d}, {d, d}, {d, d}};
                put(c, dd, to, to + KF / 2);
            }
        } else if (part == 3) {   // V: lane r16 of group g4 gets byte r16 of the group's eight keys
            const uint32_t kr = r16 >> 1, vr = 16 * (g4 >> 1) + 4 * (g4 & 1u) + (kr & 3u) + 8 * (kr >> 2);
            half.x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((LDS i32x2 *)(V + vr * HB + 16 * (b ^ swz(vr)) + 8 * (r16 & 1u)));
            half.d = *reinterpret_cast<const LDS u32x4 *>((const LDS uint16_t *)vsc + b * 32 + g4 * 8);
        } else {   // its elements 0..15 of the block, 16..31
            LDS unsigned char *to = B + KF + b * 2048 + g4 * 512 + 16 * r16 + (part == 5 ? 256 : 0);
            const f16x2 d[4] = {pair_of(half.d[0]), pair_of(half.d[1]), pair_of(half.d[2]), pair_of(half.d[3])};
            codes((uint32_t)half.x.x, (uint32_t)half.x.y, part == 5, c);
            put(c, d, to, to + VF);
        }
    };

    f32x16 O[NB];
#pragma unroll
    for (uint32_t b = 0; b < NB; b++) O[b] = f32x16{0.0f};
    float ref = REF_NONE, lsum = 0.0f;
    // (F32's sums stay in the accumulation half of the registers: left to the
    // compiler they are copied out and back around the rare paths)
    auto pin = [&] {
        if constexpr (T == SINTER_F32) {
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) asm volatile("" : "+a"(O[b]));
        }
    };
    pin();
    auto fetch = [&](int j, In &in) {
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));   // (opaque, as in issue)
#pragma unroll
        for (uint32_t p = 0; p < PIECES; p++) unpack(j + 1, in, p, ln);
        if (j + 2 < n_tile) issue(j + 2, in);
    };
    auto compute = [&](int j, uint32_t holes, In &in) {
        const int row0 = c0 + j * (int)TILE;
        if (row0 >= wmax) {   // (uniform) no row of the wave sees the tile
            if constexpr (MIX) fetch(j, in);
            return;
        }
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));   // (opaque, as in issue)
        const uint32_t hf = ln >> 5;
        const LDS unsigned char *B = F + (j & 1) * BUF;
        auto fr = [&](uint32_t at) { return *reinterpret_cast<const LDS f16x8 *>(B + at + 16 * ln); };
        auto q_at = [&](uint32_t m) { return m < QR ? Q[0][m] : ((const LDS f16x8 *)qx)[(w * QL + m - QR) * 64 + ln]; };
        f32x16 S = {0.0f};
        if constexpr (!KX) {
            f16x8 kf[PD + 1], kr[PD + 1];
#pragma unroll
            for (uint32_t m = 0; m < PD; m++) {
                kf[m] = fr(m * 1024);
                if constexpr (NS == 2) kr[m] = fr(KF / 2 + m * 1024);
            }
#pragma unroll
            for (uint32_t m = 0; m < 2 * NB; m++) {
                const f16x8 k = kf[m % (PD + 1)], r = kr[m % (PD + 1)];
                if (m + PD < 2 * NB) {
                    kf[(m + PD) % (PD + 1)] = fr((m + PD) * 1024);
                    if constexpr (NS == 2) kr[(m + PD) % (PD + 1)] = fr(KF / 2 + (m + PD) * 1024);
                }
                S = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q_at(m), S, 0, 0, 0);
                if constexpr (NS == 2) {
                    S = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, Q[NS - 1][m], S, 0, 0, 0);
                    S = __builtin_amdgcn_mfma_f32_32x32x16_f16(r, Q[0][m], S, 0, 0, 0);
                }
                if constexpr (MIX) {
#pragma unroll
                    for (uint32_t p = m * PIECES / (2 * NB); p < (m + 1) * PIECES / (2 * NB); p++) unpack(j + 1, in, p, ln);
                }
                sched_fence();
            }
        } else {
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) {
                if (b % 2 == 0) sched_fence();
                const f16x8 k0 = fr(2 * b * 1024), k1 = fr((2 * b + 1) * 1024);
                f32x16 t = {0.0f};
                t = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, q_at(2 * b), t, 0, 0, 0);
                t = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, q_at(2 * b + 1), t, 0, 0, 0);
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    const u32x2 d = *reinterpret_cast<const LDS u32x2 *>(B + KF + NS * VF + b * 64 + 16 * i + 8 * hf);
                    const f16x2 d0 = pair_of(d.x), d1 = pair_of(d.y);
                    S[4 * i] = fmaf(t[4 * i], (float)d0.x, S[4 * i]);
                    S[4 * i + 1] = fmaf(t[4 * i + 1], (float)d0.y, S[4 * i + 1]);
                    S[4 * i + 2] = fmaf(t[4 * i + 2], (float)d1.x, S[4 * i + 2]);
                    S[4 * i + 3] = fmaf(t[4 * i + 3], (float)d1.y, S[4 * i + 3]);
                }
                if constexpr (MIX) {
#pragma unroll
                    for (uint32_t p = b * PIECES / NB; p < (b + 1) * PIECES / NB; p++) unpack(j + 1, in, p, ln);
                }
            }
        }
        if (MIX && j + 2 < n_tile) issue(j + 2, in);
        const bool masked = __builtin_amdgcn_readfirstlane(row0 + (int)TILE > wmin || holes != 0 ? 1 : 0) != 0;
        auto sees = [&](uint32_t v) {
            return row0 + (int)(8 * (v >> 2) + 4 * hf + (v & 3u)) < my_vis && !(holes >> (v >> 3) & 1u);
        };
        if (masked) {
            keep_branch();
#pragma unroll
            for (uint32_t v = 0; v < 16; v++) S[v] = sees(v) ? S[v] : -INFINITY;
        }
        float mx = S[0];
#pragma unroll
        for (uint32_t v = 1; v < 16; v++) mx = fmaxf(mx, S[v]);
        mx = mx * qs;
        if (__builtin_amdgcn_ballot_w64(mx > ref + TOP) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float nr = fmaxf(ref, mx - FRESH);
            if (nr != ref) {
                const float c = __builtin_amdgcn_exp2f(ref - nr);
                lsum *= c;
#pragma unroll
                for (uint32_t b = 0; b < NB; b++)
#pragma unroll
                    for (uint32_t v = 0; v < 16; v++) O[b][v] = O[b][v] * c;
                ref = nr;
            }
            pin();
        }
        float ps[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t v = 0; v < 16; v++) {
            S[v] = __builtin_amdgcn_exp2f(fmaf(S[v], qs, -ref));   // (0 where masked)
            ps[v & 3u] += S[v];
        }
        lsum += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        f16x8 P[NP][2];
#pragma unroll
        for (uint32_t s = 0; s < 2; s++)
#pragma unroll
            for (uint32_t k = 0; k < 8; k += 2) {   // keys 0 2, 1 3, 4 6, 5 7
                const float p0 = S[8 * s + (k & 4) + ((k >> 1) & 1)], p1 = S[8 * s + (k & 4) + ((k >> 1) & 1) + 2];
                if constexpr (NP == 2) {
                    f16x2 hi, lo;
                    split2(p0, p1, hi, lo);
                    P[0][s][k] = hi.x; P[0][s][k + 1] = hi.y;
                    P[NP - 1][s][k] = lo.x; P[NP - 1][s][k + 1] = lo.y;
                } else {
                    P[0][s][k] = (_Float16)p0;
                    P[0][s][k + 1] = (_Float16)p1;
                }
            }
        f16x8 vf[PD + 1], vr[PD + 1];
#pragma unroll
        for (uint32_t m = 0; m < PD; m++) {
            vf[m] = fr(KF + m * 1024);
            if constexpr (NS == 2) vr[m] = fr(KF + VF + m * 1024);
        }
#pragma unroll
        for (uint32_t m = 0; m < 2 * NB; m++) {   // block m / 2, keys 16 (m % 2) ..
            const uint32_t b = m / 2, s = m & 1u;
            const f16x8 v = vf[m % (PD + 1)], r = vr[m % (PD + 1)];
            if (m + PD < 2 * NB) {
                vf[(m + PD) % (PD + 1)] = fr(KF + (m + PD) * 1024);
                if constexpr (NS == 2) vr[(m + PD) % (PD + 1)] = fr(KF + VF + (m + PD) * 1024);
            }
            O[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, P[0][s], O[b], 0, 0, 0);
            if constexpr (NP == 2) O[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, P[NP - 1][s], O[b], 0, 0, 0);
            if constexpr (NS == 2) O[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(r, P[0][s], O[b], 0, 0, 0);
            sched_fence();
        }
        pin();
        uint32_t any = 0;
#pragma unroll
        for (uint32_t b = 0; b < NB; b++) any |= ((const LDS uint32_t *)odd)[(j & 1) * 8 + b];
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(any) != 0, 0)) {
            const int n = my_vis - row0;
            const uint32_t mine = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
#pragma unroll
            for (uint32_t b = 0; b < NB; b++)
                if (((const LDS uint32_t *)odd)[(j & 1) * 8 + b] & mine) O[b] = O[b] + __builtin_nanf("");
            pin();
        }
    };

    if (n_tile > 0) {
        In in;
        issue(0, in);
        dma_wait();
        __syncthreads();
#pragma unroll
        for (uint32_t p = 0; p < PIECES; p++) unpack(0, in, p, lane);
        uint32_t holes = in.holes;
        if (n_tile > 1) issue(1, in);
        for (int j = 0; j < n_tile; j++) {
            dma_wait();        // tile j + 1's loads, issued an iteration ago
            __syncthreads();   // they are in from every wave; tile j is unpacked; tile j - 1 is done with
            // (behind the last tile its own loads are unpacked again, for nobody)
            const uint32_t h = in.holes;
            if (!MIX && w < 4) fetch(j, in);
            compute(j, holes, in);
            if (!MIX && w >= 4) fetch(j, in);
            holes = h;
        }
    }
    // Out through LDS, up to 128 dims of the wave's rows at a time, so that a
    // row's stores are consecutive: 16-byte unit u of row r in slot u ^ (r % UN)
    lsum += __shfl_xor(lsum, 32, 64);
    __syncthreads();   // (every wave is past its last tile: the fragments are free)
    LDS unsigned char *W = F + w * PASS;
#pragma unroll
    for (uint32_t h = 0; h < NB / PB; h++) {
#pragma unroll
        for (uint32_t b = 0; b < PB; b++)
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const f32x16 &o = O[h * PB + b];
                *reinterpret_cast<LDS f32x4 *>(W + 16 * (l32 * UN + ((8 * b + 2 * i + hf) ^ (l32 % UN)))) =
                    f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]};
            }
#pragma unroll 1
        for (uint32_t i = lane; i < 32 * UN; i += 64) {
            const uint32_t r = i / UN, u = i % UN, orow = r0 + 32 * w + r, e = 32 * PB * h + 4 * u;
            const f32x4 o = *reinterpret_cast<const LDS f32x4 *>(W + 16 * (r * UN + (u ^ (r % UN))));
            const float l = __shfl(lsum, (int)r, 64), m = __shfl(ref, (int)r, 64);
            if (orow >= M) continue;
            if (whole) {
                store_out(a, wk.tok0 + (int)(orow / a.gqa), g * a.gqa + orow % a.gqa, e, o, l);
            } else {
                const size_t rec = (((size_t)gt * NKV + g) * a.n_split + ck) * ROWS + 32 * w + r;
                *reinterpret_cast<f32x4 *>(a.tpart + rec * HD + e) = o;
                if (e == 0) a.tml[rec] = make_float2(m, l);
            }
        }
    }
}

// The chunks of kv4_tile_kernel's rows joined, one wave per (token, q head):
// reads each chunk's sums once.
template <int NW>
__global__ __launch_bounds__(256) void kv4_join_kernel(Attn a) {
    constexpr uint32_t ROWS = 32 * NW;
    const uint32_t u = blockIdx.x * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63u, HD = a.b.hd;
    if (u >= a.b.n_tok * a.nq) return;
    const uint32_t t = u / a.nq, h = u % a.nq;
    const int seq = seq_of(a.b, t);
    if (seq < 0) return;
    const Work wk = find_tile(a, ROWS, (uint32_t)seq, true);
    if (wk.seq < 0) return;
    const uint32_t i = t - (uint32_t)wk.tok0;
    if (i >= (uint32_t)wk.n_new || i >= a.max_q) return;
    const uint32_t g = h / a.gqa, row = i * a.gqa + h % a.gqa, tile = row / ROWS, M = (uint32_t)wk.n_new * a.gqa;
    const int last = wk.len - wk.n_new + (int)(min(tile * ROWS + ROWS - 1u, M - 1u) / a.gqa);
    const uint32_t seen = (uint32_t)max(0, min(last + 1, (int)row_cap(a))), per = chunk_rows(seen, a.n_split);
    if (seen <= per || wk.first + tile >= a.n_tile) return;
    const uint32_t n = (seen + per - 1u) / per;
    const size_t rec = (((size_t)(wk.first + tile) * a.b.nkv + g) * a.n_split) * ROWS + row % ROWS;
    float m = REF_NONE, l = 0.0f;
    for (uint32_t c = 0; c < n; c++) m = fmaxf(m, a.tml[rec + (size_t)c * ROWS].x);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t e = 4 * lane;
    for (uint32_t c = 0; c < n; c++) {
        const float2 ml = a.tml[rec + (size_t)c * ROWS];
        const f32x4 x = *reinterpret_cast<const f32x4 *>(a.tpart + (rec + (size_t)c * ROWS) * HD + (e < HD ? e : 0u));
        const float k = __builtin_amdgcn_exp2f(ml.x - m);
        l = fmaf(ml.y, k, l);
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = fmaf(x[j], k, o[j]);
    }
    if (e < HD) store_out(a, t, h, e, o, l);
}

// ------------------------------------------------------------------ host side

bool type_ok(int t) { return t == SINTER_F32 || t == SINTER_F16 || t == SINTER_BF16; }
int elem_bytes(int t) { return t == SINTER_F32 ? 4 : 2; }

// a launch of `blocks` workgroups has fewer than 2^32 threads
bool grid_ok(uint64_t blocks, uint32_t threads) { return blocks * threads < ((uint64_t)1 << 32); }

// the rows of a token array: pointer and strides of whole 16-byte units, no two
// rows overlapping (a stride that is never taken may be anything)
const char *check_heads(const sinter_heads &h, uint32_t n_tok, uint32_t heads, uint32_t hd, int type) {
    const int64_t eb = elem_bytes(type), ld = n_tok > 1 ? h.ld : 0, hs = heads > 1 ? h.hs : 0, most = (int64_t)1 << 40;
    if (!h.p) return "null pointer";
    if ((uintptr_t)h.p % 16u || ld % (16 / eb) || hs % (16 / eb)) return "pointer and strides must be multiples of 16 bytes";
    if ((n_tok > 1 && (ld < (int64_t)hd || ld > most)) || (heads > 1 && (hs < (int64_t)hd || hs > most)))
        return "strides must be at least hd";
    if (n_tok > 1 && heads > 1 && ld < (int64_t)(heads - 1) * hs + hd && hs < (int64_t)(n_tok - 1) * ld + hd)
        return "rows overlap";
    return nullptr;
}

int check_batch(const sinter_kv4_batch *b, const char *op, bool cache) {
    if (!b) return set_error(SINTER_ERR_ARG, "%s: null batch", op);
    if (b->hd != 64 && b->hd != 128 && b->hd != 256)
        return set_error(SINTER_ERR_ARG, "%s: head size %u (64, 128 or 256)", op, b->hd);
    if (b->nkv == 0 || b->nkv > 1024) return set_error(SINTER_ERR_ARG, "%s: %u kv heads (1..1024)", op, b->nkv);
    if (b->n_seq > 65536 || b->n_tok > (uint32_t)INT32_MAX)
        return set_error(SINTER_ERR_ARG, "%s: %u sequences (at most 65536), %u tokens", op, b->n_seq, b->n_tok);
    if (b->n_seq == 0 || b->n_tok == 0) return SINTER_OK;
    if (!b->tok_start || !b->kv_len || (uintptr_t)b->tok_start % 4u || (uintptr_t)b->kv_len % 4u)
        return set_error(SINTER_ERR_ARG, "%s: tok_start / kv_len null or misaligned", op);
    if (!cache) return SINTER_OK;
    if (!sinter_kv4_page_bytes(b->page_rows, b->nkv, b->hd))
        return set_error(SINTER_ERR_ARG, "%s: pages of %u rows (a power of two, 16..2^20, a page under 2^31 bytes)", op,
                         b->page_rows);
    if (b->max_pages == 0 || b->n_pages == 0 || b->n_pages > (uint32_t)INT32_MAX)
        return set_error(SINTER_ERR_ARG, "%s: %u table entries a sequence, %u pages", op, b->max_pages, b->n_pages);
    if (!b->pages || (uintptr_t)b->pages % 4u || !b->kc || !b->vc || (uintptr_t)b->kc % 16u || (uintptr_t)b->vc % 16u)
        return set_error(SINTER_ERR_ARG, "%s: pages (4 bytes) / caches (16 bytes) null or misaligned", op);
    return SINTER_OK;
}

int check_attn(const sinter_kv4_batch *b, const sinter_kv4_attn_args *a) {
    const int rc = check_batch(b, "kv4_attn", true);
    if (rc != SINTER_OK) return rc;
    if (!a) return set_error(SINTER_ERR_ARG, "kv4_attn: null arguments");
    if (!type_ok((int)a->type)) return set_error(SINTER_ERR_ARG, "kv4_attn: type %u (F32, F16 or BF16)", a->type);
    if (a->nq == 0 || a->nq % b->nkv || a->nq / b->nkv > 256)
        return set_error(SINTER_ERR_ARG, "kv4_attn: %u q heads over %u kv heads (a multiple, at most 256 each)", a->nq,
                         b->nkv);
    if (!(a->scale > 0.0f) || !std::isfinite(a->scale))
        return set_error(SINTER_ERR_ARG, "kv4_attn: scale must be positive and finite");
    if (b->n_seq && b->n_tok && (a->max_q == 0 || a->max_kv == 0 || a->max_kv > (uint32_t)INT32_MAX - 65536u))
        return set_error(SINTER_ERR_ARG, "kv4_attn: max_q %u / max_kv %u", a->max_q, a->max_kv);
    // (kv4_split_kernel counts its segments' tiles in 32 bits)
    const uint64_t segs = std::min<uint64_t>((uint64_t)b->n_tok * (a->nq / b->nkv) / 16 + b->n_seq, (uint64_t)b->n_seq * (SPLIT_MOST / 16));
    if (segs * ((a->max_kv + (uint64_t)TILE - 1) / TILE) > (uint64_t)INT32_MAX || (uint64_t)b->n_tok * a->nq > (uint64_t)INT32_MAX)
        return set_error(SINTER_ERR_ARG, "kv4_attn: batch too large (%u sequences of up to %u rows, %u tokens of %u heads)", b->n_seq,
                         a->max_kv, b->n_tok, a->nq);
    return SINTER_OK;
}

// Waves of a kv4_tile_kernel workgroup: F32's two parts of q and V fill the
// registers of one wave a SIMD; else two, and eight waves that unpack together
// rather than two workgroups of four (500 tokens behind 32,000 rows, 27B heads,
// bf16: 684 us against 587)
constexpr uint32_t tile_waves(bool f32) { return f32 ? 4 : 8; }

// f(the type as a constant)
template <class F>
void by_type(uint32_t type, F f) {
    if (type == SINTER_F32) f(std::integral_constant<uint32_t, SINTER_F32>());
    else if (type == SINTER_F16) f(std::integral_constant<uint32_t, SINTER_F16>());
    else f(std::integral_constant<uint32_t, SINTER_BF16>());
}

// Tokens a workgroup of append or read, and workgroups that share them, for
// `units` of a token of which a workgroup takes `wide` at a time: few tokens
// spread over many workgroups, many are taken together while that leaves
// 2048 workgroups.
uint64_t rows_grid(Rows &r, uint32_t units, uint32_t wide) {
    r.toks = std::min(TOKS, std::max(1u, r.b.n_tok / 2048u));
    const uint32_t groups = (r.b.n_tok + r.toks - 1) / r.toks;
    r.parts = std::min((units + wide - 1) / wide, std::max(1u, 2048u / groups));
    return (uint64_t)groups * r.parts;
}

// The launches of a batch.  kv4_split_kernel: row tiles a sequence, and slots,
// as many as run at once.  kv4_tile_kernel: row tiles (at most one
// partly filled one a sequence) and chunks of the cache rows a tile sees.
// Slots: the workgroups that run at once, two a CU by their LDS with heads of
// 256, three and four by registers with 128 and 64 (a reply behind 130,000 rows,
// heads of 256, 128: 48 and 42 us; half as many 51 and 52, twice as many 56 and 49)
uint32_t slots_at_once(uint32_t hd) { return hd == 256 ? 512 : hd == 128 ? 768 : 1024; }
struct Plan {
    uint32_t split_rows = 0, merge_rows = 0, n_slots = 0, n_tile = 0, n_split = 1;
    bool split = false, merge = false, join = false;
    uint64_t grid = 0, tile_grid = 0;
    size_t recs = 0, tile_recs = 0;
    size_t bytes(uint32_t hd) const { return (recs + tile_recs) * ((size_t)hd * 4 + 8); }
};
// (the work: 16-row segments of all tokens times the cache tiles they may see)
uint32_t split_rows(const sinter_kv4_batch &b, const sinter_kv4_attn_args &a) {
    const uint64_t segs = ((uint64_t)b.n_tok * (a.nq / b.nkv) + 15) / 16 * b.nkv;
    return segs * ((a.max_kv + TILE - 1) / TILE) <= 16384 ? SPLIT_MOST : SPLIT_ROWS;
}
Plan make_plan(const sinter_kv4_batch &b, const sinter_kv4_attn_args &a) {
    Plan p;
    const uint32_t gqa = a.nq / b.nkv;
    const uint64_t rows = (uint64_t)std::min(a.max_q, b.n_tok) * gqa;
    // (a sequence that all tokens may belong to, of many rows, is taken whole
    // by kv4_tile_kernel)
    p.split_rows = split_rows(b, a);
    p.split = gqa <= p.split_rows && (rows <= p.split_rows || b.n_seq > 1);
    if (p.split) {
        p.merge_rows = (uint32_t)std::min<uint64_t>(rows, p.split_rows / gqa * gqa);
        p.merge = a.max_kv > WHOLE * TILE;
        const uint64_t most = (uint64_t)b.n_seq * ((p.merge_rows + 15) / 16) * ((a.max_kv + CT_MIN * TILE - 1) / (CT_MIN * TILE) + 1);
        p.n_slots = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(1, slots_at_once(b.hd) / b.nkv), most);
        p.grid = (uint64_t)p.n_slots * b.nkv;
        p.recs = p.merge ? (size_t)p.grid * 32 : 0;
    }
    if (!p.split || rows > p.split_rows) {
        const uint64_t least = p.split ? p.split_rows / gqa + 1 : 1;   // tokens of a sequence that comes here
        const uint32_t tile_rows = 32 * tile_waves(a.type == SINTER_F32);
        p.n_tile = (uint32_t)((uint64_t)b.n_tok * gqa / tile_rows + std::min<uint64_t>(b.n_seq, b.n_tok / least));
        const uint64_t wgs = (uint64_t)p.n_tile * b.nkv, room = 256;
        // Chunks: the fewest cache tiles on the longest way through (rounds
        // of equal workgroups behind long contexts; the longest tile, or an
        // even share, of fresh prompts, whose tiles start longest first), a
        // workgroup's start and end counted as 5 cache tiles, a join as 8
        const double kv = (a.max_kv + TILE - 1) / TILE, fresh = std::min(1.0, (double)a.max_q / a.max_kv);
        double best = 1e300;
        for (uint32_t s = 1; s <= 32 && (s == 1 || a.max_kv / s >= CHUNK_MIN); s++) {
            const double rounds = std::ceil((double)(wgs * s) / room);
            const double cost = (fresh < 0.5 ? rounds / s : std::max(1.0 / s, 1.08 * wgs * (1.0 - fresh / 2) / room)) * kv +
                                5.0 * rounds + (s > 1 ? 8.0 : 0.0);
            if (cost < best) { best = cost; p.n_split = s; }
        }
        p.join = p.n_split > 1;
        p.tile_grid = wgs * p.n_split;
        p.tile_recs = p.join ? (size_t)p.tile_grid * tile_rows : 0;
    }
    return p;
}

template <int HD>
void launch_attn(const Attn &k, const Plan &p, hipStream_t s) {
    const bool f32 = k.type == SINTER_F32;
    if (p.tile_grid) {
        auto tile = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((uint32_t)p.tile_grid), dim3(64 * tile_waves(f32)), 0, s, k);
        };
        if (f32) tile(kv4_tile_kernel<HD, SINTER_F32, tile_waves(true)>);
        else if (k.type == SINTER_F16) tile(kv4_tile_kernel<HD, SINTER_F16, tile_waves(false)>);
        else tile(kv4_tile_kernel<HD, SINTER_BF16, tile_waves(false)>);
    }
    if (p.grid) {
        const dim3 grid(k.b.nkv, p.n_slots);
        if (f32) hipLaunchKernelGGL((kv4_split_kernel<HD, 2>), grid, dim3(256), 0, s, k);
        else hipLaunchKernelGGL((kv4_split_kernel<HD, 1>), grid, dim3(256), 0, s, k);
    }
}

}  // namespace

unsigned *kv4_err_cell() {
    void *p = nullptr;
    return hipGetSymbolAddress(&p, HIP_SYMBOL(g_kv4_err)) == hipSuccess ? static_cast<unsigned *>(p) : nullptr;
}

}  // namespace sinter

using namespace sinter;

extern "C" {

size_t sinter_kv4_page_bytes(uint32_t page_rows, uint32_t nkv, uint32_t hd) {
    if (page_rows < 16 || page_rows > (1u << 20) || (page_rows & (page_rows - 1u)) || nkv == 0 || nkv > 1024 ||
        (hd != 64 && hd != 128 && hd != 256))
        return 0;
    const size_t n = (size_t)page_rows * nkv * (hd / 2 + hd / 16);
    return n < ((size_t)1 << 31) ? n : 0;
}

int sinter_kv4_prep(const sinter_kv4_batch *b, const sinter_kv4_prep_args *a, void *stream) {
    const int rc = check_batch(b, "kv4_prep", false);
    if (rc != SINTER_OK) return rc;
    if (!a) return set_error(SINTER_ERR_ARG, "kv4_prep: null arguments");
    if (!type_ok((int)a->type)) return set_error(SINTER_ERR_ARG, "kv4_prep: type %u (F32, F16 or BF16)", a->type);
    if (a->rope_dims % 8 || a->rope_dims > b->hd)
        return set_error(SINTER_ERR_ARG, "kv4_prep: %u rope dims (a multiple of 8, at most the head size)", a->rope_dims);
    if (!(a->eps >= 0.0f) || (a->rope_dims && !(a->rope_base > 0.0f && std::isfinite(a->rope_base))))
        return set_error(SINTER_ERR_ARG, "kv4_prep: eps must be >= 0, rope_base positive and finite");
    if ((uintptr_t)a->q_norm % 16u || (uintptr_t)a->k_norm % 16u)
        return set_error(SINTER_ERR_ARG, "kv4_prep: norm weights must be 16-byte aligned");
    if (a->nq > 4096) return set_error(SINTER_ERR_ARG, "kv4_prep: %u q heads (at most 4096)", a->nq);
    if (b->n_seq == 0 || b->n_tok == 0) return SINTER_OK;
    const uint32_t nq = a->q.p || a->q_out.p ? a->nq : 0, nk = a->k.p || a->k_out.p ? b->nkv : 0;
    if (nq + nk == 0) return SINTER_OK;
    const char *why = nullptr;
    if (nq && ((why = check_heads(a->q, b->n_tok, nq, b->hd, (int)a->type)) || (why = check_heads(a->q_out, b->n_tok, nq, b->hd, (int)a->type))))
        return set_error(SINTER_ERR_ARG, "kv4_prep: q: %s", why);
    if (nk && ((why = check_heads(a->k, b->n_tok, nk, b->hd, (int)a->type)) || (why = check_heads(a->k_out, b->n_tok, nk, b->hd, (int)a->type))))
        return set_error(SINTER_ERR_ARG, "kv4_prep: k: %s", why);
    Prep p;
    p.b = *b;
    p.q = a->q; p.q_out = a->q_out; p.k = a->k; p.k_out = a->k_out;
    p.q_norm = a->q_norm; p.k_norm = a->k_norm;
    p.nq = nq; p.nk = nk; p.half = a->rope_dims / 2; p.eps = a->eps; p.inv_hd = 1.0f / (float)b->hd;   // (a power of two)
    p.rate = p.half ? std::log2((double)a->rope_base) / p.half : 0.0;
    // few tokens: a wave takes one group of heads; many: a workgroup a token
    const uint32_t per = 512 / b->hd, need = ((nq + per - 1) / per + (nk + per - 1) / per + 3) / 4;
    const dim3 grid(b->n_tok, b->n_tok >= 1024 ? 1u : need);
    if (!grid_ok(b->n_tok, 256)) return set_error(SINTER_ERR_ARG, "kv4_prep: too many tokens");
    by_type(a->type, [&](auto t) {
        hipLaunchKernelGGL(kv4_prep_kernel<decltype(t)::value>, grid, dim3(256), 0, (hipStream_t)stream, p);
    });
    return hip_ok(hipGetLastError(), "kv4_prep: launch") ? SINTER_OK : SINTER_ERR_HIP;
}

int sinter_kv4_append(const sinter_kv4_batch *b, const sinter_heads *k, const sinter_heads *v, int type, void *stream) {
    const int rc = check_batch(b, "kv4_append", true);
    if (rc != SINTER_OK) return rc;
    if (!type_ok(type)) return set_error(SINTER_ERR_ARG, "kv4_append: type %d (F32, F16 or BF16)", type);
    if (b->n_seq == 0 || b->n_tok == 0) return SINTER_OK;
    if (!k || !v) return set_error(SINTER_ERR_ARG, "kv4_append: null rows");
    const char *why;
    if ((why = check_heads(*k, b->n_tok, b->nkv, b->hd, type)) || (why = check_heads(*v, b->n_tok, b->nkv, b->hd, type)))
        return set_error(SINTER_ERR_ARG, "kv4_append: %s", why);
    Rows r;
    r.b = *b; r.k = *k; r.v = *v;
    const uint64_t grid = rows_grid(r, 2 * b->nkv * (b->hd / 32), 64);
    if (!grid_ok(grid, 256)) return set_error(SINTER_ERR_ARG, "kv4_append: too many tokens");
    by_type((uint32_t)type, [&](auto t) {
        hipLaunchKernelGGL(kv4_append_kernel<decltype(t)::value>, dim3((uint32_t)grid), dim3(256), 0, (hipStream_t)stream, r);
    });
    return hip_ok(hipGetLastError(), "kv4_append: launch") ? SINTER_OK : SINTER_ERR_HIP;
}

int sinter_kv4_read(const sinter_kv4_batch *b, const sinter_heads *k, const sinter_heads *v, int type, void *stream) {
    const int rc = check_batch(b, "kv4_read", true);
    if (rc != SINTER_OK) return rc;
    if (!type_ok(type)) return set_error(SINTER_ERR_ARG, "kv4_read: type %d (F32, F16 or BF16)", type);
    if (b->n_seq == 0 || b->n_tok == 0) return SINTER_OK;
    Rows r;
    r.b = *b;
    r.k = k ? *k : sinter_heads{}; r.v = v ? *v : sinter_heads{};
    if (!r.k.p && !r.v.p) return set_error(SINTER_ERR_ARG, "kv4_read: nowhere to write");
    const char *why;
    if ((r.k.p && (why = check_heads(r.k, b->n_tok, b->nkv, b->hd, type))) || (r.v.p && (why = check_heads(r.v, b->n_tok, b->nkv, b->hd, type))))
        return set_error(SINTER_ERR_ARG, "kv4_read: %s", why);
    const uint32_t el = type == SINTER_F32 ? 4 : 8, both = r.k.p && r.v.p ? 2 : 1;
    const uint64_t grid = rows_grid(r, both * b->nkv * (b->hd / el), 256);
    if (!grid_ok(grid, 256)) return set_error(SINTER_ERR_ARG, "kv4_read: too many tokens");
    by_type((uint32_t)type, [&](auto t) {
        hipLaunchKernelGGL(kv4_read_kernel<decltype(t)::value>, dim3((uint32_t)grid), dim3(256), 0, (hipStream_t)stream, r);
    });
    return hip_ok(hipGetLastError(), "kv4_read: launch") ? SINTER_OK : SINTER_ERR_HIP;
}

size_t sinter_kv4_attn_ws_bytes(const sinter_kv4_batch *b, const sinter_kv4_attn_args *a) {
    if (check_attn(b, a) != SINTER_OK || b->n_seq == 0 || b->n_tok == 0) return 0;
    return make_plan(*b, *a).bytes(b->hd);
}

int sinter_kv4_attn(const sinter_kv4_batch *b, const sinter_kv4_attn_args *a, void *stream) {
    const int rc = check_attn(b, a);
    if (rc != SINTER_OK) return rc;
    if (b->n_seq == 0 || b->n_tok == 0) return SINTER_OK;
    const char *why;
    if ((why = check_heads(a->q, b->n_tok, a->nq, b->hd, (int)a->type)) || (why = check_heads(a->out, b->n_tok, a->nq, b->hd, (int)a->type)) ||
        (a->gate.p && (why = check_heads(a->gate, b->n_tok, a->nq, b->hd, (int)a->type))))
        return set_error(SINTER_ERR_ARG, "kv4_attn: %s", why);
    const Plan p = make_plan(*b, *a);
    const size_t need = p.bytes(b->hd);
    if (need && (!a->ws || (uintptr_t)a->ws % 16u || a->ws_bytes < need))
        return set_error(SINTER_ERR_ARG, "kv4_attn: workspace of %zu bytes, 16-byte aligned (sinter_kv4_attn_ws_bytes)", need);
    const uint32_t out_rows = b->n_tok * a->nq, segs = b->n_seq * ((p.merge_rows + 15) / 16);
    // Waves of a merging workgroup: sixteen where a row may have many parts (a
    // reply behind 130,000 rows: 48.5 us, four 54), four where the rows are many
    // (64 behind 3000: 70 us, sixteen 74)
    const uint32_t wide = p.n_slots > 32 * segs ? 16 : 4;
    if (!grid_ok(p.tile_grid, 64 * tile_waves(a->type == SINTER_F32)) || (p.join && !grid_ok((out_rows + 3) / 4, 256)) ||
        (p.merge && !grid_ok((uint64_t)b->n_seq * b->nkv * p.merge_rows, 64 * wide)))
        return set_error(SINTER_ERR_ARG, "kv4_attn: batch too large");
    Attn k;
    k.b = *b;
    k.q = a->q; k.gate = a->gate; k.out = a->out;
    k.part = static_cast<float *>(a->ws);
    k.tpart = k.part + p.recs * b->hd;
    k.ml = reinterpret_cast<float2 *>(k.tpart + p.tile_recs * b->hd);
    k.tml = k.ml + p.recs;
    k.nq = a->nq; k.gqa = a->nq / b->nkv; k.max_q = a->max_q; k.max_kv = a->max_kv;
    k.n_slots = p.n_slots; k.type = a->type;
    k.n_tile = p.n_tile; k.n_split = p.n_split; k.report = !p.split; k.split_rows = p.split ? p.split_rows : 0;
    k.page_shift = (uint32_t)__builtin_ctz(b->page_rows);
    k.qscale = a->scale * 1.44269504088896341f;
    k.gqa_inv = (uint32_t)((((uint64_t)1 << 32) + k.gqa - 1) / k.gqa);
    const hipStream_t s = (hipStream_t)stream;
    if (b->hd == 256) launch_attn<256>(k, p, s);
    else if (b->hd == 128) launch_attn<128>(k, p, s);
    else launch_attn<64>(k, p, s);
    if (!hip_ok(hipGetLastError(), "kv4_attn: launch")) return SINTER_ERR_HIP;
    if (p.join) {
        if (a->type == SINTER_F32) hipLaunchKernelGGL((kv4_join_kernel<tile_waves(true)>), dim3((out_rows + 3) / 4), dim3(256), 0, s, k);
        else hipLaunchKernelGGL((kv4_join_kernel<tile_waves(false)>), dim3((out_rows + 3) / 4), dim3(256), 0, s, k);
    }
    if (p.merge) {
        const dim3 grid(b->n_seq * b->nkv * p.merge_rows);
        if (wide == 16) hipLaunchKernelGGL((kv4_merge_kernel<16>), grid, dim3(1024), 0, s, k, p.merge_rows);
        else hipLaunchKernelGGL((kv4_merge_kernel<4>), grid, dim3(256), 0, s, k, p.merge_rows);
    }
    return hip_ok(hipGetLastError(), "kv4_attn: merge launch") ? SINTER_OK : SINTER_ERR_HIP;
}

}  // extern "C"
