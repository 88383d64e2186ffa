// The 4-bit paged KV cache of a batch of sequences: q/k norm and rotation at
// the batch's positions, the quantising append, the read back and causal
// attention over the cache (sinter_kv4_*, include/sinter.h).
//
//   kv4_prep_kernel    RMSNorm + NEOX RoPE of q and k heads
//   kv4_append_kernel  k, v rows quantised into the cache's pages
//   kv4_read_kernel    cache rows back to f32 / f16 / bf16
//   kv4_split_kernel   attention of 16 (token, head) rows over a chunk of cache rows
//   kv4_merge_kernel   the chunks' partials of a row joined
//
// A page holds per kv head page_rows rows of codes (hd / 2 bytes; byte 16 b +
// i of a row holds elements 32 b + i and 32 b + 16 + i in its low and high
// four bits), then page_rows rows of hd / 32 f16 scales: both planes are whole
// 16-byte units, contiguous over a page, so that a wave streams them by
// LDS-DMA with nothing read twice.  Element = scale * (code - 8).
#include <algorithm>
#include <cmath>

#include "dev_common.h"
#include "internal.h"

namespace sinter {

// the first device error of this unit's kernels: [0] code, [1] aux (a sequence)
__device__ unsigned g_kv4_err[2];

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
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
    if (type == SINTER_BF16) return (uint32_t)f2bf(a) | ((uint32_t)f2bf(b) << 16);
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

// ------------------------------------------------------------------ the batch

// the sequence that token t belongs to (wave-uniform), or -1
__device__ __forceinline__ int seq_of(const sinter_kv4_batch &b, uint32_t t) {
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t base = 0; base < b.n_seq; base += 64) {
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

// the position of token t, or -1 where it has none (behind the last sequence,
// or before row 0 of its own)
__device__ __forceinline__ int token_pos(const sinter_kv4_batch &b, uint32_t t, int &seq) {
    seq = seq_of(b, t);
    if (seq < 0) return -1;
    return max(b.kv_len[seq] - (b.tok_start[seq + 1] - (int)t), -1);
}

// the page that row `pos` of sequence `seq` lies in, or -1 (and the error
// raised) where the table has none
__device__ __forceinline__ int page_of(const sinter_kv4_batch &b, int seq, int pos) {
    const uint32_t e = (uint32_t)pos / b.page_rows;
    const int page = e < b.max_pages ? b.pages[(size_t)seq * b.max_pages + e] : -1;
    if ((uint32_t)page < b.n_pages) return page;
    if ((threadIdx.x & 63u) == 0) raise_error(g_kv4_err, SINTER_E_BAD_SHAPE, (unsigned)seq);
    return -1;
}

// ------------------------------------------------------------------ prep

struct Prep {
    sinter_kv4_batch b;
    sinter_heads q, q_out, k, k_out;
    const float *q_norm, *k_norm;
    double rate;   // log2(base) / (rope_dims / 2)
    uint32_t nq, half, type, heads;
    float eps;
};

// y = x / sqrt(mean(x^2) + eps) * w, then the pairs (i, i + half) turned by
// pos * base^(-i / half).  The angle is held in turns in fp64 (at position
// 131072 an fp32 angle is off by thousandths of a radian), once a token and
// workgroup.  A head is hd / 4 lanes of four elements.  blockIdx.y: a
// workgroup's share of the heads.
__global__ __launch_bounds__(256) void kv4_prep_kernel(Prep a) {
    __shared__ float2 turn[128];
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 63u;
    int seq;
    const int pos = token_pos(a.b, t, seq);
    if (pos < 0) return;   // (uniform)
    if (threadIdx.x < a.half) {
        const double f = exp2(-(double)threadIdx.x * a.rate) * 0.15915494309189533577;   // 1 / (2 pi)
        const double x = (double)pos * f, fr = x - rint(x);
        double s, c;
        sincospi(2.0 * fr, &s, &c);
        turn[threadIdx.x] = make_float2((float)c, (float)s);
    }
    __syncthreads();
    const uint32_t hd = a.b.hd, lph = hd / 4, l = lane % lph, wave = threadIdx.x >> 6, per = 64 / lph;
    const uint32_t quarter = a.half / 4;
    for (uint32_t h0 = (blockIdx.y * 4 + wave) * per; h0 < a.heads; h0 += gridDim.y * 4 * per) {
        const uint32_t h = h0 + lane / lph;
        const bool live = h < a.heads;
        const bool isq = h < a.nq;
        const uint32_t hh = live ? (isq ? h : h - a.nq) : 0u;
        const sinter_heads &src = !live || isq ? a.q : a.k, &dst = !live || isq ? a.q_out : a.k_out;
        const float *w = !live || isq ? a.q_norm : a.k_norm;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (live) x = load4(src.p, (int64_t)t * src.ld + (int64_t)hh * src.hs + 4 * l, a.type);
        float ss = lanes_sum_f32(x.x * x.x + x.y * x.y + (x.z * x.z + x.w * x.w), lph);
        const float r = 1.0f / sqrtf(ss / (float)hd + a.eps);
        float y[4] = {x.x * r, x.y * r, x.z * r, x.w * r};
        if (w) {
            const float4 wt = reinterpret_cast<const float4 *>(w)[l];
            y[0] *= wt.x; y[1] *= wt.y; y[2] *= wt.z; y[3] *= wt.w;
        }
        const bool lo = l < quarter, in = l < 2 * quarter;
        const int partner = (int)(lane + (lo ? quarter : in ? 0u - quarter : 0u));
#pragma unroll
        for (uint32_t c = 0; c < 4; c++) {
            const float o = __shfl(y[c], partner, 64);
            if (in) {
                const float2 cs = turn[4 * (lo ? l : l - quarter) + c];
                y[c] = y[c] * cs.x + (lo ? -o : o) * cs.y;
            }
        }
        if (live)
            store4(dst.p, (int64_t)t * dst.ld + (int64_t)hh * dst.hs + 4 * l, a.type, make_float4(y[0], y[1], y[2], y[3]));
    }
}

// ------------------------------------------------------------------ append

struct Rows {
    sinter_kv4_batch b;
    sinter_heads k, v;
    uint32_t type, per;   // per: workgroups a token
};

// Eight lanes quantise one block of 32, four elements each: m = the first
// element of the largest magnitude (saturated at the f16 maximum), d = m / -8,
// code = min(15, trunc(x / d + 8.5)) by the product with 1 / d, in fp32 with
// every product and sum rounded (ggml's Q4_0 reference quantiser).  A block
// whose f16 scale is zero has every code 8; one with a NaN has a NaN scale.
__global__ __launch_bounds__(256) void kv4_append_kernel(Rows a) {
    const uint32_t t = blockIdx.x / a.per, lane = threadIdx.x & 63u;
    const uint32_t nb = a.b.hd / 32, nblk = a.b.nkv * nb;
    int seq;
    const int pos = token_pos(a.b, t, seq);
    if (pos < 0) return;
    const int page = page_of(a.b, seq, pos);
    if (page < 0) return;
    const uint32_t i = (blockIdx.x % a.per) * 32u + threadIdx.x / 8u;   // K's blocks, then V's
    if (i >= 2 * nblk) return;                                           // (whole groups of eight lanes)
    const bool isv = i >= nblk;
    const uint32_t j = isv ? i - nblk : i, g = j / nb, bl = j % nb, l8 = lane & 7u;
    const sinter_heads &src = isv ? a.v : a.k;
    const float4 x4 = load4(src.p, (int64_t)t * src.ld + (int64_t)g * src.hs + 32 * bl + 4 * l8, a.type);
    float x[4] = {x4.x, x4.y, x4.z, x4.w};
    float am = 0.0f;
    bool nan = false;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        nan |= x[c] != x[c];
        x[c] = fminf(fmaxf(x[c], -F16_MAX), F16_MAX);
        am = fmaxf(am, fabsf(x[c]));
    }
    am = fmaxf(am, dpp_f<DPP_XOR1>(am));
    am = fmaxf(am, dpp_f<DPP_XOR2>(am));
    am = fmaxf(am, dpp_f<DPP_HALF_MIRROR>(am));
    // the first element of that magnitude: its place and sign in one integer
    int at = 64 + (nan ? -128 : 0);
#pragma unroll
    for (int c = 3; c >= 0; c--)
        if (fabsf(x[c]) == am && !nan) at = 2 * (int)(4 * l8 + c) + (x[c] > 0.0f ? 1 : 0);
    at = min(at, dpp_i<DPP_XOR1>(at));
    at = min(at, dpp_i<DPP_XOR2>(at));
    at = min(at, dpp_i<DPP_HALF_MIRROR>(at));
    const float d = (at & 1 ? am : -am) / -8.0f;
    uint16_t dh = f2h(d);
    const bool zero = (dh & 0x7fffu) == 0;
    if (zero) dh = 0;
    if (at < 0) dh = 0x7e00u;
    const float inv = zero ? 0.0f : 1.0f / d;
    uint32_t q = 0;
#pragma unroll
    for (int c = 0; c < 4; c++) q |= (uint32_t)min(15, (int)(x[c] * inv + 8.5f)) << (8 * c);
    if (at < 0) q = 0x08080808u;
    // lane l8 < 4 joins lane l8 + 4's codes (elements 16 further) above its own
    const uint32_t hi = (uint32_t)dpp_i<0x1B>(dpp_i<DPP_HALF_MIRROR>((int)q));   // (quad_perm [3,2,1,0])
    const uint32_t rows = a.b.page_rows, hb = a.b.hd / 2, row = (uint32_t)pos & (rows - 1u);
    unsigned char *head = static_cast<unsigned char *>(isv ? a.b.vc : a.b.kc) +
                          ((size_t)(uint32_t)page * a.b.nkv + g) * ((size_t)rows * (hb + hb / 8));
    if (l8 < 4) *reinterpret_cast<uint32_t *>(head + (size_t)row * hb + 16 * bl + 4 * l8) = q | (hi << 4);
    if (l8 == 0) *reinterpret_cast<uint16_t *>(head + (size_t)rows * hb + (size_t)row * (hb / 8) + 2 * bl) = dh;
}

// ------------------------------------------------------------------ read

// A thread gives back the 16 elements of eight code bytes (half a block).
__global__ __launch_bounds__(256) void kv4_read_kernel(Rows a) {
    const uint32_t t = blockIdx.x / a.per;
    const uint32_t nb = a.b.hd / 32, nun = a.b.nkv * nb * 2;
    int seq;
    const int pos = token_pos(a.b, t, seq);
    if (pos < 0) return;
    const int page = page_of(a.b, seq, pos);
    if (page < 0) return;
    const uint32_t i = (blockIdx.x % a.per) * 256u + threadIdx.x;
    if (i >= 2 * nun) return;
    const bool isv = i >= nun;
    const sinter_heads &dst = isv ? a.v : a.k;
    if (!dst.p) return;
    const uint32_t j = isv ? i - nun : i, g = j / (2 * nb), bl = (j / 2) % nb, hf = j & 1u;
    const uint32_t rows = a.b.page_rows, hb = a.b.hd / 2, row = (uint32_t)pos & (rows - 1u);
    const unsigned char *head = static_cast<const unsigned char *>(isv ? a.b.vc : a.b.kc) +
                                ((size_t)(uint32_t)page * a.b.nkv + g) * ((size_t)rows * (hb + hb / 8));
    const u32x2 w = *reinterpret_cast<const u32x2 *>(head + (size_t)row * hb + 16 * bl + 8 * hf);
    const float d = h2f(*reinterpret_cast<const uint16_t *>(head + (size_t)rows * hb + (size_t)row * (hb / 8) + 2 * bl));
    const int64_t e = (int64_t)t * dst.ld + (int64_t)g * dst.hs + 32 * bl + 8 * hf;
#pragma unroll
    for (uint32_t s = 0; s < 2; s++)
#pragma unroll
        for (uint32_t c = 0; c < 2; c++) {
            const uint32_t u = (c ? w.y : w.x) >> (4 * s);
            auto val = [&](uint32_t k) { return (float)((int)((u >> (8 * k)) & 15u) - 8) * d; };
            store4(dst.p, e + 16 * s + 4 * c, a.type, make_float4(val(0), val(1), val(2), val(3)));
        }
}

// ------------------------------------------------------------------ attention

// Chunks of a sequence's rows that one workgroup takes, in 32-row tiles:
// at least CT_MIN (below it a workgroup's start costs more than its rows)
constexpr uint32_t TILE = 32, CT_MIN = 16;

struct Attn {
    sinter_kv4_batch b;
    sinter_heads q, gate, out;
    float *part;     // [slot][kv head][row tile][16][hd] unnormalised sums
    float2 *ml;      // [slot][kv head][row tile][16] reference and weight sum
    uint32_t nq, gqa, max_q, max_kv, n_slots, n_mt, type, page_shift;
    float qscale;    // scale * log2(e)
};

struct Work {
    int seq, len, tok0, n_new;   // the sequence: rows, first token, tokens (seq < 0: none)
    uint32_t chunk, first, ct;   // the chunk of it, the slot of its chunk 0, tiles a chunk
};

// The chunks of all sequences lie in slots one after the other: ct tiles each,
// the smallest ct for which they fit the launch's slots (sum of ceil(tiles /
// ct) <= tiles / (n_slots - n_seq) + n_seq); a sequence with tokens has at
// least one.  Finds slot `slot`'s work, or (by_seq) sequence `slot`'s first.
__device__ __forceinline__ Work find_work(const Attn &a, uint32_t slot, bool by_seq, bool report) {
    const uint32_t lane = threadIdx.x & 63u;
    const sinter_kv4_batch &b = a.b;
    auto load = [&](uint32_t base, int &len, int &t0, int &n) {
        const uint32_t i = min(base + lane, b.n_seq - 1u);
        t0 = b.tok_start[i];
        n = b.tok_start[i + 1] - t0;
        len = b.kv_len[i];
        if (base + lane >= b.n_seq) n = 0;
        const uint32_t cap = (uint32_t)min((uint64_t)a.max_kv, (uint64_t)b.max_pages << a.page_shift);
        if (report && n > 0 && (len < 0 || (uint32_t)len > cap || (uint32_t)n > a.max_q || t0 < 0 || (uint32_t)(t0 + n) > b.n_tok))
            raise_error(g_kv4_err, SINTER_E_BAD_SHAPE, base + lane);
        // (tokens outside the arrays are nobody's)
        if (t0 < 0 || n <= 0 || (uint32_t)t0 >= b.n_tok) n = 0;
        else n = min(n, (int)(b.n_tok - (uint32_t)t0));
        len = max(0, len);
    };
    auto tiles_of = [&](int len, int n) {
        const uint32_t cap = (uint32_t)min((uint64_t)a.max_kv, (uint64_t)b.max_pages << a.page_shift);
        return n > 0 ? max(1u, (min((uint32_t)len, cap) + TILE - 1u) / TILE) : 0u;
    };
    int len, t0, n;
    uint32_t total = 0;
    for (uint32_t base = 0; base < b.n_seq; base += 64) {
        load(base, len, t0, n);
        uint32_t v = tiles_of(len, n);
        v += (uint32_t)dpp_i<DPP_XOR1>((int)v);
        v += (uint32_t)dpp_i<DPP_XOR2>((int)v);
        v += (uint32_t)dpp_i<DPP_HALF_MIRROR>((int)v);
        v += (uint32_t)dpp_i<DPP_MIRROR>((int)v);
#pragma unroll
        for (int r = 0; r < 4; r++) total += (uint32_t)__builtin_amdgcn_readlane((int)v, 16 * r);
    }
    const uint32_t room = a.n_slots - b.n_seq;
    Work w;
    w.seq = -1;
    w.ct = max(CT_MIN, room ? (total + room - 1u) / room : 0x7fffffu);
    uint32_t before = 0;
    for (uint32_t base = 0; base < b.n_seq; base += 64) {
        if (b.n_seq > 64) load(base, len, t0, n);
        const uint32_t c = n > 0 ? (tiles_of(len, n) + w.ct - 1u) / w.ct : 0u;
        uint32_t sum = c;   // inclusive over the lanes
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t p = (uint32_t)__shfl_up((int)sum, o, 64);
            if (lane >= (uint32_t)o) sum += p;
        }
        const uint32_t lo = before + sum - c;
        const bool mine = by_seq ? base + lane == slot && n > 0 : slot >= lo && slot < lo + c;
        const uint64_t m = __builtin_amdgcn_ballot_w64(mine);
        if (m != 0) {
            const int l = __builtin_ctzll(m);
            w.seq = (int)base + l;
            w.len = __builtin_amdgcn_readlane(len, l);
            w.tok0 = __builtin_amdgcn_readlane(t0, l);
            w.n_new = __builtin_amdgcn_readlane(n, l);
            w.first = (uint32_t)__builtin_amdgcn_readlane((int)lo, l);
            w.chunk = by_seq ? 0u : slot - w.first;
            return w;
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    }
    return w;
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
__device__ __forceinline__ f16x2 code_pair_lo(uint32_t w) {
    const f16x2 v = __builtin_bit_cast(f16x2, (w & 0x000f000fu) | 0x64006400u);
    return v + f16x2{(_Float16)-1032.0f, (_Float16)-1032.0f};
}
__device__ __forceinline__ f16x2 code_pair_hi(uint32_t w) {
    const f16x2 v = __builtin_bit_cast(f16x2, (w & 0x00f000f0u) | 0x64006400u);
    return __builtin_elementwise_fma(v, f16x2{(_Float16)0.0625f, (_Float16)0.0625f},
                                     f16x2{(_Float16)-72.0f, (_Float16)-72.0f});
}
__device__ __forceinline__ f16x8 join8(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The reference of a row's weights: p = exp2(s - ref), with s in log2 units.
// p * d enters the matrix cores as f16, so ref keeps p * |d| <= 2^TOP for the
// largest scale seen, 2^dlog; a new reference leaves the largest at 2^FRESH.
constexpr float TOP = 15.0f, FRESH = 6.0f;

// Work item: (chunk slot, kv head, tile of 16 rows), a row being a (token, q
// head of the group) pair, token-major.  Each wave streams its own 32-row
// tiles of the chunk (every fourth) through a private double buffer filled by
// LDS-DMA, so that no barrier stands between the first tile and the last.
//
// Scores S^T = K Q^T on 16x16x32 f16 MFMA, one per block of 32 dims: the codes
// are exact in f16, the block's scale multiplies the fp32 sum (one fma), and q
// is exact (f16, bf16 after a power-of-two scale of its row) or split into two
// f16 parts (f32: 22 bits; NS = 2).  D then holds key 4 g + v, row l % 16 in
// lane l (g = l / 16), which is the B operand's layout of P^T in O^T = V^T P^T
// with the keys in that order: P never leaves its lane.  V's operand comes
// from a transposing LDS read, eight keys' byte of one dim pair per lane; its
// scales multiply P (per block, in fp32, rounded once to f16, or to two parts).
template <int HD, int NS>
__global__ __launch_bounds__(256, 2) void kv4_split_kernel(Attn a) {
    constexpr uint32_t NB = HD / 32, HB = HD / 2, SB = HD / 16, NCH = HB / 16, KC = TILE * HB, SC = TILE * SB;
    constexpr uint32_t STAGE = 2 * KC + 2 * SC, NI = TILE * NCH / 64, SH = HD == 256 ? 1 : HD == 128 ? 2 : 3;
    constexpr uint32_t OST = HD + 4, RING = 4 * 2 * STAGE, COMB = 4 * 16 * OST * 4;
    __shared__ __attribute__((aligned(16))) unsigned char sm[RING > COMB ? RING : COMB];
    __shared__ float red[2][4][16];
    const uint32_t lane = threadIdx.x & 63u, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r16 = lane & 15u, g4 = lane >> 4, NKV = a.b.nkv;
    const uint32_t per = a.n_slots * NKV, mt = blockIdx.x / per, it = blockIdx.x % per;
    const uint32_t g = it % NKV, slot = it / NKV;
    const Work wk = find_work(a, slot, false, it == 0 && mt == 0 && w == 0);
    if (wk.seq < 0) return;
    const uint32_t M = (uint32_t)wk.n_new * a.gqa;
    if (16 * mt >= M) return;
    const uint32_t rows = min(16u, M - 16 * mt);
    const int p0 = wk.len - wk.n_new;   // the first token's position
    auto row_pos = [&](uint32_t r) { return p0 + (int)((16 * mt + r) / a.gqa); };
    const int pmin = row_pos(0), pmax = row_pos(rows - 1), c0 = (int)(wk.chunk * wk.ct * TILE);
    if (wk.chunk > 0 && c0 > pmax) return;
    const int cap = (int)min((uint64_t)a.max_kv, (uint64_t)a.b.max_pages << a.page_shift);
    const int end = min(min(c0 + (int)(wk.ct * TILE), pmax + 1), cap);   // rows [c0, end)
    const int my_vis = r16 < rows ? min(row_pos(r16) + 1, end) : end;     // of them this lane's row sees [c0, my_vis)
    const int n_tile = end > c0 ? (end - c0 + (int)TILE - 1) / (int)TILE : 0;

    // the row's q: dims 32 b + {4 g, .., 4 g + 3} and 16 further, in the codes' order
    f16x8 Q[NS][NB];
    float qs;
    {
        const uint32_t r = 16 * mt + min(r16, rows - 1);
        const int64_t e0 = (int64_t)(wk.tok0 + (int)(r / a.gqa)) * a.q.ld + (int64_t)(g * a.gqa + r % a.gqa) * a.q.hs + 4 * g4;
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

    f32x4 O[2 * NB];
#pragma unroll
    for (uint32_t i = 0; i < 2 * NB; i++) O[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float ref = REF_NONE, lim = REF_NONE, lsum = 0.0f;
    float dtop = 0.0f, dlog = -24.0f;   // every V scale so far is at most dtop = 2^dlog (dtop 0: none yet)
    const int nt = (n_tile - (int)w + 3) / 4;
    if (nt > 0) issue((int)w, 0);
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
        float s[2][4];
#pragma unroll
        for (uint32_t h = 0; h < 2; h++) {
            sched_fence();
            uint32_t d[4][NB / 2];   // scales of keys 4 g + v, two blocks a word
#pragma unroll
            for (uint32_t v = 0; v < 4; v++)
#pragma unroll
                for (uint32_t b = 0; b < NB / 2; b++)
                    d[v][b] = reinterpret_cast<const LDS uint32_t *>(ks + (16 * h + 4 * g4 + v) * SB)[b];
#pragma unroll
            for (uint32_t v = 0; v < 4; v++) s[h][v] = 0.0f;
            const uint32_t r = 16 * h + r16;
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) {
                const uint32_t x = *reinterpret_cast<const LDS uint32_t *>(kt + r * HB + 16 * (b ^ swz(r)) + 4 * g4);
                const f16x8 A = join8(code_pair_lo(x), code_pair_lo(x >> 8), code_pair_hi(x), code_pair_hi(x >> 8));
                f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
                t = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, Q[0][b], t, 0, 0, 0);
                if constexpr (NS == 2) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, Q[NS - 1][b], t, 0, 0, 0);
#pragma unroll
                for (uint32_t v = 0; v < 4; v++) {
                    const f16x2 dd = __builtin_bit_cast(f16x2, d[v][b / 2]);
                    s[h][v] = fmaf(t[v], (float)(b & 1 ? dd.y : dd.x), s[h][v]);
                }
            }
        }
        sched_fence();
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
        const bool masked = row0 + (int)TILE > min(end, pmin + 1) || hole != 0;
        float p[8];
        bool ok[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            p[k] = s[k >> 2][k & 3] * qs;
            ok[k] = true;
        }
        if (masked) {
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) {
                ok[k] = row0 + (int)(16 * (k >> 2) + 4 * g4 + (k & 3)) < my_vis && !(hole >> (k >> 2) & 1u);
                p[k] = ok[k] ? p[k] : -INFINITY;
                // (a masked row's scale may be anything: 0 keeps it out)
#pragma unroll
                for (uint32_t b = 0; b < NB / 2; b++) dv[k][b] = ok[k] ? dv[k][b] : 0u;
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
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
            p[k] = __builtin_amdgcn_exp2f(p[k] - ref);
            if (masked) p[k] = ok[k] ? p[k] : 0.0f;
            lsum += p[k];
        }
        // V^T: lane i of a group of 16 reads half i % 2 of row key(i / 2) and
        // gets byte i of the block for the group's eight keys
        const uint32_t kr = (r16 >> 1), vr = 16 * (kr >> 2) + 4 * g4 + (kr & 3);
#pragma unroll
        for (uint32_t b = 0; b < NB; b++) {
            if (b % 2 == 0) sched_fence();
            const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (LDS i32x2 *)(vt + vr * HB + 16 * (b ^ swz(vr)) + 8 * (r16 & 1u)));
            const uint32_t x0 = (uint32_t)x.x, x1 = (uint32_t)x.y;
            const f16x8 Al = join8(code_pair_lo(x0), code_pair_lo(x0 >> 8), code_pair_lo(x1), code_pair_lo(x1 >> 8));
            const f16x8 Ah = join8(code_pair_hi(x0), code_pair_hi(x0 >> 8), code_pair_hi(x1), code_pair_hi(x1 >> 8));
            f16x8 P, Pl;
#pragma unroll
            for (uint32_t k = 0; k < 8; k++) {
                const uint32_t key = (k & 4) | ((k & 1) << 1) | ((k >> 1) & 1);   // 0 2 1 3 4 6 5 7
                const f16x2 dd = __builtin_bit_cast(f16x2, dv[key][b / 2]);
                const float dk = (float)(b & 1 ? dd.y : dd.x);
                if constexpr (NS == 1) {
                    P[k] = (_Float16)fmaf(p[key], dk, 0.0f);
                } else {
                    // (opaque: rounded to f16 straight from the product in one
                    // place and from the fp32 product in the other, the parts
                    // would not add up)
                    float x = p[key] * dk;
                    asm volatile("" : "+v"(x));
                    P[k] = (_Float16)x;
                    Pl[k] = (_Float16)(x - (float)P[k]);
                }
            }
            O[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Al, P, O[2 * b], 0, 0, 0);
            O[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Ah, P, O[2 * b + 1], 0, 0, 0);
            if constexpr (NS == 2) {
                O[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Al, Pl, O[2 * b], 0, 0, 0);
                O[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(Ah, Pl, O[2 * b + 1], 0, 0, 0);
            }
        }
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
        const int pos = min(row_pos(r), cap - 1);   // (cap: rows the launch and the table have room for)
        if (pos < c0 && wk.chunk > 0) continue;   // (the row ends before this chunk)
        if (pos < (int)(wk.ct * TILE)) {   // the row sees chunk 0 alone
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            const int64_t t = wk.tok0 + (int)((16 * mt + r) / a.gqa), h = g * a.gqa + (16 * mt + r) % a.gqa;
            float4 y = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            if (a.gate.p) {
                const float4 z = load4(a.gate.p, t * a.gate.ld + h * a.gate.hs + e, a.type);
                auto sig = [](float x) { return 1.0f / (1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f)); };
                y = make_float4(y.x * sig(z.x), y.y * sig(z.y), y.z * sig(z.z), y.w * sig(z.w));
            }
            store4(a.out.p, t * a.out.ld + h * a.out.hs + e, a.type, y);
        } else {
            const size_t rec = (((size_t)slot * NKV + g) * a.n_mt + mt) * 16 + r;
            *reinterpret_cast<f32x4 *>(a.part + rec * HD + e) = o;
            if (e == 0) a.ml[rec] = make_float2(m, l);
        }
    }
}

// A row that sees more than one chunk: out = sum c_i O_i / sum c_i l_i with
// c_i = exp2(ref_i - max ref).  One workgroup per (token, q head); wave w takes
// every fourth chunk.
__global__ __launch_bounds__(256) void kv4_merge_kernel(Attn a) {
    __shared__ float red[2][4];
    __shared__ __attribute__((aligned(16))) float comb[4][256];
    const uint32_t t = blockIdx.x / a.nq, h = blockIdx.x % a.nq, lane = threadIdx.x & 63u, HD = a.b.hd;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int seq = seq_of(a.b, t);
    if (seq < 0) return;
    const Work wk = find_work(a, (uint32_t)seq, true, false);
    if (wk.seq < 0) return;
    const uint32_t i = t - (uint32_t)wk.tok0, span = wk.ct * TILE;
    const int cap = (int)min((uint64_t)a.max_kv, (uint64_t)a.b.max_pages << a.page_shift);
    const int pos = min(wk.len - wk.n_new + (int)i, cap - 1);
    if (i >= (uint32_t)wk.n_new || i >= a.max_q || pos < (int)span) return;
    const uint32_t n = (uint32_t)pos / span + 1u;   // chunks the row sees
    const uint32_t g = h / a.gqa, r = i * a.gqa + h % a.gqa;
    auto rec = [&](uint32_t c) { return (((size_t)(wk.first + c) * a.b.nkv + g) * a.n_mt + r / 16) * 16 + r % 16; };
    float m = REF_NONE, l = 0.0f;
    for (uint32_t c = lane; c < n; c += 64) m = fmaxf(m, a.ml[rec(c)].x);
    m = wave_max_f32(m);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t e = 4 * lane;
    for (uint32_t c0 = w; c0 < n; c0 += 32) {
        f32x4 x[8];
        float2 ml[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            const size_t at = rec(min(c0 + 4 * k, n - 1u));
            ml[k] = a.ml[at];
            x[k] = *reinterpret_cast<const f32x4 *>(a.part + at * HD + (e < HD ? e : 0u));
        }
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
            if (c0 + 4 * k >= n) break;
            const float c = __builtin_amdgcn_exp2f(ml[k].x - m);
            l = fmaf(ml[k].y, c, l);
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = fmaf(x[k][j], c, o[j]);
        }
    }
    if (lane == 0) red[0][w] = l;
    *reinterpret_cast<f32x4 *>(&comb[w][e]) = o;
    __syncthreads();
    if (w != 0 || e >= HD) return;
    l = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
#pragma unroll
    for (uint32_t k = 1; k < 4; k++) o = o + *reinterpret_cast<const f32x4 *>(&comb[k][e]);
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    float4 y = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    if (a.gate.p) {
        const float4 z = load4(a.gate.p, (int64_t)t * a.gate.ld + (int64_t)h * a.gate.hs + e, a.type);
        auto sig = [](float x) { return 1.0f / (1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f)); };
        y = make_float4(y.x * sig(z.x), y.y * sig(z.y), y.z * sig(z.z), y.w * sig(z.w));
    }
    store4(a.out.p, (int64_t)t * a.out.ld + (int64_t)h * a.out.hs + e, a.type, y);
}

// ------------------------------------------------------------------ host side

bool type_ok(int t) { return t == SINTER_F32 || t == SINTER_F16 || t == SINTER_BF16; }
int elem_bytes(int t) { return t == SINTER_F32 ? 4 : 2; }

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
    return SINTER_OK;
}

// The launch of a batch: row tiles a sequence and chunk slots.  A slot a
// sequence, and where there may be rows to split as many more as give every CU
// two workgroups.
struct Plan {
    uint32_t n_mt, n_slots;
    bool merge;
    uint64_t grid;
    size_t recs;
};
Plan make_plan(const sinter_kv4_batch &b, const sinter_kv4_attn_args &a) {
    Plan p;
    const uint64_t rows = (uint64_t)std::min(a.max_q, b.n_tok) * (a.nq / b.nkv);
    p.n_mt = (uint32_t)((rows + 15) / 16);
    p.merge = a.max_kv > CT_MIN * TILE;
    p.n_slots = b.n_seq;
    if (p.merge) {
        const uint64_t per = (uint64_t)b.nkv * p.n_mt;
        const uint64_t most = (uint64_t)b.n_seq * ((a.max_kv + CT_MIN * TILE - 1) / (CT_MIN * TILE));
        p.n_slots += (uint32_t)std::min<uint64_t>(std::max<uint64_t>(1, 1024 / per), most);
    }
    p.grid = (uint64_t)p.n_slots * b.nkv * p.n_mt;
    p.recs = p.merge ? (size_t)p.grid * 16 : 0;
    return p;
}

template <int HD>
void launch_split(const Attn &k, uint32_t grid, hipStream_t s) {
    if (k.type == SINTER_F32) hipLaunchKernelGGL((kv4_split_kernel<HD, 2>), dim3(grid), dim3(256), 0, s, k);
    else hipLaunchKernelGGL((kv4_split_kernel<HD, 1>), dim3(grid), dim3(256), 0, s, k);
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
    p.nq = nq; p.heads = nq + nk; p.half = a->rope_dims / 2; p.type = a->type; p.eps = a->eps;
    p.rate = p.half ? std::log2((double)a->rope_base) / p.half : 0.0;
    // few tokens: a wave a head group; many: a workgroup a token
    const uint32_t per = 4 * (256 / b->hd), need = (p.heads + per - 1) / per;
    const uint32_t y = b->n_tok >= 1024 ? 1u : need;
    hipLaunchKernelGGL(kv4_prep_kernel, dim3(b->n_tok, y), dim3(256), 0, (hipStream_t)stream, p);
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
    r.b = *b; r.k = *k; r.v = *v; r.type = (uint32_t)type;
    r.per = (2 * b->nkv * (b->hd / 32) + 31) / 32;
    const uint64_t grid = (uint64_t)b->n_tok * r.per;
    if (grid > (uint64_t)INT32_MAX) return set_error(SINTER_ERR_ARG, "kv4_append: too many tokens");
    hipLaunchKernelGGL(kv4_append_kernel, dim3((uint32_t)grid), dim3(256), 0, (hipStream_t)stream, r);
    return hip_ok(hipGetLastError(), "kv4_append: launch") ? SINTER_OK : SINTER_ERR_HIP;
}

int sinter_kv4_read(const sinter_kv4_batch *b, const sinter_heads *k, const sinter_heads *v, int type, void *stream) {
    const int rc = check_batch(b, "kv4_read", true);
    if (rc != SINTER_OK) return rc;
    if (!type_ok(type)) return set_error(SINTER_ERR_ARG, "kv4_read: type %d (F32, F16 or BF16)", type);
    if (b->n_seq == 0 || b->n_tok == 0) return SINTER_OK;
    Rows r;
    r.b = *b; r.type = (uint32_t)type;
    r.k = k ? *k : sinter_heads{}; r.v = v ? *v : sinter_heads{};
    if (!r.k.p && !r.v.p) return set_error(SINTER_ERR_ARG, "kv4_read: nowhere to write");
    const char *why;
    if ((r.k.p && (why = check_heads(r.k, b->n_tok, b->nkv, b->hd, type))) || (r.v.p && (why = check_heads(r.v, b->n_tok, b->nkv, b->hd, type))))
        return set_error(SINTER_ERR_ARG, "kv4_read: %s", why);
    r.per = (2 * b->nkv * (b->hd / 16) + 255) / 256;
    const uint64_t grid = (uint64_t)b->n_tok * r.per;
    if (grid > (uint64_t)INT32_MAX) return set_error(SINTER_ERR_ARG, "kv4_read: too many tokens");
    hipLaunchKernelGGL(kv4_read_kernel, dim3((uint32_t)grid), dim3(256), 0, (hipStream_t)stream, r);
    return hip_ok(hipGetLastError(), "kv4_read: launch") ? SINTER_OK : SINTER_ERR_HIP;
}

size_t sinter_kv4_attn_ws_bytes(const sinter_kv4_batch *b, const sinter_kv4_attn_args *a) {
    if (check_attn(b, a) != SINTER_OK || b->n_seq == 0 || b->n_tok == 0) return 0;
    return make_plan(*b, *a).recs * ((size_t)b->hd * 4 + 8);
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
    const size_t need = p.recs * ((size_t)b->hd * 4 + 8);
    if (need && (!a->ws || (uintptr_t)a->ws % 16u || a->ws_bytes < need))
        return set_error(SINTER_ERR_ARG, "kv4_attn: workspace of %zu bytes, 16-byte aligned (sinter_kv4_attn_ws_bytes)", need);
    if (p.grid > (uint64_t)INT32_MAX || (uint64_t)b->n_tok * a->nq > (uint64_t)INT32_MAX)
        return set_error(SINTER_ERR_ARG, "kv4_attn: batch too large");
    Attn k;
    k.b = *b;
    k.q = a->q; k.gate = a->gate; k.out = a->out;
    k.part = static_cast<float *>(a->ws);
    k.ml = reinterpret_cast<float2 *>(k.part + p.recs * b->hd);
    k.nq = a->nq; k.gqa = a->nq / b->nkv; k.max_q = a->max_q; k.max_kv = a->max_kv;
    k.n_slots = p.n_slots; k.n_mt = p.n_mt; k.type = a->type;
    k.page_shift = (uint32_t)__builtin_ctz(b->page_rows);
    k.qscale = a->scale * 1.44269504088896341f;
    const hipStream_t s = (hipStream_t)stream;
    if (b->hd == 256) launch_split<256>(k, (uint32_t)p.grid, s);
    else if (b->hd == 128) launch_split<128>(k, (uint32_t)p.grid, s);
    else launch_split<64>(k, (uint32_t)p.grid, s);
    if (!hip_ok(hipGetLastError(), "kv4_attn: launch")) return SINTER_ERR_HIP;
    if (p.merge) hipLaunchKernelGGL(kv4_merge_kernel, dim3(b->n_tok * a->nq), dim3(256), 0, s, k);
    return hip_ok(hipGetLastError(), "kv4_attn: merge launch") ? SINTER_OK : SINTER_ERR_HIP;
}

}  // extern "C"
