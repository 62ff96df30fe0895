// 4-bit KV cache: its layout, and the streaming attention kernel that reads it (sm_100a).
//
// Every (token, KV head) row of K and of V is stored as D codes c in 0..15 with a scale s and an
// offset lo of its own, both in the model's 16-bit type; the row's values are lo + s * c.  A cache
// is a byte array [pages][kv_heads][page_size / 16] of tiles, one tile = 16 tokens of one KV head:
//
//   [K codes 8D bytes][V codes 8D bytes][K (s, lo) of token 0..15: 64 bytes][V (s, lo): 64 bytes]
//
// so that one untiled bulk copy of 16 D + 128 bytes (a multiple of 128) brings a tile, and a lane's
// operands of mma.m16n8k16 are whole 32-bit words of it - no ldmatrix, no transposition:
//
//   K: token t, 32-bit word w = 0 .. D/8 - 1 holds dims 8w .. 8w + 7; nibble j of the low half is
//      dim 8w + 2j, nibble j of the high half dim 8w + 2j + 1;
//   V: lane (g, c) = 4g + c owns dims (D/8) g .. (D/8) g + D/8 - 1 of the tokens 2c, 2c + 1 (first 4D
//      bytes) and 2c + 8, 2c + 9 (second 4D bytes), D/32 words each; word w: low half the even token,
//      high half the odd one, nibble j is dim (D/8) g + 8 (w / 2) + w % 2 + 2j.  A token owns whole
//      16-bit halves, so appending one token never rewrites another's bits.
#pragma once

#include "pat_kernels.cuh"

namespace pat {

template <int D> struct Int4Tile {
    static constexpr int kCodes = 8 * D;                  // bytes of one operand's codes
    static constexpr int kVOff = kCodes;
    static constexpr int kKPrm = 2 * kCodes;
    static constexpr int kVPrm = kKPrm + 64;
    static constexpr int kBytes = kVPrm + 64;
    static constexpr int kTokenBytes = D / 2;             // K codes of one token
    static constexpr int kLaneBytes = D / 8;              // V codes of one lane and token pair
};

// A pair of codes as a pair of 16-bit floats 16 + c: the nibble is moved to the mantissa bits that
// count ones when the exponent says 16 (bits 3-6 of bf16, bits 6-9 of fp16).  Exact, one shift and
// one logic instruction per pair; the constant 16 is taken out of the sums in fp32.
template <typename T> struct Int4Elt;
template <uint32_t kMask> __device__ __forceinline__ uint32_t mask_or(uint32_t v, uint32_t bits) {       // (v & kMask) | bits
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "n"(kMask), "r"(bits));
    return r;
}
template <> struct Int4Elt<__nv_bfloat16> {
    static constexpr bool kIsHalf = false;
    static constexpr uint32_t kSixteen = 0x41804180u;     // (16, 16)
    template <int J> __device__ static __forceinline__ uint32_t pair(uint32_t w) {
        const uint32_t x = J == 0 ? w << 3 : w >> (4 * J - 3);
        return mask_or<0x00780078u>(x, kSixteen);
    }
    __device__ static __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
};
template <> struct Int4Elt<__half> {
    static constexpr bool kIsHalf = true;
    static constexpr uint32_t kSixteen = 0x4C004C00u;
    template <int J> __device__ static __forceinline__ uint32_t pair(uint32_t w) {
        const uint32_t x = J < 2 ? w << (6 - 4 * J) : w >> (4 * J - 6);
        return mask_or<0x03C003C0u>(x, kSixteen);
    }
    __device__ static __forceinline__ float2 unpack(uint32_t v) {
        return __half22float2(*reinterpret_cast<const __half2*>(&v));
    }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// 8 x 8 matrix of 16-bit elements, lane l holding row l / 4, columns 2 (l % 4) and + 1, transposed
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <int N> __device__ __forceinline__ void lds_words(uint32_t (&w)[N], const unsigned char* p) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    }
}

struct Int4Cache {
    const unsigned char* base;
    int64_t page_stride, head_stride;      // bytes
    uint32_t sixty_four;                   // 64 (see Codes16)
};

// A warp works off one unit - a streaming item's rows (8 or fewer) of one KV head - by itself: no barrier, nothing to
// combine.  (Four warps sharing a unit, with the sums joined through shared memory, spent more instructions on the way in
// and out than on the tokens of a short unit.)
//
// Measured on a B200, 8 KV heads of 128 elements: 0.84 M tokens in 538 items 189 us = 4.9 TB/s of codes, 0.74 of the copy
// bandwidth; 512 items of 288 tokens 47.5 us; a batch of 6.9 K tokens 8.3 us.  Instructions bound it: the issue slots are
// busy 63 % of the time (the 16-bit kernel: 27 %), the half-rate integer pipe that takes the codes apart is its
// fullest one, tensor pipe 30 %, DRAM 58 %.
constexpr int kInt4Warps = 4;              // units per CTA
constexpr int kInt4Stages = 3;             // stages per warp
constexpr int kInt4Step = 2;               // tiles per stage: 32 tokens

template <int D> constexpr int int4_stream_smem_bytes() {
    return kInt4Warps * kInt4Stages * kInt4Step * Int4Tile<D>::kBytes + 128;
}

// The streaming kernel multiplies in fp16 whatever the model's type.  fp16 has ten mantissa bits, so two of a word's
// nibbles become numbers without being moved: under the exponent of 64 the bits 4-7 count ones (64 + c); bits 0-3 are
// moved to 6-9, under the exponent of 16 (16 + c).  A word costs one shift, four logic instructions (mask and
// exponent in one three-input instruction each) and two multiplications by 64, where bf16 takes four shifts and four
// logic instructions, and P' keeps eleven bits instead of eight.  The integer pipe, at half rate, bounds this kernel: the
// factor 64 is a kernel parameter because a multiplication by a constant would become a shift on that pipe.
struct Codes16 {
    uint32_t p[4];                         // pairs of nibble 0 .. 3: 16 + c, 64 + c, 16 + c, 64 + c
    __device__ __forceinline__ Codes16(uint32_t w, uint32_t sixty_four) {
        const uint32_t w8 = w >> 8;
        p[0] = mask_or<0x03C003C0u>(w * sixty_four, 0x4C004C00u);
        p[1] = mask_or<0x00F000F0u>(w, 0x54005400u);
        p[2] = mask_or<0x03C003C0u>(w8 * sixty_four, 0x4C004C00u);
        p[3] = mask_or<0x00F000F0u>(w8, 0x54005400u);
    }
};
constexpr float kInt4NormStart = 1.329227995784916e36f;     // 2^120: any scale but the tiniest exceeds 1 / this

// What one warp carries through its tokens: 8 query rows against 16-token tiles, operands
// swapped (S^T = K Q^T, O^T = V^T P^T): the tokens are the 16 rows of the first product, so that a
// single request's query heads (8 or fewer) fill a product's 8 columns.  A thread (g, c) = (lane / 4, lane % 4) owns
// the columns (query rows) 2c and 2c + 1 of every accumulator.
//
// Scores are kept in units of `unit` = scale * log2 e * 2^e, where 2^e scales the row of Q to below 2 (exact; a bf16
// row does not fit fp16 otherwise).
template <int D> struct Int4State {
    uint2 q[D / 16];           // B fragments of Q^T, k-step ks: dims (D/4) c + 4 ks .. + 3 of row g
    float qsum[2];             // sum of the row's elements
    float qoff[2];             // - sum of 16 or 64 times the element: what the products' constants add up to
    float unit[2];
    float o[D / 16][4];        // O^T: [0],[1] dim (D/8) g + 2i of rows 2c, 2c + 1; [2],[3] dim + 1
    float off[4];              // sum of the rounded P' since int4_settle ([2], [3] repeat [0], [1])
    float omid[2];             // sum of p * (lo + 7.5 s) over the thread's tokens
    float l[2];                // sum of p over the thread's tokens
    float m[2];                // reference maximum, -inf before the first visible score
    float base[2];             // m * unit, or 0 while m = -inf
    float limit[2];            // m + 8 / unit
    float vnorm;
};

// One step: 32 tokens (two tiles) in shared memory, `valid` of them inside the item.
// lim: tokens of the step that the thread's two columns may see (only with kLimits).
//
// With codes c and rows' (s, lo):  s_t (q . c_t) + lo_t sum(q) is the score, and
// sum_t p_t v_t = sum_t (p_t s_t) (c_t - 7.5) + sum_t p_t (lo_t + 7.5 s_t) the output, so the products run
// on the exact codes; only P' = p s is rounded, to fp16.  (About 7.5 because that rounding error is multiplied by
// what stands beside P': with the codes as they are, 0..15, it would be 2.8 times that of a zero-mean V.)
// fp16 has too few exponents for p * s of any s: s is taken relative to 1 / `vnorm`, a power of two near the
// largest scale seen.
template <typename T, int D, bool kLimits>
__device__ __forceinline__ void int4_attend_step(Int4State<D>& st, const unsigned char* stage, int valid, int lim0, int lim1, uint32_t k64,
                                                 int lane) {
    using E = Int4Elt<T>;
    using H = Elt<__half>;
    using L = Int4Tile<D>;
    constexpr int W4 = D / 32, U = kInt4Step;      // words per lane chunk
    const int g = lane >> 2, c = lane & 3;
    float x[U][4];
    float vs[U][2], vmid[U][2];                    // scale, middle of the range
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned char* tile = stage + u * L::kBytes;
        uint32_t k0[W4], k1[W4];
        lds_words(k0, tile + g * L::kTokenBytes + c * (D / 8));
        lds_words(k1, tile + (g + 8) * L::kTokenBytes + c * (D / 8));
        x[u][0] = x[u][2] = st.qoff[0];
        x[u][1] = x[u][3] = st.qoff[1];
#pragma unroll
        for (int w = 0; w < W4; ++w) {
            const Codes16 f0(k0[w], k64), f1(k1[w], k64);
            const uint32_t a[4] = {f0.p[0], f1.p[0], f0.p[1], f1.p[1]};
            const uint32_t b[4] = {f0.p[2], f1.p[2], f0.p[3], f1.p[3]};
            H::mma(x[u], a, st.q[2 * w].x, st.q[2 * w].y);
            H::mma(x[u], b, st.q[2 * w + 1].x, st.q[2 * w + 1].y);
        }
        const float2 kp0 = E::unpack(*reinterpret_cast<const uint32_t*>(tile + L::kKPrm + g * 4));
        const float2 kp1 = E::unpack(*reinterpret_cast<const uint32_t*>(tile + L::kKPrm + (g + 8) * 4));
        const float2 vp0 = E::unpack(*reinterpret_cast<const uint32_t*>(tile + L::kVPrm + g * 4));
        const float2 vp1 = E::unpack(*reinterpret_cast<const uint32_t*>(tile + L::kVPrm + (g + 8) * 4));
        vs[u][0] = vp0.x; vmid[u][0] = fmaf(7.5f, vp0.x, vp0.y);
        vs[u][1] = vp1.x; vmid[u][1] = fmaf(7.5f, vp1.x, vp1.y);
        x[u][0] = fmaf(x[u][0], kp0.x, kp0.y * st.qsum[0]);
        x[u][1] = fmaf(x[u][1], kp0.x, kp0.y * st.qsum[1]);
        x[u][2] = fmaf(x[u][2], kp1.x, kp1.y * st.qsum[0]);
        x[u][3] = fmaf(x[u][3], kp1.x, kp1.y * st.qsum[1]);
    }
    if (kLimits || valid < 16 * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // Tokens past the end hold anything, NaN scales included: they must not reach a product.
            const int t0 = u * 16 + g, t1 = t0 + 8;
            if (t0 >= valid) vs[u][0] = vmid[u][0] = 0.f;
            if (t1 >= valid) vs[u][1] = vmid[u][1] = 0.f;
            const int v0 = kLimits ? lim0 : valid, v1 = kLimits ? lim1 : valid;
            if (t0 >= v0) x[u][0] = -INFINITY;
            if (t0 >= v1) x[u][1] = -INFINITY;
            if (t1 >= v0) x[u][2] = -INFINITY;
            if (t1 >= v1) x[u][3] = -INFINITY;
        }
    }
    float mx[2] = {fmaxf(x[0][0], x[0][2]), fmaxf(x[0][1], x[0][3])}, top = fmaxf(vs[0][0], vs[0][1]);
#pragma unroll
    for (int u = 1; u < U; ++u) {
        mx[0] = fmaxf(mx[0], fmaxf(x[u][0], x[u][2]));
        mx[1] = fmaxf(mx[1], fmaxf(x[u][1], x[u][3]));
        top = fmaxf(top, fmaxf(vs[u][0], vs[u][1]));
    }
    // The reference maximum is only raised when a score exceeds it by more than 2^8 (it cancels in
    // O / l), so the shuffles and the rescaling below are rare.  (limit = -inf at the start: the first visible score
    // raises it.)
    if (__any_sync(kFullMask, mx[0] > st.limit[0] || mx[1] > st.limit[1] || top * st.vnorm > 64.f)) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, d));
        top = fminf(top, kInt4NormStart);
        float f = 1.f;
        if (top * st.vnorm > 1.f) {
            // 1 / 2^e with 2^e <= top < 2^(e + 1)
            const float next = __uint_as_float((254u << 23) - (__float_as_uint(top) & 0x7f800000u));
            f = next / st.vnorm;
            st.vnorm = next;
        }
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float y = fmaxf(mx[e], st.m[e]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) y = fmaxf(y, __shfl_xor_sync(kFullMask, y, d));
            alpha[e] = st.m[e] == -INFINITY ? 0.f : fast_exp2((st.m[e] - y) * st.unit[e]);
            st.m[e] = y;
            st.base[e] = y == -INFINITY ? 0.f : y * st.unit[e];
            st.limit[e] = y + 8.f / st.unit[e];
            st.l[e] *= alpha[e];
            st.omid[e] *= alpha[e];
            alpha[e] *= f;
            st.off[e] *= alpha[e];
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            st.o[i][0] *= alpha[0]; st.o[i][1] *= alpha[1];
            st.o[i][2] *= alpha[0]; st.o[i][3] *= alpha[1];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned char* vt = stage + u * L::kBytes + L::kVOff;
        uint32_t v0[W4], v1[W4];
        lds_words(v0, vt + lane * L::kLaneBytes);
        lds_words(v1, vt + 4 * D + lane * L::kLaneBytes);
        const float s0 = vs[u][0] * st.vnorm, s1 = vs[u][1] * st.vnorm;
        // (a column that has seen nothing yet has only -inf scores: exp2(-inf - 0) = 0)
        float p[4], w[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[e] = fast_exp2(fmaf(x[u][e], st.unit[e & 1], -st.base[e & 1]));
            w[e] = p[e] * (e < 2 ? s0 : s1);
            y[e] = e < 2 ? vmid[u][0] : vmid[u][1];
            if constexpr (kLimits) {    // a token that one row sees and another does not may hold NaN
                if (x[u][e] == -INFINITY) w[e] = y[e] = 0.f;
            }
        }
        st.l[0] += p[0] + p[2];
        st.l[1] += p[1] + p[3];
        st.omid[0] = fmaf(p[2], y[2], fmaf(p[0], y[0], st.omid[0]));
        st.omid[1] = fmaf(p[3], y[3], fmaf(p[1], y[1], st.omid[1]));
        const uint32_t pb0 = transpose8x8(H::pack(w[0], w[1])), pb1 = transpose8x8(H::pack(w[2], w[3]));
        const uint32_t ones[4] = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
        H::mma(st.off, ones, pb0, pb1);
#pragma unroll
        for (int wp = 0; wp < D / 64; ++wp) {
            const Codes16 a0(v0[2 * wp], k64), a1(v0[2 * wp + 1], k64), a2(v1[2 * wp], k64), a3(v1[2 * wp + 1], k64);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t f[4] = {a0.p[j], a1.p[j], a2.p[j], a3.p[j]};
                H::mma(st.o[4 * wp + j], f, pb0, pb1);
            }
        }
    }
}

// Takes out of the sums what the codes stand above c - 7.5.  Carried along to a long unit's end it would outgrow the sums
// that it stands in (the output is then the small mean of large terms of either sign): 0.5 % of the output's norm over
// 2048 tokens, against 0.02 % when it is done every 128.  In every tile it cost 2.6 us of 47 and 15 of 185 (a
// deep tree, long contexts).
constexpr int kInt4Settle = 4;             // steps
template <int D> __device__ __forceinline__ void int4_settle(Int4State<D>& st) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const float above = i & 1 ? -71.5f : -23.5f;          // i % 4 is the nibble
        st.o[i][0] = fmaf(above, st.off[0], st.o[i][0]); st.o[i][1] = fmaf(above, st.off[1], st.o[i][1]);
        st.o[i][2] = fmaf(above, st.off[0], st.o[i][2]); st.o[i][3] = fmaf(above, st.off[1], st.o[i][3]);
    }
    st.off[0] = st.off[1] = st.off[2] = st.off[3] = 0.f;
}

// A pair of the model's type, scaled by a power of two, as a pair of fp16.
template <typename T> __device__ __forceinline__ uint32_t to_half_pair(uint32_t v, float scale) {
    if constexpr (Int4Elt<T>::kIsHalf) return v;
    const float2 e = Int4Elt<T>::unpack(v);
    return Elt<__half>::pack(e.x * scale, e.y * scale);
}

// Query rows row0 .. row0 + 7 of a unit into a warp's state.  lim: tokens of the item the thread's columns may see.
template <typename T, int D, bool kLimits>
__device__ __forceinline__ void int4_load_rows(Int4State<D>& st, int (&lim)[2], const AttnParams& p, int q_off, int row0, int rows_valid,
                                               int kvh, int kv_len, int tok_lo, int lane) {
    const int g = lane >> 2, c = lane & 3, row = row0 + g;
    const uint4* src = nullptr;
    if (row < rows_valid) {
        const int qi = row / p.hratio, gg = row - qi * p.hratio;
        src = reinterpret_cast<const uint4*>(q_row_ptr<T>(p, __ldg(p.queries + q_off + qi), kvh * p.hratio + gg)) + c * (D / 32);
    }
    uint4 raw[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) raw[i] = src ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
    // 2^-e for 2^e <= max < 2^(e + 1); rows of zeros, infinities or NaN as they are
    float down = 1.f;
    if constexpr (!Int4Elt<T>::kIsHalf) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 e = Int4Elt<T>::unpack(w[k]);
                top = fmaxf(top, fmaxf(fabsf(e.x), fabsf(e.y)));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
        if (top >= 1.17549435e-38f && top < INFINITY)
            down = __uint_as_float(min(253u << 23, (254u << 23) - (__float_as_uint(top) & 0x7f800000u)));
    }
    float sum = 0.f, off = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const uint32_t w[4] = {to_half_pair<T>(raw[i].x, down), to_half_pair<T>(raw[i].y, down),
                               to_half_pair<T>(raw[i].z, down), to_half_pair<T>(raw[i].w, down)};
        st.q[2 * i] = make_uint2(w[0], w[1]);
        st.q[2 * i + 1] = make_uint2(w[2], w[3]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 e = Int4Elt<__half>::unpack(w[k]);
            const float pair = e.x + e.y;
            sum += pair;
            off = fmaf(k & 1 ? -64.f : -16.f, pair, off);
        }
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
        sum += __shfl_xor_sync(kFullMask, sum, d);
        off += __shfl_xor_sync(kFullMask, off, d);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int from = (2 * c + e) * 4;
        st.qsum[e] = __shfl_sync(kFullMask, sum, from);
        st.qoff[e] = __shfl_sync(kFullMask, off, from);
        st.unit[e] = p.scale_log2 / __shfl_sync(kFullMask, down, from);
        st.m[e] = st.limit[e] = -INFINITY;
        st.base[e] = st.l[e] = st.omid[e] = 0.f;
        lim[e] = kv_len;
        if constexpr (kLimits) {
            const int col = row0 + 2 * c + e;
            lim[e] = col < rows_valid ? visible_tokens(p, q_off + col / p.hratio, tok_lo, kv_len) : 0;
        }
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) st.o[i][0] = st.o[i][1] = st.o[i][2] = st.o[i][3] = 0.f;
    st.off[0] = st.off[1] = st.off[2] = st.off[3] = 0.f;
    st.vnorm = kInt4NormStart;
}

template <typename T, int D, bool kLimits>
__global__ void __launch_bounds__(kInt4Warps * 32, 4) int4_stream_kernel(const AttnParams p, const Int4Cache cache) {
    using L = Int4Tile<D>;
    constexpr int W = kInt4Warps, S = kInt4Stages, U = kInt4Step;
    constexpr int kStage = U * L::kBytes;
    constexpr int kAhead = 32 / U;          // steps whose page ids one load of the warp covers
    static_assert((U & (U - 1)) == 0 && S <= kAhead, "");
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t bars[W * S];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    unsigned char* my_stage = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127)) +
                              warp * S * kStage;
    const uint32_t my_stage_addr = smem_u32(my_stage), my_bar = smem_u32(bars + warp * S);
    // units: the KV heads of an item next to each other (they touch the same pages)
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * W + warp;
    const int item_idx = static_cast<int>(unit / p.kv_heads);
    const int kvh = static_cast<int>(unit - static_cast<int64_t>(item_idx) * p.kv_heads);
    if (item_idx >= p.num_items) return;    // (the warps of a CTA never wait for one another)
    if (lane < S) {
        mbar_init(my_bar + lane * 8, 1);
        mbar_fence_init();
    }
    __syncwarp();
    const int4* it = reinterpret_cast<const int4*>(p.items + static_cast<size_t>(item_idx) * 8);
    const int4 ra = __ldg(it), rb = __ldg(it + 1);            // {q_off, nq, page_off, kv_len}, {entry_base, kv_head, cost, tok_lo}
    const int q_off = ra.x, rows_valid = ra.y * p.hratio, kv_len = ra.w;
    const int n_tiles = (kv_len + 15) >> 4, n_steps = (n_tiles + U - 1) / U;
    const int tiles_per_page = p.page_size >> 4;
    const int32_t* item_pages = p.pages + ra.z;
    const unsigned char* head_base = cache.base + kvh * cache.head_stride;
    int issued = 0;                         // steps requested since the start (ring position and parity go by it)

    // Lane l holds the place of tile l % U of step first + l / U in the cache.
    int64_t ahead = 0;
    auto fetch = [&](int first) {
        const int t = first * U + lane;
        if (t >= n_tiles) return;
        const int at = t / tiles_per_page;
        ahead = __ldg(item_pages + at) * cache.page_stride + (t - at * tiles_per_page) * L::kBytes;
    };
    auto issue = [&](int j) {
        const int s = issued % S, tiles = min(U, n_tiles - j * U);
        const int64_t off = __shfl_sync(kFullMask, ahead, (j % kAhead) * U + (lane & (U - 1)));
        if (lane == 0) mbar_expect_tx(my_bar + s * 8, tiles * L::kBytes);
        __syncwarp();
        if (lane < tiles) bulk_load(my_stage_addr + s * kStage + lane * L::kBytes, head_base + off, L::kBytes, my_bar + s * 8);
        ++issued;
    };

    int s = 0;
    uint32_t phase = 0;
    // (lists made for this kernel have 8 rows or fewer per item; any list is worked off in groups of 8)
    for (int row0 = 0; row0 < rows_valid; row0 += 8) {
        fetch(0);
        for (int j = 0; j < min(S, n_steps); ++j) issue(j);
        Int4State<D> st;
        int lim[2];
        int4_load_rows<T, D, kLimits>(st, lim, p, q_off, row0, rows_valid, kvh, kv_len, rb.w, lane);
        for (int j = 0; j < n_steps; ++j) {
            if (!__all_sync(kFullMask, mbar_wait(my_bar + s * 8, phase, p.wait_ns))) {
                // Give up: nothing more is requested; what is in flight gets a short second wait so that
                // none of it lands after the CTA has gone.
                for (int k = 0; k < min(S, n_steps - j); ++k) {
                    mbar_wait(my_bar + s * 8, phase, kDrainWaitNs);
                    if (++s == S) { s = 0; phase ^= 1; }
                }
                if (lane == 0 && p.status) atomicExch(p.status, 1);
                return;
            }
            int4_attend_step<T, D, kLimits>(st, my_stage + s * kStage, kv_len - j * 16 * U, lim[0] - j * 16 * U, lim[1] - j * 16 * U,
                                            cache.sixty_four, lane);
            if (j % kInt4Settle == kInt4Settle - 1 || j + 1 == n_steps) int4_settle(st);
            __syncwarp();
            if ((j + S) % kAhead == 0) fetch(j + S);
            if (j + S < n_steps) issue(j + S);
            if (++s == S) { s = 0; phase ^= 1; }
        }
        // true output = o / vnorm + omid, over l
        const float back = 1.f / st.vnorm;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = st.l[e], omid = st.omid[e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l += __shfl_xor_sync(kFullMask, l, d);
                omid += __shfl_xor_sync(kFullMask, omid, d);
            }
            const int row = row0 + 2 * c + e;
            if (row >= rows_valid) continue;
            // a row that sees none of the item's tokens has weight -inf; a NaN in the cache stays a NaN
            const bool none = st.m[e] == -INFINITY && l == 0.f;
            const float inv = none ? 0.f : 1.f / l;
            const float scale = back * inv, add = omid * inv;
            const int qi = row / p.hratio, gg = row - qi * p.hratio;
            const size_t slot = (static_cast<size_t>(rb.x) + static_cast<size_t>(qi) * p.kv_heads + kvh) * p.hratio + gg;
            float4* dst = reinterpret_cast<float4*>(p.part_o + slot * D + g * (D / 8));
#pragma unroll
            for (int i = 0; i < D / 16; i += 2)
                dst[i / 2] = make_float4(fmaf(st.o[i][e], scale, add), fmaf(st.o[i][2 + e], scale, add),
                                         fmaf(st.o[i + 1][e], scale, add), fmaf(st.o[i + 1][2 + e], scale, add));
            if (g == 0) p.part_lse[slot] = none ? -INFINITY : st.m[e] * st.unit[e] * 0.6931471805599453f + logf(l);
        }
    }
}

}  // namespace pat
