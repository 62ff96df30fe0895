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
template <> struct Int4Elt<__nv_bfloat16> {
    static constexpr bool kNarrowRange = false;
    static constexpr uint32_t kSixteen = 0x41804180u;     // (16, 16)
    static constexpr uint32_t kCentre = 0x41BC41BCu;      // (23.5, 23.5): the middle of 16 + c
    template <int J> __device__ static __forceinline__ uint32_t pair(uint32_t w) {
        const uint32_t x = J == 0 ? w << 3 : w >> (4 * J - 3);
        return (x & 0x00780078u) | kSixteen;
    }
    __device__ static __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
};
template <> struct Int4Elt<__half> {
    static constexpr bool kNarrowRange = true;
    static constexpr uint32_t kSixteen = 0x4C004C00u;
    static constexpr uint32_t kCentre = 0x4DE04DE0u;
    template <int J> __device__ static __forceinline__ uint32_t pair(uint32_t w) {
        const uint32_t x = J < 2 ? w << (6 - 4 * J) : w >> (4 * J - 6);
        return (x & 0x03C003C0u) | kSixteen;
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
};

constexpr int kInt4Warps = 4;
constexpr float kInt4NormStart = 1152921504606846976.f;     // 2^60: any scale but 0 exceeds 1 / this
constexpr int kInt4Stages = 3;             // stages per warp
constexpr int kInt4Step = 2;               // tiles per stage: 32 tokens

template <int D> constexpr int int4_stream_smem_bytes() {
    return kInt4Warps * kInt4Stages * kInt4Step * Int4Tile<D>::kBytes + 128;
}

// What one warp carries through its tokens: 8 * NT query rows against 16-token tiles, operands
// swapped (S^T = K Q^T, O^T = V^T P^T): the tokens are the 16 rows of the first product, so that a
// single request's query heads (8 or fewer) fill a product's 8 columns, and an unpacked code word
// serves every group of 8 rows.  A thread (g, c) = (lane / 4, lane % 4) owns the columns (query rows)
// 2c and 2c + 1 of every accumulator.
template <int D, int NT> struct Int4State {
    // B fragments of Q^T, k-step ks: dims (D/4) c + 4 ks .. + 3 of row g.  With 16 rows the registers do
    // not hold them: they are read from shared memory (kQShared), one load per k-step and step of 32 tokens.
    static constexpr bool kQShared = NT > 1;
    uint2 q[kQShared ? 1 : NT][kQShared ? 1 : D / 16];
    const uint2* q_shared;         // [NT][D / 16][32 lanes]
    float qsum[NT][2];             // sum of the row's elements, times scale * log2 e
    float o[NT][D / 16][4];        // O^T: [0],[1] dim (D/8) g + 2i of rows 2c, 2c + 1; [2],[3] dim + 1
    float off[NT][4];              // 23.5 * sum of the rounded P' ([2], [3] repeat [0], [1])
    float omid[NT][2];             // sum of p * (lo + 7.5 s) over the thread's tokens
    float l[NT][2];                // sum of p over the thread's tokens
    float m[NT][2];                // reference maximum, in units of log2
};

// One step: 32 tokens (two tiles) in shared memory, `valid` of them inside the item.
// lim: tokens of the step that the thread's two columns may see (only with kLimits).
//
// With codes c and rows' (s, lo):  s_t (q . c_t) + lo_t sum(q) is the score, and
// sum_t p_t v_t = sum_t (p_t s_t) (c_t - 7.5) + sum_t p_t (lo_t + 7.5 s_t) the output, so the products run
// on the exact codes; only P' = p s is rounded, to the model's type, like P in the 16-bit kernels.  (About
// 7.5 because that rounding error is multiplied by what stands beside P': with the codes as they are, 0..15,
// it would be 2.8 times that of a zero-mean V.)
// fp16 has too few exponents for p * s of any s: s is taken relative to 2^(-log2 of `vnorm`), a power
// of two near the largest scale seen.
template <typename T, int D, int NT, bool kLimits>
__device__ __forceinline__ void int4_attend_step(Int4State<D, NT>& st, const unsigned char* stage, int valid,
                                                 const int (&lim)[NT][2], float scale_log2, float& vnorm, int lane) {
    using E = Int4Elt<T>;
    using L = Int4Tile<D>;
    constexpr int W4 = D / 32;                 // words per lane chunk
    const int g = lane >> 2, c = lane & 3;
    float x[kInt4Step][NT][4];
    float vs[kInt4Step][2], vmid[kInt4Step][2];      // scale, middle of the range
    bool raise = false;
    float acc[kInt4Step][NT][4];
    {
        uint32_t k0[kInt4Step][W4], k1[kInt4Step][W4];
#pragma unroll
        for (int u = 0; u < kInt4Step; ++u) {
            const unsigned char* tile = stage + u * L::kBytes;
            lds_words(k0[u], tile + g * L::kTokenBytes + c * (D / 8));
            lds_words(k1[u], tile + (g + 8) * L::kTokenBytes + c * (D / 8));
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[u][n][0] = acc[u][n][1] = acc[u][n][2] = acc[u][n][3] = 0.f;
        }
#pragma unroll
        for (int w = 0; w < W4; ++w) {
            uint2 qa[NT], qb[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if constexpr (Int4State<D, NT>::kQShared) {
                    qa[n] = st.q_shared[(n * (D / 16) + 2 * w) * 32 + lane];
                    qb[n] = st.q_shared[(n * (D / 16) + 2 * w + 1) * 32 + lane];
                } else {
                    qa[n] = st.q[n][2 * w];
                    qb[n] = st.q[n][2 * w + 1];
                }
            }
#pragma unroll
            for (int u = 0; u < kInt4Step; ++u) {
                const uint32_t a[4] = {E::template pair<0>(k0[u][w]), E::template pair<0>(k1[u][w]),
                                       E::template pair<1>(k0[u][w]), E::template pair<1>(k1[u][w])};
                const uint32_t b[4] = {E::template pair<2>(k0[u][w]), E::template pair<2>(k1[u][w]),
                                       E::template pair<3>(k0[u][w]), E::template pair<3>(k1[u][w])};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    Elt<T>::mma(acc[u][n], a, qa[n].x, qa[n].y);
                    Elt<T>::mma(acc[u][n], b, qb[n].x, qb[n].y);
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kInt4Step; ++u) {
        const unsigned char* tile = stage + u * L::kBytes;
        const float2 kp0 = E::unpack(*reinterpret_cast<const uint32_t*>(tile + L::kKPrm + g * 4));
        const float2 kp1 = E::unpack(*reinterpret_cast<const uint32_t*>(tile + L::kKPrm + (g + 8) * 4));
        const float2 vp0 = E::unpack(*reinterpret_cast<const uint32_t*>(tile + L::kVPrm + g * 4));
        const float2 vp1 = E::unpack(*reinterpret_cast<const uint32_t*>(tile + L::kVPrm + (g + 8) * 4));
        vs[u][0] = vp0.x; vmid[u][0] = fmaf(7.5f, vp0.x, vp0.y);
        vs[u][1] = vp1.x; vmid[u][1] = fmaf(7.5f, vp1.x, vp1.y);
        const float b0 = kp0.y - 16.f * kp0.x, b1 = kp1.y - 16.f * kp1.x;
        const float s0 = kp0.x * scale_log2, s1 = kp1.x * scale_log2;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            x[u][n][0] = fmaf(acc[u][n][0], s0, b0 * st.qsum[n][0]);
            x[u][n][1] = fmaf(acc[u][n][1], s0, b0 * st.qsum[n][1]);
            x[u][n][2] = fmaf(acc[u][n][2], s1, b1 * st.qsum[n][0]);
            x[u][n][3] = fmaf(acc[u][n][3], s1, b1 * st.qsum[n][1]);
        }
        if (kLimits || valid < 16 * kInt4Step) {
            // Tokens past the end hold anything, NaN scales included: they must not reach a product.
            const int t0 = u * 16 + g, t1 = t0 + 8;
            if (t0 >= valid) vs[u][0] = vmid[u][0] = 0.f;
            if (t1 >= valid) vs[u][1] = vmid[u][1] = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int v0 = kLimits ? lim[n][0] : valid, v1 = kLimits ? lim[n][1] : valid;
                if (t0 >= v0) x[u][n][0] = -INFINITY;
                if (t0 >= v1) x[u][n][1] = -INFINITY;
                if (t1 >= v0) x[u][n][2] = -INFINITY;
                if (t1 >= v1) x[u][n][3] = -INFINITY;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            // m = -inf at the start: the first visible score raises it
            raise = raise || fmaxf(x[u][n][0], x[u][n][2]) > st.m[n][0] + 8.f || fmaxf(x[u][n][1], x[u][n][3]) > st.m[n][1] + 8.f;
        }
        if constexpr (E::kNarrowRange) raise = raise || fmaxf(vs[u][0], vs[u][1]) * vnorm > 64.f;
    }
    // The reference maximum is only raised when a score exceeds it by more than 2^8 (it cancels in
    // O / l), so the shuffles and the rescaling below are rare.
    if (__any_sync(kFullMask, raise)) {
        if constexpr (E::kNarrowRange) {
            float top = 0.f;
#pragma unroll
            for (int u = 0; u < kInt4Step; ++u) top = fmaxf(top, fmaxf(vs[u][0], vs[u][1]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, d));
            top = fminf(top, 65504.f);
            if (top * vnorm > 1.f) {
                // 1 / 2^e with 2^e <= top < 2^(e + 1)
                const float next = __uint_as_float((254u << 23) - (__float_as_uint(top) & 0x7f800000u));
                const float f = next / vnorm;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) { st.o[n][i][0] *= f; st.o[n][i][1] *= f; st.o[n][i][2] *= f; st.o[n][i][3] *= f; }
                    st.off[n][0] *= f; st.off[n][1] *= f;
                }
                vnorm = next;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float mx0 = st.m[n][0], mx1 = st.m[n][1];
#pragma unroll
            for (int u = 0; u < kInt4Step; ++u) {
                mx0 = fmaxf(mx0, fmaxf(x[u][n][0], x[u][n][2]));
                mx1 = fmaxf(mx1, fmaxf(x[u][n][1], x[u][n][3]));
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                mx0 = fmaxf(mx0, __shfl_xor_sync(kFullMask, mx0, d));
                mx1 = fmaxf(mx1, __shfl_xor_sync(kFullMask, mx1, d));
            }
            const float a0 = st.m[n][0] == -INFINITY ? 0.f : fast_exp2(st.m[n][0] - mx0);
            const float a1 = st.m[n][1] == -INFINITY ? 0.f : fast_exp2(st.m[n][1] - mx1);
            st.m[n][0] = mx0;
            st.m[n][1] = mx1;
            st.l[n][0] *= a0; st.omid[n][0] *= a0; st.off[n][0] *= a0;
            st.l[n][1] *= a1; st.omid[n][1] *= a1; st.off[n][1] *= a1;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                st.o[n][i][0] *= a0; st.o[n][i][1] *= a1;
                st.o[n][i][2] *= a0; st.o[n][i][3] *= a1;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kInt4Step; ++u) {
        const unsigned char* vt = stage + u * L::kBytes + L::kVOff;
        uint32_t v0[W4], v1[W4];
        lds_words(v0, vt + lane * L::kLaneBytes);
        lds_words(v1, vt + 4 * D + lane * L::kLaneBytes);
        const float s0 = E::kNarrowRange ? vs[u][0] * vnorm : vs[u][0], s1 = E::kNarrowRange ? vs[u][1] * vnorm : vs[u][1];
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            // a column that has seen nothing yet has m = -inf and only -inf scores: exp2(-inf - 0) = 0
            const float m0 = st.m[n][0] == -INFINITY ? 0.f : st.m[n][0], m1 = st.m[n][1] == -INFINITY ? 0.f : st.m[n][1];
            const float p0 = fast_exp2(x[u][n][0] - m0), p1 = fast_exp2(x[u][n][1] - m1);
            const float p2 = fast_exp2(x[u][n][2] - m0), p3 = fast_exp2(x[u][n][3] - m1);
            st.l[n][0] += p0 + p2;
            st.l[n][1] += p1 + p3;
            float w0 = p0 * s0, w1 = p1 * s0, w2 = p2 * s1, w3 = p3 * s1;
            float y0 = p0 * vmid[u][0], y1 = p1 * vmid[u][0], y2 = p2 * vmid[u][1], y3 = p3 * vmid[u][1];
            if constexpr (kLimits) {    // a token that one row sees and another does not may hold NaN
                if (x[u][n][0] == -INFINITY) w0 = y0 = 0.f;
                if (x[u][n][1] == -INFINITY) w1 = y1 = 0.f;
                if (x[u][n][2] == -INFINITY) w2 = y2 = 0.f;
                if (x[u][n][3] == -INFINITY) w3 = y3 = 0.f;
            }
            st.omid[n][0] += y0 + y2;
            st.omid[n][1] += y1 + y3;
            pb[n][0] = transpose8x8(Elt<T>::pack(w0, w1));
            pb[n][1] = transpose8x8(Elt<T>::pack(w2, w3));
            const uint32_t mid[4] = {E::kCentre, E::kCentre, E::kCentre, E::kCentre};
            Elt<T>::mma(st.off[n], mid, pb[n][0], pb[n][1]);
        }
#pragma unroll
        for (int wp = 0; wp < D / 64; ++wp) {
            const uint32_t a0 = v0[2 * wp], a1 = v0[2 * wp + 1], a2 = v1[2 * wp], a3 = v1[2 * wp + 1];
            const uint32_t f0[4] = {E::template pair<0>(a0), E::template pair<0>(a1), E::template pair<0>(a2), E::template pair<0>(a3)};
            const uint32_t f1[4] = {E::template pair<1>(a0), E::template pair<1>(a1), E::template pair<1>(a2), E::template pair<1>(a3)};
            const uint32_t f2[4] = {E::template pair<2>(a0), E::template pair<2>(a1), E::template pair<2>(a2), E::template pair<2>(a3)};
            const uint32_t f3[4] = {E::template pair<3>(a0), E::template pair<3>(a1), E::template pair<3>(a2), E::template pair<3>(a3)};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                Elt<T>::mma(st.o[n][4 * wp + 0], f0, pb[n][0], pb[n][1]);
                Elt<T>::mma(st.o[n][4 * wp + 1], f1, pb[n][0], pb[n][1]);
                Elt<T>::mma(st.o[n][4 * wp + 2], f2, pb[n][0], pb[n][1]);
                Elt<T>::mma(st.o[n][4 * wp + 3], f3, pb[n][0], pb[n][1]);
            }
        }
    }
}

// One streaming item (<= 8 * NT query rows of one KV head over one range of tokens) by the CTA's
// four warps, each with a private pipeline over every fourth step of 32 tokens.
template <typename T, int D, int NT, bool kLimits>
__device__ __forceinline__ void int4_stream_item(const AttnParams& p, const Int4Cache& cache, int q_off, int rows_valid,
                                                 int kv_len, int page_off, int entry_base, int tok_lo, int kvh,
                                                 unsigned char* smem, uint64_t* bars, float (*sm_m)[16], float (*sm_l)[16],
                                                 int* sm_abort, uint2* sm_q) {
    using L = Int4Tile<D>;
    constexpr int W = kInt4Warps, S = kInt4Stages, U = kInt4Step;
    constexpr int kStage = U * L::kBytes;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int n_tiles = (kv_len + 15) >> 4;
    const int n_steps = (n_tiles + U - 1) / U;
    const int my_n = warp < n_steps ? (n_steps - warp + W - 1) / W : 0;
    const int tiles_per_page = p.page_size >> 4;
    unsigned char* my_stage = smem + warp * S * kStage;
    const uint32_t my_stage_addr = smem_u32(my_stage);
    const uint32_t my_bar = smem_u32(bars + warp * S);
    const int32_t* item_pages = p.pages + page_off;

    // Lane u < U requests tile u of a step; its page id is fetched one step ahead.
    const unsigned char* head_base = cache.base + kvh * cache.head_stride;
    auto tile_of = [&](int j) { return (warp + j * W) * U + lane; };
    auto fetch_page = [&](int j) -> int {
        const int t = tile_of(j);
        return (lane < U && j < my_n && t < n_tiles) ? __ldg(item_pages + t / tiles_per_page) : 0;
    };
    auto issue = [&](int j, int page) {
        const int s = j % S;
        const uint32_t bar = my_bar + s * 8;
        if (lane == 0) mbar_expect_tx(bar, min(U, n_tiles - (warp + j * W) * U) * L::kBytes);
        __syncwarp();
        const int t = tile_of(j);
        if (lane < U && t < n_tiles)
            bulk_load(my_stage_addr + s * kStage + lane * L::kBytes,
                      head_base + page * cache.page_stride + (t % tiles_per_page) * L::kBytes, L::kBytes, bar);
    };
    for (int j = 0; j < S; ++j) {
        const int page = fetch_page(j);
        if (j < my_n) issue(j, page);
    }
    int page_next = fetch_page(S);

    Int4State<D, NT> st;
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int row = n * 8 + g;
        const uint4* src = nullptr;
        if (row < rows_valid) {
            const int qi = row / p.hratio, gg = row - qi * p.hratio;
            src = reinterpret_cast<const uint4*>(q_row_ptr<T>(p, __ldg(p.queries + q_off + qi), kvh * p.hratio + gg)) + c * (D / 32);
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const uint4 v = src ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
            if constexpr (Int4State<D, NT>::kQShared) {
                if (warp == 0) {
                    sm_q[(n * (D / 16) + 2 * i) * 32 + lane] = make_uint2(v.x, v.y);
                    sm_q[(n * (D / 16) + 2 * i + 1) * 32 + lane] = make_uint2(v.z, v.w);
                }
            } else {
                st.q[n][2 * i] = make_uint2(v.x, v.y);
                st.q[n][2 * i + 1] = make_uint2(v.z, v.w);
            }
            const float2 e0 = Int4Elt<T>::unpack(v.x), e1 = Int4Elt<T>::unpack(v.y), e2 = Int4Elt<T>::unpack(v.z), e3 = Int4Elt<T>::unpack(v.w);
            sum += ((e0.x + e0.y) + (e1.x + e1.y)) + ((e2.x + e2.y) + (e3.x + e3.y));
        }
        sum += __shfl_xor_sync(kFullMask, sum, 1);
        sum += __shfl_xor_sync(kFullMask, sum, 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            st.qsum[n][e] = __shfl_sync(kFullMask, sum, (2 * c + e) * 4) * p.scale_log2;
            st.m[n][e] = -INFINITY;
            st.l[n][e] = st.omid[n][e] = 0.f;
            const int col = n * 8 + 2 * c + e;
            lim[n][e] = kv_len;
            if constexpr (kLimits)
                lim[n][e] = col < rows_valid ? visible_tokens(p, q_off + col / p.hratio, tok_lo, kv_len) : 0;
        }
        st.off[n][0] = st.off[n][1] = st.off[n][2] = st.off[n][3] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) st.o[n][i][0] = st.o[n][i][1] = st.o[n][i][2] = st.o[n][i][3] = 0.f;
    }
    if constexpr (Int4State<D, NT>::kQShared) {
        st.q_shared = sm_q;
        __syncthreads();
    }
    float vnorm = kInt4NormStart;
    bool ok = true;
    for (int j = 0; j < my_n; ++j) {
        const int s = j % S;
        if (!__all_sync(kFullMask, mbar_wait(my_bar + s * 8, (j / S) & 1, p.wait_ns))) {
            // Give up: nothing more is requested; what is in flight gets a short second wait so that
            // none of it lands after the CTA has gone.
            ok = false;
            for (int jj = j; jj < min(j + S, my_n); ++jj) mbar_wait(my_bar + (jj % S) * 8, (jj / S) & 1, kDrainWaitNs);
            break;
        }
        const int first = (warp + j * W) * (16 * U);
        int step_lim[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) { step_lim[n][0] = lim[n][0] - first; step_lim[n][1] = lim[n][1] - first; }
        int4_attend_step<T, D, NT, kLimits>(st, my_stage + s * kStage, kv_len - first, step_lim, p.scale_log2, vnorm, lane);
        __syncwarp();
        if (j + S < my_n) issue(j + S, page_next);
        page_next = fetch_page(j + S + 1);
    }
    if (!ok && lane == 0) { *sm_abort = 1; if (p.status) atomicExch(p.status, 1); }

    // ---- combine the warps' partial states ----------------------------------------
    // true output = (o - off) * 2^k + omid (2^k = 1 / vnorm where the scales were taken relative)
    const float unit = Int4Elt<T>::kNarrowRange ? 1.f / vnorm : 1.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                st.l[n][e] += __shfl_xor_sync(kFullMask, st.l[n][e], d);
                st.omid[n][e] += __shfl_xor_sync(kFullMask, st.omid[n][e], d);
            }
            if (g == 0) {
                sm_m[warp][n * 8 + 2 * c + e] = st.m[n][e];
                sm_l[warp][n * 8 + 2 * c + e] = st.l[n][e];
            }
        }
    __syncthreads();        // every warp is done with its stages
    if (*sm_abort) return;
    constexpr int kRow = D + kScratchPad;
    float* scratch = reinterpret_cast<float*>(smem);        // [W][8 NT][D + pad]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int col = n * 8 + 2 * c + e;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, sm_m[w][col]);
            const float f = st.m[n][e] == -INFINITY ? 0.f : fast_exp2(st.m[n][e] - top);
            float* dst = scratch + (warp * 8 * NT + col) * kRow + g * (D / 8);
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                *reinterpret_cast<float2*>(dst + 2 * i) =
                    make_float2(((st.o[n][i][e] - st.off[n][e]) * unit + st.omid[n][e]) * f,
                                ((st.o[n][i][2 + e] - st.off[n][e]) * unit + st.omid[n][e]) * f);
        }
    __syncthreads();
    constexpr int kVec = D / 4;
    for (int idx = tid; idx < rows_valid * kVec; idx += W * 32) {
        const int row = idx / kVec, v4 = idx - row * kVec;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, sm_m[w][row]);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float mw = sm_m[w][row];
            sum += sm_l[w][row] * (mw == -INFINITY ? 0.f : fast_exp2(mw - top));
            const float4 y = *reinterpret_cast<const float4*>(scratch + (w * 8 * NT + row) * kRow + v4 * 4);
            acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
        }
        // a row that sees none of the item's tokens has weight -inf; a NaN in the cache stays a NaN
        const bool none = top == -INFINITY && sum == 0.f;
        const float inv = none ? 0.f : 1.f / sum;
        const int qi = row / p.hratio, gg = row - qi * p.hratio;
        const size_t slot = (static_cast<size_t>(entry_base) + static_cast<size_t>(qi) * p.kv_heads + kvh) * p.hratio + gg;
        *reinterpret_cast<float4*>(p.part_o + slot * D + v4 * 4) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        if (v4 == 0) p.part_lse[slot] = none ? -INFINITY : top * 0.6931471805599453f + logf(sum);
    }
}

template <typename T, int D, bool kLimits>
__global__ void __launch_bounds__(kInt4Warps * 32, 4) int4_stream_kernel(const AttnParams p, const Int4Cache cache) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
    __shared__ __align__(8) uint64_t bars[kInt4Warps * kInt4Stages];
    __shared__ float sm_m[kInt4Warps][16], sm_l[kInt4Warps][16];
    __shared__ int sm_abort;
    __shared__ uint2 sm_q[2 * (D / 16) * 32];
    const int item_idx = blockIdx.x / p.kv_heads;
    const int kvh = blockIdx.x - item_idx * p.kv_heads;
    const int4* it = reinterpret_cast<const int4*>(p.items + static_cast<size_t>(item_idx) * 8);
    const int4 a = __ldg(it), b = __ldg(it + 1);            // {q_off, nq, page_off, kv_len}, {entry_base, kv_head, cost, tok_lo}
    if (threadIdx.x == 0) {
        sm_abort = 0;
        for (int i = 0; i < kInt4Warps * kInt4Stages; ++i) mbar_init(smem_u32(&bars[i]), 1);
        mbar_fence_init();
    }
    __syncthreads();
    const int rows = a.y * p.hratio;
    if (rows <= 8)
        int4_stream_item<T, D, 1, kLimits>(p, cache, a.x, rows, a.w, a.z, b.x, b.w, kvh, smem, bars, sm_m, sm_l, &sm_abort, sm_q);
    else
        int4_stream_item<T, D, 2, kLimits>(p, cache, a.x, rows, a.w, a.z, b.x, b.w, kvh, smem, bars, sm_m, sm_l, &sm_abort, sm_q);
}

}  // namespace pat
