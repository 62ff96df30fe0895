// 4-bit KV cache: append, read-back, and the launcher of the attention over it (C ABI).
//
// The layout is described in pat_int4.cuh.  The reference's cache is 16-bit only (its serving backend
// appends through vLLM's reshape_and_cache_flash, plugin/vllm/attention/backends/prefix_attn.py:828-837);
// these are the same three operations over a cache a quarter of that size.
#include "../../include/pat_b200.h"

#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <cmath>

#include "pat_dense_tc.cuh"
#include "pat_int4.cuh"

namespace {

using namespace pat;

constexpr int kMaxDevices = 64;

struct RowsParams {            // append and read-back: rows of 16-bit elements <-> cache tiles
    void* key;
    void* value;
    unsigned char* cache;
    const int64_t* slots;
    int64_t key_token, key_head, value_token, value_head;     // elements
    int64_t page_stride, head_stride;                         // bytes
    int64_t num_slots;                                        // pages * page_size
    int num_tokens, heads, page_size;
    int heads_per_cta;
};

// Byte offsets, from the start of a tile, of the codes of dims 8i .. 8i + 7 of token `tok`: one word of K,
// two 16-bit halves of V (the second 4 bytes on).
template <int D> __device__ __forceinline__ int k_word_off(int tok, int i) { return tok * Int4Tile<D>::kTokenBytes + i * 4; }
template <int D> __device__ __forceinline__ int v_half_off(int tok, int i) {
    constexpr int kPerLane = D / 64;                          // groups of 8 dims per V lane
    const int g = i / kPerLane, wh = i - g * kPerLane;
    return Int4Tile<D>::kVOff + (tok >> 3) * 4 * D + (g * 4 + ((tok & 7) >> 1)) * Int4Tile<D>::kLaneBytes + wh * 8 + (tok & 1) * 2;
}

// Both kernels: one CTA = 16 consecutive tokens of the call x some KV heads, one after the other, the next head's bytes
// on their way while one is worked on.  When the 16 slots are one tile in order - a prefill chunk, a cached prefix -
// the tile passes through shared memory and is moved by 16-byte accesses; otherwise every row goes to its place by
// itself, V in 2-byte pieces (a token owns 16-bit halves of the V words).
constexpr int kRowThreads = 256;

struct TileGroup {
    int64_t slot[16];          // -1: padding, or outside the cache
    unsigned char* tile;       // head 0's tile of a whole run, or null
};

// All threads call this; `grp` is shared memory.
template <int D> __device__ __forceinline__ void load_group(const RowsParams& p, TileGroup& grp, int token0) {
    if (threadIdx.x < 32) {
        const int t = threadIdx.x;
        int64_t slot = -1;
        if (t < 16 && token0 + t < p.num_tokens) {
            slot = __ldg(p.slots + token0 + t);
            if (slot < 0 || slot >= p.num_slots) slot = -1;
        }
        const int64_t first = __shfl_sync(kFullMask, slot, 0);
        const bool run = __all_sync(kFullMask, t >= 16 || (first >= 0 && slot == first + t)) && (first & 15) == 0;
        if (t < 16) grp.slot[t] = slot;
        if (t == 0) {
            unsigned char* tile = nullptr;
            if (run) {
                const int64_t page = first / p.page_size;
                tile = p.cache + page * p.page_stride + ((first - page * p.page_size) >> 4) * Int4Tile<D>::kBytes;
            }
            grp.tile = tile;
        }
    }
    __syncthreads();
}

template <int D> __device__ __forceinline__ unsigned char* tile_of_slot(const RowsParams& p, int64_t slot, int head, int& tok) {
    const int64_t page = slot / p.page_size;
    const int row = static_cast<int>(slot - page * p.page_size);
    tok = row & 15;
    return p.cache + page * p.page_stride + head * p.head_stride + (row >> 4) * Int4Tile<D>::kBytes;
}

template <typename T> __device__ __forceinline__ float elt_round(float x);
template <> __device__ __forceinline__ float elt_round<__nv_bfloat16>(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
template <> __device__ __forceinline__ float elt_round<__half>(float x) { return __half2float(__float2half_rn(x)); }

// Smallest and largest of two pairs, NaN if one holds a NaN.
template <typename T> __device__ __forceinline__ void min_max_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
    using V = typename Pack2<T>::V;
    const V v = *reinterpret_cast<const V*>(&w), l = __hmin2_nan(v, *reinterpret_cast<const V*>(&lo)),
            h = __hmax2_nan(v, *reinterpret_cast<const V*>(&hi));
    lo = *reinterpret_cast<const uint32_t*>(&l);
    hi = *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float min_or_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The codes of 16 elements: per 8 of them, low half dims 0, 2, 4, 6, high half 1, 3, 5, 7.
//
// code = rint((x - lo) / scale), halves to the even code, at most 15, without a division: x - lo is exact in fp32
// unless a row spans more than 2^13 times its smallest step, and (x - lo) * (1 / scale) is within 2^-18 of the quotient,
// which decides everything that does not lie that near to a half.  Adding 1.5 * 2^23 in the product's own fma rounds to
// an integer that then stands in the low mantissa bits, and a second fma gives the distance from it; both, like the
// differences, two elements at a time.  (scale is max - min over 15 rounded by 2^-9 at most, so nothing exceeds 15.5,
// unless it is subnormal: `normal` says that it is not.)
__device__ __forceinline__ void encode16(const float (&x)[16], float lo, float scale, bool normal, uint32_t (&code)[2]) {
    constexpr float kMagic = 12582912.f;
    constexpr uint32_t kMagicBits = 0x4B400000u;
    const float inv = 1.f / scale;
    const uint64_t inv2 = pack_f32x2(inv, inv), magic2 = pack_f32x2(kMagic, kMagic), less2 = pack_f32x2(-kMagic, -kMagic),
                   one2 = pack_f32x2(1.f, 1.f), minus2 = pack_f32x2(-1.f, -1.f), lo2 = pack_f32x2(-lo, -lo);
    code[0] = code[1] = 0;
    float worst = 0.f;
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
        const uint64_t d = fma_f32x2(pack_f32x2(x[j], x[j + 1]), one2, lo2);
        const uint64_t u = fma_f32x2(d, inv2, magic2);
        const uint64_t r = fma_f32x2(u, one2, less2);
        const uint64_t e = fma_f32x2(d, inv2, mul_f32x2(r, minus2));
        float u0, u1, e0, e1;
        unpack_f32x2(u, u0, u1);
        unpack_f32x2(e, e0, e1);
        worst = fmaxf(worst, fmaxf(fabsf(e0), fabsf(e1)));
        const int k = (j & 7) >> 1;          // nibble of the even element in the low half, of the odd one in the high half
        code[j >> 3] += ((__float_as_uint(u0) - kMagicBits) << (4 * k)) + ((__float_as_uint(u1) - kMagicBits) << (4 * k + 16));
    }
    if (!normal) {
        code[0] = code[1] = 0;
#pragma unroll 1
        for (int j = 0; j < 16; ++j) {
            float v = x[0];
#pragma unroll
            for (int k = 1; k < 16; ++k) v = j == k ? x[k] : v;
            const float t = fminf(rintf((v - lo) / scale), 15.f);
            const uint32_t bits = static_cast<uint32_t>(t) << (4 * ((j & 7) >> 1) + 16 * (j & 1));
            if (j < 8) code[0] |= bits; else code[1] |= bits;
        }
    } else if (worst > 0.5f - 4e-6f) {
        // Near a half (16-bit numbers meet exact halves often: about every second warp has one): the distance
        // x - lo - r scale is exact in one fma, and says whether r is the nearest, or which of two to take.
        code[0] = code[1] = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float d = x[j] - lo, u = fmaf(d, inv, kMagic), rest = fmaf(kMagic - u, scale, d);
            uint32_t r = __float_as_uint(u) - kMagicBits;
            const float twice = 2.f * fabsf(rest);
            if (twice > scale || (twice == scale && (r & 1u))) r += rest > 0.f ? 1u : ~0u;
            code[j >> 3] |= r << (4 * ((j & 7) >> 1) + 16 * (j & 1));
        }
    }
}

// D / 16 threads per row (one token, K or V), 16 elements each; the CTA's 32 rows in one or two passes.
// 8192 tokens of 8 heads of 128 elements: 18.1 us, 85 MB at 4.7 TB/s; the arithmetic of the codes beside the loads keeps it
// from the copy bandwidth (13 us).  A decode step's 256 tokens: 2.9 us, a launch and two trips to memory.
// A row with a NaN or an infinity is stored as NaN scale and offset: whoever attends it sees it.
template <typename T, int D> __global__ void __launch_bounds__(kRowThreads) append_int4_kernel(const RowsParams p) {
    using L = Int4Tile<D>;
    constexpr int kLanes = D / 16;
    __shared__ __align__(16) unsigned char image[L::kBytes];
    __shared__ TileGroup grp;
    const int splits = (p.heads + p.heads_per_cta - 1) / p.heads_per_cta;
    const int token0 = static_cast<int>(blockIdx.x / splits) * 16;
    const int head0 = static_cast<int>(blockIdx.x % splits) * p.heads_per_cta, head1 = min(head0 + p.heads_per_cta, p.heads);
    const int row = threadIdx.x / kLanes, i = threadIdx.x % kLanes;
    const int tok_in = row & 15;
    const bool is_v = row >= 16;
    // the rows are requested before the slots are looked at: a padding token's row is read for nothing
    const bool have = row < 32 && token0 + tok_in < p.num_tokens;
    const int64_t token = token0 + tok_in, head_step = is_v ? p.value_head : p.key_head;
    const T* src = (is_v ? static_cast<const T*>(p.value) + token * p.value_token : static_cast<const T*>(p.key) + token * p.key_token) +
                   head0 * head_step + 16 * i;
    uint4 next[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    auto request = [&]() {
        if (!have) return;
        next[0] = __ldg(reinterpret_cast<const uint4*>(src));
        next[1] = __ldg(reinterpret_cast<const uint4*>(src) + 1);
        src += head_step;
    };
    request();
    load_group<D>(p, grp, token0);
#pragma unroll 1
    for (int head = head0; head < head1; ++head) {
        const uint32_t words[8] = {next[0].x, next[0].y, next[0].z, next[0].w, next[1].x, next[1].y, next[1].z, next[1].w};
        if (head + 1 < head1) request();
        uint32_t lo2 = words[0], hi2 = words[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) min_max_pairs<T>(words[j], lo2, hi2);
        const float2 lo_pair = Int4Elt<T>::unpack(lo2), hi_pair = Int4Elt<T>::unpack(hi2);
        float lo = min_or_nan(lo_pair.x, lo_pair.y), hi = max_or_nan(hi_pair.x, hi_pair.y);
#pragma unroll
        for (int d = kLanes / 2; d > 0; d >>= 1) {
            lo = min_or_nan(lo, __shfl_xor_sync(kFullMask, lo, d));
            hi = max_or_nan(hi, __shfl_xor_sync(kFullMask, hi, d));
        }
        float x[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 e = Int4Elt<T>::unpack(words[j]);
            x[2 * j] = e.x;
            x[2 * j + 1] = e.y;
        }
        const bool bad = !(fabsf(lo) <= FLT_MAX && fabsf(hi) <= FLT_MAX);
        float scale, half = 1.f;
        if (bad || hi - lo <= FLT_MAX) {
            scale = elt_round<T>((hi - lo) / 15.f);
        } else {                   // a bf16 row may span more than fp32 can hold: everything halved, which is exact
            scale = elt_round<T>((0.5f * hi - 0.5f * lo) / 7.5f);
            half = 0.5f;
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] *= 0.5f;
        }
        if (bad) scale = NAN;
        const uint32_t prm = Elt<T>::pack(scale, bad ? NAN : lo);
        uint32_t code[2] = {0, 0};
        constexpr float kNormal = Int4Elt<T>::kIsHalf ? 6.103515625e-05f : 2.35098870164457501594e-38f;    // (bf16: a reciprocal stays finite)
        if (scale > 0.f) encode16(x, half * lo, half * scale, scale >= kNormal, code);
        // where the row goes: the image of the tile, or straight to the cache
        unsigned char* tile = image;
        int tok = tok_in;
        if (!grp.tile) {
            const int64_t slot = grp.slot[tok_in];
            tile = have && slot >= 0 ? tile_of_slot<D>(p, slot, head, tok) : nullptr;
        }
        if (tile && row < 32) {
            if (!is_v) {
                *reinterpret_cast<uint2*>(tile + k_word_off<D>(tok, 2 * i)) = make_uint2(code[0], code[1]);
            } else {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    uint16_t* dst = reinterpret_cast<uint16_t*>(tile + v_half_off<D>(tok, 2 * i + b));
                    dst[0] = static_cast<uint16_t>(code[b]);
                    dst[2] = static_cast<uint16_t>(code[b] >> 16);
                }
            }
            if (i == 0) *reinterpret_cast<uint32_t*>(tile + (is_v ? L::kVPrm : L::kKPrm) + tok * 4) = prm;
        }
        if (grp.tile) {
            __syncthreads();
            for (int j = threadIdx.x; j < L::kBytes / 16; j += kRowThreads)
                reinterpret_cast<uint4*>(grp.tile + head * p.head_stride)[j] = reinterpret_cast<const uint4*>(image)[j];
            __syncthreads();
        }
    }
}

// The inverse: value = lo + scale * code in fp32 (one rounding, the product is exact), rounded to T.
// D / 8 threads per row, 8 elements each.  65536 tokens of 8 heads of 128 elements: 64.3 us, 340 MB at 5.3 TB/s (0.81 of the
// copy bandwidth); four fifths of the bytes are writes.
template <typename T, int D> __global__ void __launch_bounds__(kRowThreads, 8) gather_int4_kernel(const RowsParams p) {
    using L = Int4Tile<D>;
    constexpr int kLanes = D / 8, kRowsPerPass = kRowThreads / kLanes;
    __shared__ __align__(16) unsigned char image[L::kBytes];
    __shared__ TileGroup grp;
    const int splits = (p.heads + p.heads_per_cta - 1) / p.heads_per_cta;
    const int token0 = static_cast<int>(blockIdx.x / splits) * 16;
    const int head0 = static_cast<int>(blockIdx.x % splits) * p.heads_per_cta, head1 = min(head0 + p.heads_per_cta, p.heads);
    load_group<D>(p, grp, token0);
    constexpr int kVecs = L::kBytes / 16;
    static_assert(kVecs <= kRowThreads, "one 16-byte piece of a tile per thread");
    uint4 next = make_uint4(0, 0, 0, 0);
    const int i = threadIdx.x % kLanes;
    if (grp.tile && threadIdx.x < kVecs) next = __ldg(reinterpret_cast<const uint4*>(grp.tile + head0 * p.head_stride) + threadIdx.x);
#pragma unroll 1
    for (int head = head0; head < head1; ++head) {
        if (grp.tile) {
            if (threadIdx.x < kVecs) {
                reinterpret_cast<uint4*>(image)[threadIdx.x] = next;
                if (head + 1 < head1) next = __ldg(reinterpret_cast<const uint4*>(grp.tile + (head + 1) * p.head_stride) + threadIdx.x);
            }
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < 32 / kRowsPerPass; ++r) {
            const int row = threadIdx.x / kLanes + r * kRowsPerPass;
            const int tok_in = row & 15;
            const bool is_v = row >= 16;
            const unsigned char* tile = image;
            int tok = tok_in;
            if (!grp.tile) {
                const int64_t slot = grp.slot[tok_in];
                if (slot < 0) continue;
                tile = tile_of_slot<D>(p, slot, head, tok);
            }
            uint32_t word;
            if (!is_v) {
                word = *reinterpret_cast<const uint32_t*>(tile + k_word_off<D>(tok, i));
            } else {
                const uint16_t* src = reinterpret_cast<const uint16_t*>(tile + v_half_off<D>(tok, i));
                word = src[0] | (static_cast<uint32_t>(src[2]) << 16);
            }
            const float2 prm = Int4Elt<T>::unpack(*reinterpret_cast<const uint32_t*>(tile + (is_v ? L::kVPrm : L::kKPrm) + tok * 4));
            const uint32_t pairs[4] = {Int4Elt<T>::template pair<0>(word), Int4Elt<T>::template pair<1>(word),
                                       Int4Elt<T>::template pair<2>(word), Int4Elt<T>::template pair<3>(word)};
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 c = Int4Elt<T>::unpack(pairs[j]);       // 16 + code
                out[j] = Elt<T>::pack(fmaf(c.x - 16.f, prm.x, prm.y), fmaf(c.y - 16.f, prm.x, prm.y));
            }
            const int64_t token = token0 + tok_in;
            T* dst = is_v ? static_cast<T*>(p.value) + token * p.value_token + head * p.value_head
                          : static_cast<T*>(p.key) + token * p.key_token + head * p.key_head;
            reinterpret_cast<uint4*>(dst)[i] = make_uint4(out[0], out[1], out[2], out[3]);
        }
        if (grp.tile) __syncthreads();
    }
}

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

int check_device(int* dev) {
    if (cudaGetDevice(dev) != cudaSuccess) return PAT_ERR_CUDA;
    if (*dev < 0 || *dev >= kMaxDevices) return PAT_ERR_UNSUPPORTED;
    static thread_local int checked = -1;
    if (checked != *dev) {
        int major = 0;
        if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *dev) != cudaSuccess) return PAT_ERR_CUDA;
        if (major != 10) return PAT_ERR_NO_DEVICE_CODE;
        checked = *dev;
    }
    return PAT_OK;
}

// KV heads per CTA: with a CTA for each of them (head by head) a short call fills more SMs; a long one is faster when a
// CTA walks the heads of its tokens, since it then waits for memory once.  Half a wave of 8 CTAs per SM divides the two.
// One head per CTA / all eight / this rule, heads of 128 elements on a B200: append of 256 tokens 2.9 / 9.5 / 2.9 us, of
// 8192 tokens 22.0 / 19.8 / 18.1; read-back of 65536 tokens 89.6 / 64.3 / 64.3.
int heads_per_cta(const pat_int4_rows_args& a) {
    const int64_t groups = (static_cast<int64_t>(a.num_tokens) + 15) / 16;
    int n = 1;
    while (n < a.num_kv_heads && groups * ((a.num_kv_heads + 2 * n - 1) / (2 * n)) >= 4 * 148) n *= 2;
    return n;
}
int64_t row_blocks(const pat_int4_rows_args& a) {
    const int n = heads_per_cta(a);
    return (static_cast<int64_t>(a.num_tokens) + 15) / 16 * ((a.num_kv_heads + n - 1) / n);
}

int rows_params(const pat_int4_rows_args& a, RowsParams* out) {
    if (a.num_tokens < 0 || a.num_kv_heads <= 0 || a.num_pages <= 0) return PAT_ERR_BAD_ARGUMENT;
    if (a.dtype != PAT_DTYPE_FP16 && a.dtype != PAT_DTYPE_BF16) return PAT_ERR_UNSUPPORTED;
    if (a.head_dim != 64 && a.head_dim != 128) return PAT_ERR_UNSUPPORTED;
    if (a.page_size < 16 || a.page_size % 16 != 0 || a.page_size > 256) return PAT_ERR_UNSUPPORTED;
    if (a.num_tokens == 0) return PAT_OK;
    if (!a.key || !a.value || !a.cache || !a.slot_mapping) return PAT_ERR_BAD_ARGUMENT;
    if (!aligned16(a.key) || !aligned16(a.value) || !aligned16(a.cache)) return PAT_ERR_UNSUPPORTED;
    const int64_t elts[] = {a.key_token_stride, a.key_head_stride, a.value_token_stride, a.value_head_stride};
    for (int64_t s : elts)
        if (s <= 0 || s % 8 != 0) return PAT_ERR_UNSUPPORTED;
    if (a.page_stride <= 0 || a.page_stride % 16 != 0 || a.head_stride <= 0 || a.head_stride % 16 != 0) return PAT_ERR_UNSUPPORTED;
    RowsParams p{};
    p.key = a.key;
    p.value = a.value;
    p.cache = static_cast<unsigned char*>(a.cache);
    p.slots = a.slot_mapping;
    p.key_token = a.key_token_stride;
    p.key_head = a.key_head_stride;
    p.value_token = a.value_token_stride;
    p.value_head = a.value_head_stride;
    p.page_stride = a.page_stride;
    p.head_stride = a.head_stride;
    p.num_slots = a.num_pages * static_cast<int64_t>(a.page_size);
    p.num_tokens = a.num_tokens;
    p.heads = a.num_kv_heads;
    p.page_size = a.page_size;
    p.heads_per_cta = heads_per_cta(a);
    if (row_blocks(a) > 0x7fffffffLL || a.num_tokens > 0x7fffffff - 16) return PAT_ERR_TOO_LARGE;
    *out = p;
    return PAT_OK;
}

template <typename T, int D> int launch_attention(const pat_decode_int4_args& a, cudaStream_t stream, int dev) {
    const size_t rows = static_cast<size_t>(a.work.num_entries) * a.work.hratio;
    float* part_o = reinterpret_cast<float*>(static_cast<unsigned char*>(a.workspace) + kWorkspaceHeadBytes);
    float* part_lse = part_o + rows * D;
    const int q_per_req = a.q_per_req > 1 ? a.q_per_req : 1;
    const bool limits = a.work.limits_off >= 0;
    AttnParams p{};
    p.q = a.q;
    p.part_o = part_o;
    p.part_lse = part_lse;
    p.items = a.work_blob + a.work.items_off;
    p.num_items = a.work.num_stream_items;
    p.queries = a.work_blob + a.work.queries_off;
    p.pages = a.work_blob + a.work.pages_off;
    p.limits = limits ? a.work_blob + a.work.limits_off : nullptr;
    p.q_per_req = q_per_req;
    p.q_batch_stride = a.q_batch_stride;
    p.q_head_stride = a.q_head_stride;
    p.q_pos_stride = q_per_req > 1 ? a.q_pos_stride : 0;
    p.kv_heads = a.num_kv_heads;
    p.hratio = a.work.hratio;
    p.num_q_heads = a.num_q_heads;
    p.page_size = a.page_size;
    p.scale = a.softmax_scale;
    p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
    p.status = a.status_word;
    p.wait_ns = a.wait_limit_us > 0 ? static_cast<uint64_t>(a.wait_limit_us) * 1000ull : kDefaultWaitNs;
    const Int4Cache cache{static_cast<const unsigned char*>(a.kv_cache), a.page_stride, a.head_stride, 64u};

    // The order of the 16-bit path: dense kernel, streaming kernel as its programmatic dependent, merge (which
    // waits for the last dense CTA through a control word of the workspace).
    const bool streaming = a.work.num_stream_items > 0 && !(a.flags & PAT_SKIP_STREAM);
    const bool dense = a.work.num_dense_items > 0 && !(a.flags & PAT_SKIP_DENSE);
    const bool merge = !(a.flags & PAT_SKIP_MERGE);
    const bool overlap = streaming && dense && !(a.flags & PAT_NO_OVERLAP);
    int32_t* sync = overlap && merge ? static_cast<int32_t*>(a.workspace) : nullptr;
    if (dense) {
        static std::atomic<bool> configured[kMaxDevices][2];
        auto kern = limits ? dense_tc_int4_kernel<T, D, true> : dense_tc_int4_kernel<T, D, false>;
        constexpr int smem = TcSmem<D, true>::kRequest;
        if (!configured[dev][limits].load(std::memory_order_acquire)) {
            if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return PAT_ERR_CUDA;
            configured[dev][limits].store(true, std::memory_order_release);
        }
        DenseTcParams dp{};
        dp.a = p;
        dp.a.items = p.items + static_cast<size_t>(a.work.num_stream_items) * 8;
        dp.a.num_items = a.work.num_dense_items;
        dp.cta_begin = a.work_blob + a.work.dense_cta_off;
        dp.dense_q = a.work_blob + a.work.dense_q_off;
        dp.dense_q_width = a.work.dense_q_width;
        dp.sync = sync;
        kern<<<static_cast<unsigned>(a.work.num_dense_ctas), kTcInt4Threads, smem, stream>>>(dp, cache);
    }
    if (streaming) {
        static std::atomic<bool> configured[kMaxDevices][2];
        auto kern = limits ? int4_stream_kernel<T, D, true> : int4_stream_kernel<T, D, false>;
        constexpr int smem = int4_stream_smem_bytes<D>();
        if (!configured[dev][limits].load(std::memory_order_acquire)) {
            if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return PAT_ERR_CUDA;
            configured[dev][limits].store(true, std::memory_order_release);
        }
        const long long grid = (static_cast<long long>(p.num_items) * a.num_kv_heads + kInt4Warps - 1) / kInt4Warps;
        if (grid > 0x7fffffffLL) return PAT_ERR_TOO_LARGE;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>(grid));
        cfg.blockDim = dim3(kInt4Warps * 32);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = overlap ? 1 : 0;
        if (cudaLaunchKernelEx(&cfg, kern, p, cache) != cudaSuccess) return PAT_ERR_CUDA;
    }
    if (!merge) return cudaGetLastError() == cudaSuccess ? PAT_OK : PAT_ERR_CUDA;
    MergeParams mp{};
    mp.sync = sync;
    mp.status = a.status_word;
    mp.wait_ns = p.wait_ns;
    mp.part_o = part_o;
    mp.part_lse = part_lse;
    mp.indptr = a.work_blob + a.work.merge_indptr_off;
    mp.entries = a.work_blob + a.work.merge_entries_off;
    mp.out = a.out;
    mp.lse_out = a.lse_out;
    mp.out_batch_stride = a.out_batch_stride;
    mp.out_head_stride = a.out_head_stride;
    mp.out_pos_stride = q_per_req > 1 ? a.out_pos_stride : 0;
    mp.q_per_req = q_per_req;
    mp.batch = a.batch * q_per_req;
    mp.num_q_heads = a.num_q_heads;
    mp.kv_heads = a.num_kv_heads;
    mp.hratio = a.work.hratio;
    const int total = a.batch * q_per_req * a.num_q_heads;
    merge_kernel<T, D><<<(total + 7) / 8, 256, 0, stream>>>(mp);
    return cudaGetLastError() == cudaSuccess ? PAT_OK : PAT_ERR_CUDA;
}

}  // namespace

extern "C" {

size_t pat_b200_int4_tile_bytes(int head_dim) {
    return head_dim == 64 || head_dim == 128 ? static_cast<size_t>(16 * head_dim + 128) : 0;
}

int pat_b200_append_int4(const pat_int4_rows_args* args, void* stream_handle) {
    if (!args) return PAT_ERR_BAD_ARGUMENT;
    RowsParams p{};
    int rc = rows_params(*args, &p);
    if (rc != PAT_OK || args->num_tokens == 0) return rc;
    int dev = 0;
    if ((rc = check_device(&dev)) != PAT_OK) return rc;
    const bool bf16 = args->dtype == PAT_DTYPE_BF16;
    auto kern = args->head_dim == 128 ? (bf16 ? append_int4_kernel<__nv_bfloat16, 128> : append_int4_kernel<__half, 128>)
                                      : (bf16 ? append_int4_kernel<__nv_bfloat16, 64> : append_int4_kernel<__half, 64>);
    kern<<<static_cast<unsigned>(row_blocks(*args)), kRowThreads, 0, static_cast<cudaStream_t>(stream_handle)>>>(p);
    return cudaGetLastError() == cudaSuccess ? PAT_OK : PAT_ERR_CUDA;
}

int pat_b200_gather_int4(const pat_int4_rows_args* args, void* stream_handle) {
    if (!args) return PAT_ERR_BAD_ARGUMENT;
    RowsParams p{};
    int rc = rows_params(*args, &p);
    if (rc != PAT_OK || args->num_tokens == 0) return rc;
    int dev = 0;
    if ((rc = check_device(&dev)) != PAT_OK) return rc;
    const bool bf16 = args->dtype == PAT_DTYPE_BF16;
    auto kern = args->head_dim == 128 ? (bf16 ? gather_int4_kernel<__nv_bfloat16, 128> : gather_int4_kernel<__half, 128>)
                                      : (bf16 ? gather_int4_kernel<__nv_bfloat16, 64> : gather_int4_kernel<__half, 64>);
    kern<<<static_cast<unsigned>(row_blocks(*args)), kRowThreads, 0, static_cast<cudaStream_t>(stream_handle)>>>(p);
    return cudaGetLastError() == cudaSuccess ? PAT_OK : PAT_ERR_CUDA;
}

int pat_b200_decode_int4(const pat_decode_int4_args* args, void* stream_handle) {
    if (!args) return PAT_ERR_BAD_ARGUMENT;
    const pat_decode_int4_args& a = *args;
    if (!a.q || !a.kv_cache || !a.out || !a.work_blob) return PAT_ERR_BAD_ARGUMENT;
    if (a.batch <= 0 || a.num_q_heads <= 0 || a.num_kv_heads <= 0 || a.num_pages <= 0) return PAT_ERR_BAD_ARGUMENT;
    if (a.num_q_heads % a.num_kv_heads != 0) return PAT_ERR_BAD_ARGUMENT;
    const int positions = a.q_per_req > 1 ? a.q_per_req : 1;
    if (a.work.q_per_req != positions || static_cast<int64_t>(a.work.batch) != static_cast<int64_t>(a.batch) * positions)
        return PAT_ERR_BAD_PLAN;
    if (a.work.hratio != a.num_q_heads / a.num_kv_heads || a.work.page_size != a.page_size || a.work.kv_heads != a.num_kv_heads)
        return PAT_ERR_BAD_PLAN;
    if (a.work.max_page_id >= a.num_pages) return PAT_ERR_BAD_PLAN;
    if (a.head_dim != 64 && a.head_dim != 128) return PAT_ERR_UNSUPPORTED;
    if (a.dtype != PAT_DTYPE_FP16 && a.dtype != PAT_DTYPE_BF16) return PAT_ERR_UNSUPPORTED;
    if (a.page_size < 16 || a.page_size % 16 != 0 || a.page_size > 256) return PAT_ERR_UNSUPPORTED;
    if (a.work.hratio < 1 || a.work.hratio > 16) return PAT_ERR_UNSUPPORTED;
    if (!(a.softmax_scale > 0.f) || !std::isfinite(a.softmax_scale)) return PAT_ERR_BAD_ARGUMENT;
    if (!aligned16(a.kv_cache) || !aligned16(a.q) || !aligned16(a.out) || !aligned16(a.work_blob)) return PAT_ERR_UNSUPPORTED;
    if (a.page_stride <= 0 || a.page_stride % 16 != 0 || a.head_stride <= 0 || a.head_stride % 16 != 0) return PAT_ERR_UNSUPPORTED;
    const int64_t strides[] = {a.q_batch_stride, a.q_head_stride, a.out_batch_stride, a.out_head_stride};
    for (int64_t s : strides)
        if (s <= 0 || s % 8 != 0) return PAT_ERR_UNSUPPORTED;
    if (positions > 1 && (a.q_pos_stride <= 0 || a.q_pos_stride % 8 != 0 || a.out_pos_stride <= 0 || a.out_pos_stride % 8 != 0))
        return PAT_ERR_UNSUPPORTED;
    const size_t need = pat_b200_workspace_bytes(&a.work, a.num_q_heads, a.head_dim);
    if (!a.workspace || a.workspace_bytes < need || (reinterpret_cast<uintptr_t>(a.workspace) & 31) != 0) return PAT_ERR_WORKSPACE;
    int dev = 0;
    const int rc = check_device(&dev);
    if (rc != PAT_OK) return rc;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
    const bool bf16 = a.dtype == PAT_DTYPE_BF16;
    if (a.head_dim == 128)
        return bf16 ? launch_attention<__nv_bfloat16, 128>(a, stream, dev) : launch_attention<__half, 128>(a, stream, dev);
    return bf16 ? launch_attention<__nv_bfloat16, 64>(a, stream, dev) : launch_attention<__half, 64>(a, stream, dev);
}

}  // extern "C"
