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
    int64_t num_slots, num_rows;                              // pages * page_size; tokens * 2 * heads
    int heads, page_size;
};

// Byte offsets, from the start of the tile, of what the thread that owns dims 8i .. 8i + 7 of token
// `tok` reads or writes: one word of K, two 16-bit halves of V (the second 4 bytes on).
template <int D> __device__ __forceinline__ int k_word_off(int tok, int i) { return tok * Int4Tile<D>::kTokenBytes + i * 4; }
template <int D> __device__ __forceinline__ int v_half_off(int tok, int i) {
    constexpr int kThreadsPerLane = D / 64;                   // 16-byte pieces of a row per V lane
    const int g = i / kThreadsPerLane, wh = i - g * kThreadsPerLane;
    return Int4Tile<D>::kVOff + (tok >> 3) * 4 * D + (g * 4 + ((tok & 7) >> 1)) * Int4Tile<D>::kLaneBytes + wh * 8 + (tok & 1) * 2;
}

// Address of the tile of (slot, head), or null for a padding slot / a slot outside the cache.
template <int D> __device__ __forceinline__ unsigned char* tile_of_slot(const RowsParams& p, int64_t slot, int head, int& tok) {
    if (slot < 0 || slot >= p.num_slots) return nullptr;
    const int64_t page = slot / p.page_size;
    const int row = static_cast<int>(slot - page * p.page_size);
    tok = row & 15;
    return p.cache + page * p.page_stride + head * p.head_stride + (row >> 4) * Int4Tile<D>::kBytes;
}

template <typename T> __device__ __forceinline__ float elt_round(float x);
template <> __device__ __forceinline__ float elt_round<__nv_bfloat16>(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
template <> __device__ __forceinline__ float elt_round<__half>(float x) { return __half2float(__float2half_rn(x)); }

// D / 8 threads per row (a row = one token, one head, K or V), 8 elements each.
//
// scale = round16((max - lo) / 15), code = rint((x - lo) / scale) clipped to 15.  All quotients are IEEE
// divisions of differences that are exact in fp32 unless the row spans more than 2^13: then every
// code and scale is the one the definition gives in exact arithmetic.  A row with a NaN or an infinity is stored as
// NaN scale and offset: whoever attends it sees it.
template <typename T, int D> __global__ void __launch_bounds__(256) append_int4_kernel(const RowsParams p) {
    constexpr int kLanes = D / 8;
    const int64_t idx = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
    const int64_t r = idx / kLanes;
    const int i = static_cast<int>(idx) % kLanes;
    const bool have = r < p.num_rows;
    const int per_token = 2 * p.heads;
    const int64_t token = have ? r / per_token : 0;
    const int rem = static_cast<int>(r - token * per_token);
    const bool is_v = rem >= p.heads;
    const int head = is_v ? rem - p.heads : rem;
    int tok = 0;
    unsigned char* tile = have ? tile_of_slot<D>(p, __ldg(p.slots + token), head, tok) : nullptr;

    uint4 raw = make_uint4(0, 0, 0, 0);
    if (tile) {
        const T* src = is_v ? static_cast<const T*>(p.value) + token * p.value_token + head * p.value_head
                            : static_cast<const T*>(p.key) + token * p.key_token + head * p.key_head;
        raw = __ldg(reinterpret_cast<const uint4*>(src) + i);
    }
    float x[8];
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 e = Int4Elt<T>::unpack(words[j]);
        x[2 * j] = e.x;
        x[2 * j + 1] = e.y;
    }
    float lo = x[0], hi = x[0];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
        bad = bad || !(fabsf(x[j]) <= FLT_MAX);
    }
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(kFullMask, lo, d));
        hi = fmaxf(hi, __shfl_xor_sync(kFullMask, hi, d));
    }
    const uint32_t bad_lanes = __ballot_sync(kFullMask, bad);
    const int lane = threadIdx.x & 31;
    bad = ((bad_lanes >> (lane & ~(kLanes - 1))) & ((1u << kLanes) - 1u)) != 0;
    if (!tile) return;
    // (a bf16 row may span more than fp32 can hold: then everything is halved, which is exact)
    const float h = isinf(hi - lo) ? 0.5f : 1.f;
    const float scale = bad ? NAN : elt_round<T>((h * hi - h * lo) / (15.f * h));
    uint32_t word = 0;
    if (scale > 0.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = fminf(rintf((h * x[j] - h * lo) / (h * scale)), 15.f);
            // dims 0, 2, 4, 6 in the low half, 1, 3, 5, 7 in the high one
            word |= static_cast<uint32_t>(t) << (4 * (j >> 1) + 16 * (j & 1));
        }
    }
    if (!is_v) {
        *reinterpret_cast<uint32_t*>(tile + k_word_off<D>(tok, i)) = word;
    } else {
        uint16_t* dst = reinterpret_cast<uint16_t*>(tile + v_half_off<D>(tok, i));
        dst[0] = static_cast<uint16_t>(word);
        dst[2] = static_cast<uint16_t>(word >> 16);
    }
    if (i == 0)
        *reinterpret_cast<uint32_t*>(tile + (is_v ? Int4Tile<D>::kVPrm : Int4Tile<D>::kKPrm) + tok * 4) =
            Elt<T>::pack(scale, bad ? NAN : lo);
}

// The inverse: value = lo + scale * code in fp32 (one rounding, the product is exact), rounded to T.
template <typename T, int D> __global__ void __launch_bounds__(256) gather_int4_kernel(const RowsParams p) {
    constexpr int kLanes = D / 8;
    const int64_t idx = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
    const int64_t r = idx / kLanes;
    const int i = static_cast<int>(idx) % kLanes;
    if (r >= p.num_rows) return;
    const int per_token = 2 * p.heads;
    const int64_t token = r / per_token;
    const int rem = static_cast<int>(r - token * per_token);
    const bool is_v = rem >= p.heads;
    const int head = is_v ? rem - p.heads : rem;
    int tok = 0;
    const unsigned char* tile = tile_of_slot<D>(p, __ldg(p.slots + token), head, tok);
    if (!tile) return;
    uint32_t word;
    if (!is_v) {
        word = *reinterpret_cast<const uint32_t*>(tile + k_word_off<D>(tok, i));
    } else {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(tile + v_half_off<D>(tok, i));
        word = src[0] | (static_cast<uint32_t>(src[2]) << 16);
    }
    const float2 prm = Int4Elt<T>::unpack(
        *reinterpret_cast<const uint32_t*>(tile + (is_v ? Int4Tile<D>::kVPrm : Int4Tile<D>::kKPrm) + tok * 4));
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = fmaf(static_cast<float>((word >> (4 * j)) & 15u), prm.x, prm.y);
        const float b = fmaf(static_cast<float>((word >> (4 * j + 16)) & 15u), prm.x, prm.y);
        out[j] = Elt<T>::pack(a, b);
    }
    T* dst = is_v ? static_cast<T*>(p.value) + token * p.value_token + head * p.value_head
                  : static_cast<T*>(p.key) + token * p.key_token + head * p.key_head;
    reinterpret_cast<uint4*>(dst)[i] = make_uint4(out[0], out[1], out[2], out[3]);
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
    p.num_rows = static_cast<int64_t>(a.num_tokens) * 2 * a.num_kv_heads;
    p.heads = a.num_kv_heads;
    p.page_size = a.page_size;
    const int64_t blocks = (p.num_rows * (a.head_dim / 8) + 255) / 256;
    if (blocks > 0x7fffffffLL) return PAT_ERR_TOO_LARGE;
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
    const Int4Cache cache{static_cast<const unsigned char*>(a.kv_cache), a.page_stride, a.head_stride};

    if (a.work.num_stream_items > 0) {
        static std::atomic<bool> configured[kMaxDevices][2];
        auto kern = limits ? int4_stream_kernel<T, D, true> : int4_stream_kernel<T, D, false>;
        constexpr int smem = int4_stream_smem_bytes<D>();
        if (!configured[dev][limits].load(std::memory_order_acquire)) {
            if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return PAT_ERR_CUDA;
            configured[dev][limits].store(true, std::memory_order_release);
        }
        const long long grid = static_cast<long long>(p.num_items) * a.num_kv_heads;
        if (grid > 0x7fffffffLL) return PAT_ERR_TOO_LARGE;
        kern<<<static_cast<unsigned>(grid), kInt4Warps * 32, smem, stream>>>(p, cache);
    }
    MergeParams mp{};
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
    const unsigned blocks = static_cast<unsigned>((p.num_rows * (args->head_dim / 8) + 255) / 256);
    kern<<<blocks, 256, 0, static_cast<cudaStream_t>(stream_handle)>>>(p);
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
    const unsigned blocks = static_cast<unsigned>((p.num_rows * (args->head_dim / 8) + 255) / 256);
    kern<<<blocks, 256, 0, static_cast<cudaStream_t>(stream_handle)>>>(p);
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
    if (a.work.max_page_id >= a.num_pages || a.work.num_dense_items > 0) return PAT_ERR_BAD_PLAN;
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
