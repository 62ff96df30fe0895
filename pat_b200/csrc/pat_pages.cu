// Copies of whole pages inside paged caches: forking a request whose last page is part-filled, and
// compaction (C ABI: pat_b200_copy_pages).
//
// The reference leaves both to its serving engine.  A step copies few pages of many tensors (K and V of
// every layer), so one launch handles all of them; the (from, to) pairs of a plan made on the host travel
// in the kernel's parameters - no upload, nothing that has to stay alive, capturable - and a plan that
// lives on the device is read from there.
// 16-byte accesses, several in flight per thread.  268 MB (read and written): 37.5 us, 7.1 TB/s with the L2's help, 1.09 of
// the plain copy bandwidth; a fork's 16 MB: 4 us, launch and latency.
#include <cuda_runtime.h>

#include <cstdint>
#include <vector>

#include "../../include/pat_b200.h"

namespace {

constexpr int kMaxCaches = 64;         // tensors per launch
constexpr int kFewPairs = 64;          // host-planned pairs per launch: the two sizes of the parameter block
constexpr int kManyPairs = 2048;
constexpr int kThreads = 256;
constexpr int kUnroll = 4;             // 16-byte pieces in flight per thread

template <int kCap> struct CopyParams {
    unsigned char* caches[kMaxCaches];
    const int64_t* device_pairs;       // [num_pairs][2], or null: `pairs`
    int64_t page_stride, row_stride;   // bytes
    int64_t num_pages;
    int32_t rows, row_vecs;            // a page = `rows` runs of row_vecs 16-byte pieces
    int32_t num_pairs, blocks_per_page;
    int32_t pairs[kCap][2];
};

// blockIdx.x = (pair * blocks_per_page + part), blockIdx.y = tensor.
template <int kCap> __global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ CopyParams<kCap> p) {
    const int pair = blockIdx.x / p.blocks_per_page, part = blockIdx.x - pair * p.blocks_per_page;
    int64_t from, to;
    if (p.device_pairs) {
        from = __ldg(p.device_pairs + 2 * pair);
        to = __ldg(p.device_pairs + 2 * pair + 1);
        if (from < 0 || to < 0 || from >= p.num_pages || to >= p.num_pages) return;
    } else {
        from = p.pairs[pair][0];
        to = p.pairs[pair][1];
    }
    unsigned char* base = p.caches[blockIdx.y];
    const unsigned char* src = base + from * p.page_stride;
    unsigned char* dst = base + to * p.page_stride;
    const int total = p.rows * p.row_vecs;
    const int first = part * (kThreads * kUnroll) + threadIdx.x;
    uint4 v[kUnroll];
    int64_t off[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int at = first + i * kThreads;
        if (at < total) {
            const int row = at / p.row_vecs;
            off[i] = row * p.row_stride + static_cast<int64_t>(at - row * p.row_vecs) * 16;
            v[i] = *reinterpret_cast<const uint4*>(src + off[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
        if (first + i * kThreads < total) *reinterpret_cast<uint4*>(dst + off[i]) = v[i];
}

// No page may be the target of two pairs, nor a source and a target: the blocks run in any order.
// One bit per page; the words that were set are cleared again, so the array stays zero between calls.
int check_pairs(const int64_t* pairs, int64_t n, int64_t num_pages) {
    static thread_local std::vector<uint64_t> marked;
    for (int64_t i = 0; i < 2 * n; ++i)
        if (pairs[i] < 0 || pairs[i] >= num_pages) return PAT_ERR_BAD_PLAN;
    if (marked.size() < static_cast<size_t>(num_pages + 63) / 64) marked.resize(static_cast<size_t>(num_pages + 63) / 64, 0);
    bool fine = true;
    for (int64_t i = 0; i < n; ++i) {
        uint64_t& w = marked[static_cast<size_t>(pairs[2 * i + 1]) >> 6];
        const uint64_t bit = 1ull << (pairs[2 * i + 1] & 63);
        fine = fine && !(w & bit);
        w |= bit;
    }
    for (int64_t i = 0; i < n; ++i) fine = fine && !(marked[static_cast<size_t>(pairs[2 * i]) >> 6] >> (pairs[2 * i] & 63) & 1);
    for (int64_t i = 0; i < n; ++i) marked[static_cast<size_t>(pairs[2 * i + 1]) >> 6] = 0;
    return fine ? PAT_OK : PAT_ERR_BAD_PLAN;
}

template <int kCap> int launch_copies(const pat_copy_args& a, cudaStream_t stream) {
    const int64_t vecs = static_cast<int64_t>(a.rows) * (a.row_bytes / 16);
    CopyParams<kCap> p;
    p.page_stride = a.page_stride;
    p.row_stride = a.row_stride;
    p.num_pages = a.num_pages;
    p.rows = a.rows;
    p.row_vecs = static_cast<int32_t>(a.row_bytes / 16);
    p.blocks_per_page = static_cast<int32_t>((vecs + kThreads * kUnroll - 1) / (kThreads * kUnroll));
    p.device_pairs = a.device_pairs;
    const int chunk = a.host_pairs ? kCap : a.num_pairs;
    if (static_cast<int64_t>(chunk < a.num_pairs ? chunk : a.num_pairs) * p.blocks_per_page > 0x7fffffffLL) return PAT_ERR_TOO_LARGE;
    for (int c0 = 0; c0 < a.num_caches; c0 += kMaxCaches) {
        const int nc = a.num_caches - c0 < kMaxCaches ? a.num_caches - c0 : kMaxCaches;
        for (int i = 0; i < nc; ++i) p.caches[i] = static_cast<unsigned char*>(a.caches[c0 + i]);
        for (int p0 = 0; p0 < a.num_pairs; p0 += chunk) {
            const int np = a.num_pairs - p0 < chunk ? a.num_pairs - p0 : chunk;
            if (a.host_pairs)
                for (int i = 0; i < np; ++i) {
                    p.pairs[i][0] = static_cast<int32_t>(a.host_pairs[2 * static_cast<int64_t>(p0 + i)]);
                    p.pairs[i][1] = static_cast<int32_t>(a.host_pairs[2 * static_cast<int64_t>(p0 + i) + 1]);
                }
            copy_pages_kernel<kCap><<<dim3(static_cast<unsigned>(static_cast<int64_t>(np) * p.blocks_per_page), static_cast<unsigned>(nc)),
                                      kThreads, 0, stream>>>(p);
        }
    }
    return cudaGetLastError() == cudaSuccess ? PAT_OK : PAT_ERR_CUDA;
}

}  // namespace

extern "C" int pat_b200_copy_pages(const pat_copy_args* args, void* stream_handle) {
    if (!args) return PAT_ERR_BAD_ARGUMENT;
    const pat_copy_args& a = *args;
    if (a.num_caches < 0 || a.num_pairs < 0 || a.num_pages <= 0 || a.rows <= 0 || a.row_bytes <= 0) return PAT_ERR_BAD_ARGUMENT;
    if (a.num_caches == 0 || a.num_pairs == 0) return PAT_OK;
    if (!a.caches || (!a.host_pairs && !a.device_pairs) || (a.host_pairs && a.device_pairs)) return PAT_ERR_BAD_ARGUMENT;
    if (a.row_bytes % 16 != 0 || a.row_stride % 16 != 0 || a.page_stride % 16 != 0 || a.page_stride <= 0) return PAT_ERR_UNSUPPORTED;
    if (a.rows > 1 && a.row_stride < a.row_bytes) return PAT_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(a.rows) * (a.row_bytes / 16) > 0x7fffffffLL - kThreads * kUnroll || a.num_pages > 0x7fffffffLL)
        return PAT_ERR_TOO_LARGE;
    for (int i = 0; i < a.num_caches; ++i)
        if (!a.caches[i] || (reinterpret_cast<uintptr_t>(a.caches[i]) & 15)) return PAT_ERR_UNSUPPORTED;
    if (a.host_pairs) {
        try {
            const int rc = check_pairs(a.host_pairs, a.num_pairs, a.num_pages);
            if (rc != PAT_OK) return rc;
        } catch (...) { return PAT_ERR_NO_MEMORY; }
    }
    cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
    return a.num_pairs <= kFewPairs || a.device_pairs ? launch_copies<kFewPairs>(a, stream) : launch_copies<kManyPairs>(a, stream);
}
