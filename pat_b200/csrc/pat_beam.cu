// Selection of the next beams from a step's logits (C ABI: pat_b200_beam_select).
//
// For batch entry b, beam k and token v:  value = score[b,k] + x[b,k,v] - log sum_v exp(x[b,k,v]);
// the num_out largest values of an entry, larger first, ties to the lower k * vocab + v.  (The
// reference has no sampling; its serving engine does that.)
//
// Two kernels.  beam_scan reads the logits once: a CTA takes 8192 consecutive logits of a row into
// registers, sums their exponentials against the chunk's maximum, and lists the chunk's num_out largest.
// Inside a beam the order of the values is the order of the logits, so the lists need no softmax.
// beam_pick has one CTA per entry: it joins the chunks' sums, and draws num_out times the largest of
// the heads of the lists.
//
// Candidates of different beams are compared by a value that contains two log-sums, so these are
// kept to about 1e-8: exponentials in fp32 with the argument in two parts, sums of at most 32 of them
// in fp32, everything above in fp64.  Which thread adds which logit depends on the index alone, not on
// where a row starts in memory: equal rows give equal sums, and equal candidates meet as ties.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/pat_b200.h"

namespace {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kGroups = 4;                         // groups of 8 consecutive logits per thread
constexpr int kPer = kGroups * 8;
constexpr int kChunk = kThreads * kPer;            // 8192
constexpr int kMaxOut = 128;
constexpr int kListCap = 1024;

struct BeamParams {
    const void* logits;
    const float* scores;
    const uint8_t* finished;       // optional
    int64_t batch_stride, beam_stride;             // elements
    int64_t score_stride, finished_stride;         // per batch entry
    float* out_scores;             // [batch, num_out]
    int32_t* out_parents;
    int32_t* out_tokens;
    // scratch, per (row, chunk): the chunk's largest logits in order, their number, its maximum and sum
    float* list_x;                 // [rows][chunks][num_out]
    int32_t* list_v;
    int32_t* list_n;               // [rows][chunks]
    float* chunk_max;
    double* chunk_sum;
    int batch, beams, vocab, num_out, chunks, pad_token;
};

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// exp(d) for d <= 0, argument d * log2(e) in two parts
__device__ __forceinline__ float exp_neg(float d) {
    constexpr float kHi = 1.44269502162933349609375f, kLo = 1.925963033500011e-08f;
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(d, kHi, d * kLo)));
    return y;
}

// a is preferred to b: larger value, or equal and lower index
__device__ __forceinline__ bool before(float xa, int ia, float xb, int ib) { return xa > xb || (xa == xb && ia < ib); }

// Eight consecutive logits from `at` on, by the widest loads the address allows.
template <typename T> __device__ __forceinline__ void load8(const T* at, float (&x)[8]) {
    constexpr int kBytes = 8 * sizeof(T);
    union { uint4 q[kBytes / 16]; uint32_t w[kBytes / 4]; T e[8]; } u;
    const uintptr_t a = reinterpret_cast<uintptr_t>(at);
    if ((a & 15) == 0) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) u.q[i] = __ldg(reinterpret_cast<const uint4*>(at) + i);
    } else if ((a & 3) == 0) {
#pragma unroll
        for (int i = 0; i < kBytes / 4; ++i) u.w[i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) u.e[i] = at[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float<T>(u.e[i]);
}

__device__ __forceinline__ bool beam_is_live(const BeamParams& p, int64_t b, int k) {
    if (p.finished && p.finished[b * p.finished_stride + k]) return false;
    return isfinite(p.scores[b * p.score_stride + k]);
}

template <typename T> __global__ void __launch_bounds__(kThreads) beam_scan_kernel(const BeamParams p) {
    const int64_t row = blockIdx.x / p.chunks;
    const int chunk = static_cast<int>(blockIdx.x - row * p.chunks);
    const int64_t b = row / p.beams;
    const int k = static_cast<int>(row - b * p.beams);
    if (!beam_is_live(p, b, k)) return;            // nobody reads this row's lists
    const T* src = static_cast<const T*>(p.logits) + b * p.batch_stride + static_cast<int64_t>(k) * p.beam_stride;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kWarps = kThreads / 32;
    __shared__ float s_top[kThreads];
    __shared__ float s_red[kWarps];
    __shared__ double s_sum[kWarps];
    __shared__ int s_bad, s_count;
    __shared__ float s_x[kListCap];
    __shared__ int s_v[kListCap];
    if (tid == 0) { s_bad = 0; s_count = 0; }

    // logits past the end of the row, and -inf ones, are no candidates and add nothing to the sum
    float x[kPer];
    const int base = chunk * kChunk;
#pragma unroll
    for (int gi = 0; gi < kGroups; ++gi) {
        const int at = base + gi * (kThreads * 8) + tid * 8;
        if (at + 8 <= p.vocab) {
            float y[8];
            load8<T>(src + at, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[gi * 8 + i] = y[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[gi * 8 + i] = at + i < p.vocab ? to_float<T>(src[at + i]) : -INFINITY;
        }
    }
    auto token_of = [&](int i) { return base + (i >> 3) * (kThreads * 8) + tid * 8 + (i & 7); };
    float top = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        top = fmaxf(top, x[i]);
        bad = bad || !(x[i] < INFINITY);           // NaN or +inf: the beam takes no part
    }
    s_top[tid] = top;
    float m = top;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, d));
    if (lane == 0) s_red[warp] = m;
    __syncthreads();
    if (__any_sync(kFull, bad) && lane == 0) s_bad = 1;
    m = s_red[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_red[w]);

    float sum = 0.f;
    if (m > -INFINITY) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += exp_neg(x[i] - m);
    }
    double total = sum;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(kFull, total, d);
    if (lane == 0) s_sum[warp] = total;

    // The num_out-th largest of the threads' maxima is a lower bound of the num_out-th largest logit:
    // only what reaches it can be among the num_out largest.
    int rank = 0;
    for (int i = 0; i < kThreads; ++i) {
        const float o = s_top[i];
        rank += (o > top || (o == top && i < tid)) ? 1 : 0;
    }
    __syncthreads();                               // (also: everyone has read s_red)
    if (rank == p.num_out - 1) s_red[0] = top;     // exactly one thread has this rank
    __syncthreads();
    const float edge = s_red[0];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (x[i] > -INFINITY && x[i] >= edge) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kListCap) { s_x[at] = x[i]; s_v[at] = token_of(i); }
        }
    }
    __syncthreads();
    const int found = s_count;
    const size_t slot = static_cast<size_t>(row) * p.chunks + chunk;
    float* out_x = p.list_x + slot * p.num_out;
    int32_t* out_v = p.list_v + slot * p.num_out;
    if (tid == 0) {
        double z = 0.0;
        for (int w = 0; w < kWarps; ++w) z += s_sum[w];
        p.chunk_max[slot] = s_bad ? NAN : m;
        p.chunk_sum[slot] = z;
        p.list_n[slot] = found < p.num_out ? found : p.num_out;
    }
    if (found <= kListCap) {
        for (int i = tid; i < found; i += kThreads) {
            const float xi = s_x[i];
            const int vi = s_v[i];
            int r = 0;
            for (int j = 0; j < found; ++j) r += before(s_x[j], s_v[j], xi, vi) ? 1 : 0;
            if (r < p.num_out) { out_x[r] = xi; out_v[r] = vi; }
        }
        return;
    }
    // Many equal logits: draw the largest remaining one num_out times.
    uint32_t taken = 0;
    for (int n = 0; n < p.num_out; ++n) {
        float bx = -INFINITY;
        int bv = 0x7fffffff, bi = -1;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const bool open = !((taken >> i) & 1u) && x[i] > -INFINITY;
            if (open && before(x[i], token_of(i), bx, bv)) { bx = x[i]; bv = token_of(i); bi = i; }
        }
        float wx = bx;
        int wv = bv;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const float ox = __shfl_xor_sync(kFull, wx, d);
            const int ov = __shfl_xor_sync(kFull, wv, d);
            if (before(ox, ov, wx, wv)) { wx = ox; wv = ov; }
        }
        if (lane == 0) { s_x[warp] = wx; s_v[warp] = wv; }
        __syncthreads();
        wx = s_x[0];
        wv = s_v[0];
        for (int w = 1; w < kWarps; ++w)
            if (before(s_x[w], s_v[w], wx, wv)) { wx = s_x[w]; wv = s_v[w]; }
        if (bi >= 0 && bv == wv) { taken |= 1u << bi; out_x[n] = wx; out_v[n] = wv; }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kThreads) beam_pick_kernel(const BeamParams p) {
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kWarps = kThreads / 32;
    const int lists = p.beams * p.chunks;          // heads of all lists, plus one entry per finished beam
    extern __shared__ double s_shift[];            // [beams] score - log-sum, or NaN: the beam takes no part
    int* s_cursor = reinterpret_cast<int*>(s_shift + p.beams);      // [lists]
    __shared__ double s_val[kWarps];
    __shared__ int64_t s_idx[kWarps];
    __shared__ int s_list[kWarps];
    __shared__ int64_t s_chosen[kMaxOut];

    for (int k = tid; k < p.beams; k += kThreads) {
        double shift = NAN;
        if (beam_is_live(p, b, k)) {
            const size_t slot = (static_cast<size_t>(b) * p.beams + k) * p.chunks;
            float m = -INFINITY;
            bool bad = false;
            for (int c = 0; c < p.chunks; ++c) {
                const float cm = p.chunk_max[slot + c];
                bad = bad || cm != cm;
                m = fmaxf(m, cm);
            }
            if (!bad && m > -INFINITY) {
                double z = 0.0;
                for (int c = 0; c < p.chunks; ++c) {
                    const float cm = p.chunk_max[slot + c];
                    if (cm > -INFINITY) z += p.chunk_sum[slot + c] * exp(static_cast<double>(cm) - static_cast<double>(m));
                }
                shift = static_cast<double>(p.scores[b * p.score_stride + k]) - (static_cast<double>(m) + log(z));
            }
        }
        s_shift[k] = shift;
    }
    for (int i = tid; i < lists; i += kThreads) s_cursor[i] = 0;
    __syncthreads();

    int n = 0;
    for (; n < p.num_out; ++n) {
        double best = -INFINITY;
        int64_t best_idx = INT64_MAX;
        int best_list = -1;
        for (int i = tid; i < lists; i += kThreads) {
            const int k = i / p.chunks, c = i - k * p.chunks;
            double val;
            int64_t idx;
            const bool done = p.finished && p.finished[b * p.finished_stride + k];
            if (done) {
                if (c != 0 || s_cursor[i] > 0) continue;
                const float sc = p.scores[b * p.score_stride + k];
                if (!isfinite(sc)) continue;
                val = sc;
                idx = static_cast<int64_t>(k) * p.vocab + p.pad_token;
            } else {
                const double shift = s_shift[k];
                const size_t slot = (static_cast<size_t>(b) * p.beams + k) * p.chunks + c;
                if (shift != shift || s_cursor[i] >= p.list_n[slot]) continue;
                val = shift + static_cast<double>(p.list_x[slot * p.num_out + s_cursor[i]]);
                idx = static_cast<int64_t>(k) * p.vocab + p.list_v[slot * p.num_out + s_cursor[i]];
            }
            if (val > best || (val == best && idx < best_idx)) { best = val; best_idx = idx; best_list = i; }
        }
        double wv = best;
        int64_t wi = best_idx;
        int wl = best_list;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const double ov = __shfl_xor_sync(kFull, wv, d);
            const int64_t oi = __shfl_xor_sync(kFull, wi, d);
            const int ol = __shfl_xor_sync(kFull, wl, d);
            if (ov > wv || (ov == wv && oi < wi)) { wv = ov; wi = oi; wl = ol; }
        }
        if (lane == 0) { s_val[warp] = wv; s_idx[warp] = wi; s_list[warp] = wl; }
        __syncthreads();
        wv = s_val[0]; wi = s_idx[0]; wl = s_list[0];
        for (int w = 1; w < kWarps; ++w)
            if (s_val[w] > wv || (s_val[w] == wv && s_idx[w] < wi)) { wv = s_val[w]; wi = s_idx[w]; wl = s_list[w]; }
        if (wl < 0) break;                         // uniform: nothing finite is left
        if (tid == 0) {
            s_cursor[wl] += 1;
            s_chosen[n] = wi;
            p.out_scores[b * p.num_out + n] = static_cast<float>(wv);
            p.out_parents[b * p.num_out + n] = static_cast<int32_t>(wi / p.vocab);
            p.out_tokens[b * p.num_out + n] = static_cast<int32_t>(wi % p.vocab);
        }
        __syncthreads();
    }
    // Fewer finite values than asked for: the rest are -inf, all equal, so the lowest indices not
    // chosen yet follow.  Every finite value of the entry has been chosen by now.
    if (n < p.num_out && tid == 0) {
        const int finite = n;
        for (int64_t idx = 0; n < p.num_out; ++idx) {
            bool used = false;
            for (int i = 0; i < finite; ++i) used = used || s_chosen[i] == idx;
            if (used) continue;
            p.out_scores[b * p.num_out + n] = -INFINITY;
            p.out_parents[b * p.num_out + n] = static_cast<int32_t>(idx / p.vocab);
            p.out_tokens[b * p.num_out + n] = static_cast<int32_t>(idx % p.vocab);
            ++n;
        }
    }
}

int beam_shape(int batch, int beams, int vocab, int num_out) {
    if (batch < 0 || beams <= 0 || vocab <= 0 || num_out <= 0) return PAT_ERR_BAD_ARGUMENT;
    if (num_out > static_cast<int64_t>(beams) * vocab) return PAT_ERR_BAD_ARGUMENT;
    if (num_out > kMaxOut || beams > 512) return PAT_ERR_TOO_LARGE;
    const int64_t chunks = (static_cast<int64_t>(vocab) + kChunk - 1) / kChunk;
    if (static_cast<int64_t>(beams) * chunks > 8192 || static_cast<int64_t>(batch) * beams * chunks > 0x7fffffffLL) return PAT_ERR_TOO_LARGE;
    return PAT_OK;
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

extern "C" size_t pat_b200_beam_workspace_bytes(int batch, int beams, int vocab, int num_out) {
    if (beam_shape(batch, beams, vocab, num_out) != PAT_OK) return 0;
    const size_t lists = static_cast<size_t>(batch) * beams * ((static_cast<size_t>(vocab) + kChunk - 1) / kChunk);
    return 2 * align256(lists * num_out * 4) + 2 * align256(lists * 4) + align256(lists * 8);
}

extern "C" int pat_b200_beam_select(const pat_beam_args* args, void* stream_handle) {
    if (!args) return PAT_ERR_BAD_ARGUMENT;
    const pat_beam_args& a = *args;
    const int rc = beam_shape(a.batch, a.beams, a.vocab, a.num_out);
    if (rc != PAT_OK) return rc;
    if (a.batch == 0) return PAT_OK;
    if (!a.logits || !a.scores || !a.out_scores || !a.out_parents || !a.out_tokens) return PAT_ERR_BAD_ARGUMENT;
    if (a.pad_token < 0 || a.pad_token >= a.vocab) return PAT_ERR_BAD_ARGUMENT;
    if (a.dtype != PAT_DTYPE_FP16 && a.dtype != PAT_DTYPE_BF16 && a.dtype != PAT_DTYPE_FP32) return PAT_ERR_UNSUPPORTED;
    if (reinterpret_cast<uintptr_t>(a.logits) & (a.dtype == PAT_DTYPE_FP32 ? 3 : 1)) return PAT_ERR_UNSUPPORTED;
    if (!a.workspace || a.workspace_bytes < pat_b200_beam_workspace_bytes(a.batch, a.beams, a.vocab, a.num_out) ||
        (reinterpret_cast<uintptr_t>(a.workspace) & 15))
        return PAT_ERR_WORKSPACE;
    BeamParams p{};
    p.logits = a.logits;
    p.scores = a.scores;
    p.finished = a.finished;
    p.batch_stride = a.logits_batch_stride;
    p.beam_stride = a.logits_beam_stride;
    p.score_stride = a.scores_batch_stride;
    p.finished_stride = a.finished_batch_stride;
    p.out_scores = a.out_scores;
    p.out_parents = a.out_parents;
    p.out_tokens = a.out_tokens;
    p.batch = a.batch;
    p.beams = a.beams;
    p.vocab = a.vocab;
    p.num_out = a.num_out;
    p.pad_token = a.pad_token;
    p.chunks = static_cast<int>((static_cast<int64_t>(a.vocab) + kChunk - 1) / kChunk);
    const size_t lists = static_cast<size_t>(a.batch) * a.beams * p.chunks;
    unsigned char* ws = static_cast<unsigned char*>(a.workspace);
    p.chunk_sum = reinterpret_cast<double*>(ws);
    ws += align256(lists * 8);
    p.list_x = reinterpret_cast<float*>(ws);
    ws += align256(lists * a.num_out * 4);
    p.list_v = reinterpret_cast<int32_t*>(ws);
    ws += align256(lists * a.num_out * 4);
    p.list_n = reinterpret_cast<int32_t*>(ws);
    ws += align256(lists * 4);
    p.chunk_max = reinterpret_cast<float*>(ws);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
    const unsigned grid = static_cast<unsigned>(lists);
    if (a.dtype == PAT_DTYPE_FP32) beam_scan_kernel<float><<<grid, kThreads, 0, stream>>>(p);
    else if (a.dtype == PAT_DTYPE_BF16) beam_scan_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
    else beam_scan_kernel<__half><<<grid, kThreads, 0, stream>>>(p);
    const size_t smem = static_cast<size_t>(a.beams) * 8 + static_cast<size_t>(a.beams) * p.chunks * 4;   // <= 36 KB by beam_shape
    beam_pick_kernel<<<static_cast<unsigned>(a.batch), kThreads, smem, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? PAT_OK : PAT_ERR_CUDA;
}
