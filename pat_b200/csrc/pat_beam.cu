// Selection of the next beams from a step's logits (C ABI: pat_b200_beam_select).
//
// For batch entry b, beam k and token v:  value = score[b,k] + x[b,k,v] - log sum_v exp(x[b,k,v]);
// the num_out largest values of an entry, larger first, ties to the lower k * vocab + v.  (The
// reference has no sampling; its serving engine does that.)
//
// Two kernels.  beam_scan reads the logits once: a CTA takes up to 8192 consecutive logits of a row into
// registers, sums their exponentials against the chunk's maximum, and lists the chunk's num_out largest.
// Inside a beam the order of the values is the order of the logits, so the lists need no softmax.
// beam_pick, its programmatic dependent, has one CTA per entry: it joins the chunks' sums and picks the
// num_out best of the lists.  Both find a lower bound of the num_out-th largest from the threads' maxima -
// every warp sorts its 32 - collect the few that reach it, and order those by counting.
//
// Candidates of different beams are compared by a value that contains two log-sums, so these are
// kept to about 1e-8: exponentials in fp32 with log2(e) in two parts, sums of at most 32 of them
// in fp32, everything above in fp64.  Which thread adds which logit depends on the index alone, not on
// where a row starts in memory: equal rows give equal sums, and equal candidates meet as ties.
//
// 32 x 8 beams x 128000 fp32 logits (131 MB), 16 candidates: beam_scan 41.6 us = 3.2 TB/s, bound by its instructions per
// logit (maximum, exponential, comparison with the bound) and by the waits between its passes, not by memory; beam_pick
// 12 us behind it, one CTA per entry ordering up to 4096 lists' heads: latency.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/pat_b200.h"

namespace {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxGroups = 4;                      // groups of 8 consecutive logits per thread
constexpr int kMaxOut = 128;
constexpr int kMaxBeams = 512;
static_assert(2 * kMaxOut == kThreads, "s_used is cleared by one store per thread");
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
    // scratch, per (row, chunk): the chunk's largest logits in order, their number, its sum
    float* list_x;                 // [rows][chunks][num_out]
    int32_t* list_v;
    int32_t* list_n;               // [rows][chunks]
    float* chunk_ref;              // largest logit, which the sum is relative to; +inf: NaN or +inf seen, -inf: nothing but -inf
    double* chunk_sum;
    int batch, beams, vocab, num_out, chunks, chunk_len, pad_token;
};

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// e^d of a difference d <= 0, log2(e) in two parts.  The difference to the maximum is rounded, not the two logits times
// log2(e): logits of any finite size keep their sum (a difference d's rounding weighs e^d d 2^-24), and -3e38 beside
// 3e38 becomes -inf.
constexpr float kLog2eHi = 1.44269502162933349609375f, kLog2eLo = 1.925963033500011e-08f;
__device__ __forceinline__ float exp_below(float d) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(d, kLog2eHi, d * kLog2eLo)));
    return y;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
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

// The values of the warp's lanes in descending order (bitonic sort): lane i gets the (i + 1)-th largest.
__device__ __forceinline__ float warp_sorted(float v, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
        for (int d = size / 2; d > 0; d >>= 1) {
            const float o = __shfl_xor_sync(kFull, v, d);
            const bool keep_max = ((lane & size) == 0) == ((lane & d) == 0);
            v = keep_max ? fmaxf(v, o) : fminf(v, o);
        }
    }
    return v;
}

template <typename T, int kGroups> __global__ void __launch_bounds__(kThreads, 5) beam_scan_kernel(const BeamParams p) {
    constexpr int kPer = kGroups * 8;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int64_t row = blockIdx.x / p.chunks;
    const int chunk = static_cast<int>(blockIdx.x - row * p.chunks);
    const int64_t b = row / p.beams;
    const int k = static_cast<int>(row - b * p.beams);
    if (!beam_is_live(p, b, k)) return;            // nobody reads this row's lists
    const T* src = static_cast<const T*>(p.logits) + b * p.batch_stride + static_cast<int64_t>(k) * p.beam_stride;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    __shared__ float s_max[kWarps], s_edge[kWarps];
    __shared__ double s_sum[kWarps];
    __shared__ int s_count;
    __shared__ float s_x[kListCap];
    __shared__ int s_v[kListCap];
    if (tid == 0) s_count = 0;

    // logits past the end of the chunk, and -inf ones, are no candidates and add nothing to the sum
    float x[kPer];
    const int base = chunk * p.chunk_len, end = min(base + p.chunk_len, p.vocab);
#pragma unroll
    for (int gi = 0; gi < kGroups; ++gi) {
        const int at = base + gi * (kThreads * 8) + tid * 8;
        if (at + 8 <= end) {
            float y[8];
            load8<T>(src + at, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[gi * 8 + i] = y[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[gi * 8 + i] = at + i < end ? to_float<T>(src[at + i]) : -INFINITY;
        }
    }
    auto token_of = [&](int i) { return base + (i >> 3) * (kThreads * 8) + tid * 8 + (i & 7); };
    float group[kGroups], top = -INFINITY;
#pragma unroll
    for (int gi = 0; gi < kGroups; ++gi) {
        group[gi] = x[gi * 8];
#pragma unroll
        for (int i = 1; i < 8; ++i) group[gi] = max_or_nan(group[gi], x[gi * 8 + i]);
        top = max_or_nan(top, group[gi]);
    }
    // At least q of every warp's maxima reach `edge`, so at least num_out logits of the chunk do.
    const int q = (p.num_out + kWarps - 1) / kWarps;
    const bool bad = __any_sync(kFull, !(top < INFINITY));      // NaN or +inf: the beam takes no part
    const float sorted = warp_sorted(top, lane);
    if (lane == 0) s_max[warp] = bad ? INFINITY : sorted;
    if (lane == q - 1) s_edge[warp] = sorted;
    __syncthreads();
    float m = s_max[0], edge = s_edge[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) { m = fmaxf(m, s_max[w]); edge = fminf(edge, s_edge[w]); }
    const size_t slot = static_cast<size_t>(row) * p.chunks + chunk;
    if (!(m < INFINITY) || m == -INFINITY) {       // uniform: nothing to sum, nothing to list
        if (tid == 0) {
            p.chunk_ref[slot] = m;                 // +inf: bad, -inf: empty
            p.list_n[slot] = 0;
        }
        return;
    }

    float sum = 0.f;
#pragma unroll
    for (int gi = 0; gi < kGroups; ++gi) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += exp_below(x[gi * 8 + i] - m);
        if (group[gi] >= edge && group[gi] > -INFINITY) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (x[gi * 8 + i] >= edge && x[gi * 8 + i] > -INFINITY) {
                    const int at = atomicAdd(&s_count, 1);
                    if (at < kListCap) { s_x[at] = x[gi * 8 + i]; s_v[at] = token_of(gi * 8 + i); }
                }
            }
        }
    }
    double total = sum;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(kFull, total, d);
    if (lane == 0) s_sum[warp] = total;
    __syncthreads();
    const int found = s_count;
    float* out_x = p.list_x + slot * p.num_out;
    int32_t* out_v = p.list_v + slot * p.num_out;
    if (tid == 0) {
        double z = 0.0;
        for (int w = 0; w < kWarps; ++w) z += s_sum[w];
        p.chunk_ref[slot] = m;
        p.chunk_sum[slot] = z;
        p.list_n[slot] = found < p.num_out ? found : p.num_out;
    }
    if (found <= kListCap) {
        // place of a candidate = how many are preferred to it; four threads count for each
        for (int i0 = 0; i0 < found; i0 += kThreads / 4) {
            const int i = i0 + tid / 4;
            const float xi = i < found ? s_x[i] : 0.f;
            const int vi = i < found ? s_v[i] : 0;
            int r = 0;
            for (int j = tid & 3; j < found; j += 4) r += before(s_x[j], s_v[j], xi, vi) ? 1 : 0;
            r += __shfl_xor_sync(kFull, r, 1);
            r += __shfl_xor_sync(kFull, r, 2);
            if ((tid & 3) == 0 && i < found && r < p.num_out) { out_x[r] = xi; out_v[r] = vi; }
        }
        return;
    }
    // Very many equal logits, or maxima in few warps only: draw the largest remaining one num_out times.
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
        __syncthreads();                           // (everyone has read the lists / the last round)
        if (lane == 0) { s_x[warp] = wx; s_v[warp] = wv; }
        __syncthreads();
        wx = s_x[0];
        wv = s_v[0];
        for (int w = 1; w < kWarps; ++w)
            if (before(s_x[w], s_v[w], wx, wv)) { wx = s_x[w]; wv = s_v[w]; }
        if (bi >= 0 && bv == wv) { taken |= 1u << bi; out_x[n] = wx; out_v[n] = wv; }
    }
}

__device__ __forceinline__ bool before(double xa, int64_t ia, double xb, int64_t ib) { return xa > xb || (xa == xb && ia < ib); }

__global__ void __launch_bounds__(kThreads) beam_pick_kernel(const BeamParams p) {
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    __shared__ double s_shift[kMaxBeams];          // score - log(sum); NaN: the beam takes no part
    __shared__ float s_top[kMaxBeams];             // largest logit
    __shared__ float s_edge[kWarps];
    __shared__ double s_val[kListCap];
    __shared__ int64_t s_idx[kListCap];
    __shared__ int s_count;
    __shared__ uint8_t s_used[2 * kMaxOut];
    if (tid == 0) s_count = 0;
    s_used[tid] = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // log-sum of every beam: its largest logit + log(sum)
    for (int k = warp; k < p.beams; k += kWarps) {
        double shift = NAN;
        float m = -INFINITY;
        if (beam_is_live(p, b, k)) {
            const size_t slot = (static_cast<size_t>(b) * p.beams + k) * p.chunks;
            for (int c = lane; c < p.chunks; c += 32) m = fmaxf(m, p.chunk_ref[slot + c]);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, d));
            if (m < INFINITY && m > -INFINITY) {
                double z = 0.0;
                for (int c = lane; c < p.chunks; c += 32) {
                    const float ref = p.chunk_ref[slot + c];
                    if (ref > -INFINITY) z += p.chunk_sum[slot + c] * exp(static_cast<double>(ref) - static_cast<double>(m));
                }
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) z += __shfl_xor_sync(kFull, z, d);
                shift = static_cast<double>(p.scores[b * p.score_stride + k]) - log(z);
            }
        }
        if (lane == 0) { s_shift[k] = shift; s_top[k] = m; }
    }
    __syncthreads();

    // Candidates: the places of all lists, then one candidate per finished beam.
    const int lists = p.beams * p.chunks;
    const int shift_out = 32 - __clz(p.num_out - 1 | 1);       // places per list, rounded up to a power of two
    const int total = (lists << shift_out) + (p.finished ? p.beams : 0);
    const float* my_x = p.list_x + static_cast<size_t>(b) * lists * p.num_out;
    const int32_t* my_v = p.list_v + static_cast<size_t>(b) * lists * p.num_out;
    auto value_of = [&](int j) -> double {                     // -inf: no candidate
        const int list = j >> shift_out, pos = j & ((1 << shift_out) - 1);
        if (list < lists) {
            if (pos >= p.num_out) return -INFINITY;
            const float x = my_x[list * p.num_out + pos];      // (may hold anything behind the list's end)
            const int n = p.list_n[static_cast<size_t>(b) * lists + list];
            const double shift = s_shift[list / p.chunks];
            return pos < n && shift == shift ? shift + (static_cast<double>(x) - static_cast<double>(s_top[list / p.chunks])) : -INFINITY;
        }
        const int k = j - (lists << shift_out);
        const float score = p.scores[b * p.score_stride + k];
        return p.finished[b * p.finished_stride + k] && isfinite(score) ? static_cast<double>(score) : -INFINITY;
    };
    auto index_of = [&](int j) -> int64_t {
        const int list = j >> shift_out, pos = j & ((1 << shift_out) - 1);
        if (list < lists) return static_cast<int64_t>(list / p.chunks) * p.vocab + my_v[list * p.num_out + pos];
        return static_cast<int64_t>(j - (lists << shift_out)) * p.vocab + p.pad_token;
    };
    // the first kKeep values of every thread stay in registers between the two passes
    constexpr int kKeep = 8;
    double kept[kKeep];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
        const int j = tid + i * kThreads;
        kept[i] = j < total ? value_of(j) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < kKeep; ++i) top = fmaxf(top, __double2float_rd(kept[i]));
    for (int j = tid + kKeep * kThreads; j < total; j += kThreads) top = fmaxf(top, __double2float_rd(value_of(j)));
    const float sorted = warp_sorted(top, lane);
    if (lane == (p.num_out + kWarps - 1) / kWarps - 1) s_edge[warp] = sorted;
    __syncthreads();
    float edge = s_edge[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) edge = fminf(edge, s_edge[w]);
    auto collect = [&](int j, double val) {
        if (val > -INFINITY && val >= static_cast<double>(edge)) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kListCap) { s_val[at] = val; s_idx[at] = index_of(j); }
        }
    };
#pragma unroll
    for (int i = 0; i < kKeep; ++i) collect(tid + i * kThreads, kept[i]);
    for (int j = tid + kKeep * kThreads; j < total; j += kThreads) collect(j, value_of(j));
    __syncthreads();
    const int found = s_count;
    auto put = [&](int n, double v, int64_t i) {
        p.out_scores[b * p.num_out + n] = static_cast<float>(v);
        p.out_parents[b * p.num_out + n] = static_cast<int32_t>(i / p.vocab);
        p.out_tokens[b * p.num_out + n] = static_cast<int32_t>(i % p.vocab);
    };
    if (found <= kListCap) {
        for (int i0 = 0; i0 < found; i0 += kThreads / 4) {
            const int i = i0 + tid / 4;
            const double vi = i < found ? s_val[i] : 0.0;
            const int64_t ii = i < found ? s_idx[i] : 0;
            int r = 0;
            for (int j = tid & 3; j < found; j += 4) r += before(s_val[j], s_idx[j], vi, ii) ? 1 : 0;
            r += __shfl_xor_sync(kFull, r, 1);
            r += __shfl_xor_sync(kFull, r, 2);
            if ((tid & 3) == 0 && i < found) {
                if (r < p.num_out) put(r, vi, ii);
                if (ii < 2 * kMaxOut) s_used[ii] = 1;
            }
        }
        if (found >= p.num_out) return;
        // Fewer finite values than asked for, and all of them are listed: the rest are -inf, all equal, so the
        // lowest indices not among the listed follow.  They lie below num_out + found < 2 kMaxOut.
        __syncthreads();
        if (tid == 0)
            for (int64_t i = 0, n = found; n < p.num_out; ++i)
                if (!s_used[i]) put(static_cast<int>(n++), -INFINITY, i);
        return;
    }
    // Very many equal values: num_out times the best behind the last one chosen.
    double last = INFINITY;
    int64_t last_idx = -1;
    for (int n = 0; n < p.num_out; ++n) {
        double best = -INFINITY;
        int64_t best_idx = INT64_MAX;
        for (int j = tid; j < total; j += kThreads) {
            const double val = value_of(j);
            if (val == -INFINITY || !(val < last || (val == last && index_of(j) > last_idx))) continue;
            const int64_t idx = index_of(j);
            if (before(val, idx, best, best_idx)) { best = val; best_idx = idx; }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const double ov = __shfl_xor_sync(kFull, best, d);
            const int64_t oi = __shfl_xor_sync(kFull, best_idx, d);
            if (before(ov, oi, best, best_idx)) { best = ov; best_idx = oi; }
        }
        __syncthreads();
        if (lane == 0) { s_val[warp] = best; s_idx[warp] = best_idx; }
        __syncthreads();
        last = s_val[0];
        last_idx = s_idx[0];
        for (int w = 1; w < kWarps; ++w)
            if (before(s_val[w], s_idx[w], last, last_idx)) { last = s_val[w]; last_idx = s_idx[w]; }
        if (tid == 0) put(n, last, last_idx);
    }
}

// How a row is cut.  8192 logits per CTA keep 4 x 16 bytes (or more) of every thread in flight, and lists
// few; with less than two CTAs per SM then, shorter chunks spread the rows over more SMs.
struct Cut { int groups, chunks, chunk_len; };
Cut cut_rows(int64_t rows, int vocab) {
    Cut c{kMaxGroups, 0, 0};
    while (true) {
        const int64_t len = static_cast<int64_t>(c.groups) * kThreads * 8;
        const int64_t chunks = (vocab + len - 1) / len;
        if (c.groups > 1 && rows * chunks < 2 * 148) { c.groups /= 2; continue; }
        c.chunks = static_cast<int>(chunks);
        c.chunk_len = static_cast<int>(((vocab + chunks - 1) / chunks + 7) / 8 * 8);       // chunks of equal length
        c.chunks = (vocab + c.chunk_len - 1) / c.chunk_len;
        return c;
    }
}

int beam_shape(int batch, int beams, int vocab, int num_out) {
    if (batch < 0 || beams <= 0 || vocab <= 0 || num_out <= 0) return PAT_ERR_BAD_ARGUMENT;
    if (num_out > static_cast<int64_t>(beams) * vocab) return PAT_ERR_BAD_ARGUMENT;
    if (num_out > kMaxOut || beams > kMaxBeams || vocab > (1 << 24)) return PAT_ERR_TOO_LARGE;
    const int64_t rows = static_cast<int64_t>(batch) * beams;
    const int64_t chunks = cut_rows(rows, vocab).chunks;
    if (rows * chunks > 0x7fffffffLL || beams * chunks * kMaxOut > 0x3fffffffLL) return PAT_ERR_TOO_LARGE;
    return PAT_OK;
}

template <typename T> void (*scan_of(int groups))(BeamParams) {
    return groups == 4 ? beam_scan_kernel<T, 4> : groups == 2 ? beam_scan_kernel<T, 2> : beam_scan_kernel<T, 1>;
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

extern "C" size_t pat_b200_beam_workspace_bytes(int batch, int beams, int vocab, int num_out) {
    if (beam_shape(batch, beams, vocab, num_out) != PAT_OK) return 0;
    const int64_t rows = static_cast<int64_t>(batch) * beams;
    const size_t lists = static_cast<size_t>(rows) * cut_rows(rows, vocab).chunks;
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
    const Cut cut = cut_rows(static_cast<int64_t>(a.batch) * a.beams, a.vocab);
    p.chunks = cut.chunks;
    p.chunk_len = cut.chunk_len;
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
    p.chunk_ref = reinterpret_cast<float*>(ws);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
    const unsigned grid = static_cast<unsigned>(lists);
    void (*scan)(BeamParams);
    if (a.dtype == PAT_DTYPE_FP32) scan = scan_of<float>(cut.groups);
    else if (a.dtype == PAT_DTYPE_BF16) scan = scan_of<__nv_bfloat16>(cut.groups);
    else scan = scan_of<__half>(cut.groups);
    scan<<<grid, kThreads, 0, stream>>>(p);
    // starts while the scan runs, and waits for its end before it reads anything the scan wrote
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.batch));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, beam_pick_kernel, p) != cudaSuccess) return PAT_ERR_CUDA;
    return cudaGetLastError() == cudaSuccess ? PAT_OK : PAT_ERR_CUDA;
}
