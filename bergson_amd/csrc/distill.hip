// Distillation from a teacher's highest logits: per token the divergence of the student's distribution over the
// whole vocabulary from the teacher's over its K kept entries, and its gradient.
//
//   p = softmax_k(t_k / tau) over the entries with 0 <= id < V,  q = softmax_v(z_v / tau)
//   loss = tau^2 sum_k p_k (log p_k - log q_{id_k}),  dz_v = g tau (q_v - sum_{k: id_k = v} p_k)
//
// Bound by the logits: the forward pass reads them once (running maximum and sum per thread, joined at the row's
// end), the backward pass reads them once and writes their gradient; the K entries are a few hundred bytes.  The
// forward pass keeps a row's maximum and sum of exponentials apart rather than as one logarithm: a gradient then
// carries the rounding of z - max, not that of a logarithm of the size of the logits.  All sums in fp32.
//
// Measured on 4096 x 50304 bf16 logits, 64 entries: forward 76 us after a backward pass, 70 us alone (0.41 GB: 5.4 and
// 5.9 TB/s), backward 152 us (0.82 GB: 5.4 TB/s).  One workgroup per row: of 256 threads, or of 1024 below DISTILL_FEW rows,
// where a row's walk is the whole time (3 x 50257 fp32: forward 8.2 -> 6.5 us, backward 8.6 -> 7.4).
#include "rows.hpp"

namespace bgx {

constexpr int DISTILL_MAX_K = 1024;
constexpr int DISTILL_FEW = 512;
constexpr int DEEP = 4;  // chunks a thread has on their way at once

struct DistillArgs {
  const void* logits;
  const int64_t* ids;       // [rows, K]
  const void* teacher;      // [rows, K]
  const uint8_t* valid;     // [rows] or NULL
  float* losses;            // [rows]
  float* stats;             // [rows, 2]: maximum of z, sum of exp((z - max) / tau)
  const float* grad;        // [rows]
  void* dlogits;
  int64_t rows, stride, dstride;
  int V, K;
  int teacher_dtype;
  float tau;
};

template <int THREADS>
__device__ inline float block_sum(float v, float* slot) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & (WAVE - 1)) == 0) slot[threadIdx.x / WAVE] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / WAVE; ++i) s += slot[i];
  return s;
}
template <int THREADS>
__device__ inline float block_max(float v, float* slot) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & (WAVE - 1)) == 0) slot[threadIdx.x / WAVE] = v;
  __syncthreads();
  float s = slot[0];
#pragma unroll
  for (int i = 1; i < THREADS / WAVE; ++i) s = fmaxf(s, slot[i]);
  return s;
}

constexpr float LOG2E = 1.4426950408889634f;

// 2^x; x = -inf gives 0
__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The teacher's distribution of a row into LDS: prob[k], and id[k] = -1 for entries that are none.  Returns whether
// the row has any entry with a finite weight.  Ends with the values visible to the whole workgroup.
template <int THREADS>
__device__ inline bool teacher_row(const DistillArgs& A, int64_t r, int* id, float* prob, float* slot, float& t_max,
                                   float& t_sum) {
  const int64_t* ids = A.ids + r * A.K;
  float m = -INFINITY, bad = 0.f;
  for (int k = threadIdx.x; k < A.K; k += THREADS) {
    const int64_t i = ids[k];
    const bool in = i >= 0 && i < A.V;
    const float t = in ? load_as(A.teacher, r * A.K + k, A.teacher_dtype) : -INFINITY;
    id[k] = in ? (int)i : -1;
    prob[k] = t;
    m = fmaxf(m, t);
    bad = t != t ? 1.f : bad;
  }
  t_max = block_max<THREADS>(m, slot);
  if (block_max<THREADS>(bad, slot) != 0.f) t_max = NAN;  // the maximum alone drops a NaN entry
  float s = 0.f;
  const float c = LOG2E / A.tau;
  for (int k = threadIdx.x; k < A.K; k += THREADS) {
    const float e = id[k] < 0 ? 0.f : exp2_hw((prob[k] - t_max) * c);
    s += e;
  }
  t_sum = block_sum<THREADS>(s, slot);
  return t_max != -INFINITY;
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void distill_forward_kernel(DistillArgs A) {
  constexpr int EPL = Chunk<T>::N;
  __shared__ float slot[THREADS / WAVE];
  __shared__ int id[DISTILL_MAX_K];
  __shared__ float prob[DISTILL_MAX_K];
  const int64_t r = blockIdx.x;
  float t_max, t_sum;
  const bool used = (A.valid == nullptr || A.valid[r] != 0) && teacher_row<THREADS>(A, r, id, prob, slot, t_max, t_sum);
  if (!used) {
    if (threadIdx.x == 0) {
      A.losses[r] = 0.f;
      if (A.stats != nullptr) {
        A.stats[2 * r] = 0.f;
        A.stats[2 * r + 1] = -1.f;  // no sum of exponentials is negative: the row takes no part
      }
    }
    return;
  }
  const T* z = (const T*)A.logits + r * A.stride;
  const float c = LOG2E / A.tau;
  float m = -INFINITY, s = 0.f;
  auto take = [&](const float* v, auto count) {
    float top = m;
#pragma unroll
    for (int e = 0; e < count; ++e) top = fmaxf(top, v[e]);  // drops NaN; the sum keeps it
    if (top > m) {
      s *= exp2_hw((m - top) * c);
      m = top;
    }
    // nothing but -inf so far: weights of 0.  The difference first: m c may leave the numbers where m does not.
    const float shift = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < count; ++e) s += exp2_hw((v[e] - shift) * c);
  };
  const int chunks = A.V / EPL;  // whole ones; the row's last elements go one by one
  int i = threadIdx.x;
  for (; i + (DEEP - 1) * THREADS < chunks; i += DEEP * THREADS) {
    uint4 w[DEEP];
    float v[DEEP * EPL];
#pragma unroll
    for (int k = 0; k < DEEP; ++k) w[k] = load_chunk_any(z + (int64_t)(i + k * THREADS) * EPL);
#pragma unroll
    for (int k = 0; k < DEEP; ++k) Chunk<T>::unpack(w[k], v + k * EPL);
    take(v, std::integral_constant<int, DEEP * EPL>());
  }
  for (; i < chunks; i += THREADS) {
    float v[EPL];
    Chunk<T>::unpack(load_chunk_any(z + (int64_t)i * EPL), v);
    take(v, std::integral_constant<int, EPL>());
  }
  if ((int)threadIdx.x < A.V - chunks * EPL) {
    const float v = Elem<T>::load(z + (int64_t)chunks * EPL + threadIdx.x);
    take(&v, std::integral_constant<int, 1>());
  }
  const float top = block_max<THREADS>(m, slot);
  s = block_sum<THREADS>(m == -INFINITY ? s : s * exp2_hw((m - top) * c), slot);
  const float log_s = logf(s), log_t = logf(t_sum), inv_tau = 1.f / A.tau;
  float loss = 0.f;
  for (int k = threadIdx.x; k < A.K; k += THREADS) {
    if (id[k] < 0) continue;
    const float log_p = (prob[k] - t_max) * inv_tau - log_t;
    const float p = exp2_hw((prob[k] - t_max) * c) / t_sum;
    const float log_q = (Elem<T>::load(z + id[k]) - top) * inv_tau - log_s;
    if (p != 0.f) loss += p * (log_p - log_q);  // 0 log 0 = 0, whatever the student gives the entry
  }
  loss = block_sum<THREADS>(loss, slot);
  if (threadIdx.x == 0) {
    A.losses[r] = A.tau * A.tau * loss;
    if (A.stats != nullptr) {
      A.stats[2 * r] = top;
      A.stats[2 * r + 1] = s;
    }
  }
}

template <typename T, int THREADS, bool STREAM>
__global__ __launch_bounds__(THREADS) void distill_backward_kernel(DistillArgs A) {
  constexpr int EPL = Chunk<T>::N;
  __shared__ float slot[THREADS / WAVE];
  __shared__ int id[DISTILL_MAX_K];
  __shared__ float prob[DISTILL_MAX_K];
  __shared__ int head[DISTILL_MAX_K], next[DISTILL_MAX_K];  // entries by the low bits of their ids, in lists
  // from the last row on: what the forward pass read last may still be in the memory-side cache
  const int64_t r = A.rows - 1 - blockIdx.x;
  const float top = A.stats[2 * r], s = A.stats[2 * r + 1];
  T* dz = (T*)A.dlogits + r * A.dstride;
  const int chunks = A.V / EPL, rest = A.V - chunks * EPL;
  if (s < 0.f) {
    for (int i = threadIdx.x; i < chunks; i += THREADS)
      store_chunk_any(dz + (int64_t)i * EPL, make_uint4(0u, 0u, 0u, 0u));
    if ((int)threadIdx.x < rest) store_bits(dz + (int64_t)chunks * EPL + threadIdx.x, 0u);
    return;
  }
  const int mask = (1 << (32 - __clz(A.K - 1))) - 1;  // as many lists as entries, rounded up to a power of two
  for (int k = threadIdx.x; k <= mask; k += THREADS) head[k] = -1;
  float t_max, t_sum;
  teacher_row<THREADS>(A, r, id, prob, slot, t_max, t_sum);
  for (int k = threadIdx.x; k < A.K; k += THREADS)
    if (id[k] >= 0) next[k] = atomicExch(&head[id[k] & mask], k);
  const T* z = (const T*)A.logits + r * A.stride;
  const float c = LOG2E / A.tau, g = A.grad[r] * A.tau, scale = g / s;
  int i = threadIdx.x;
  for (; i + (DEEP - 1) * THREADS < chunks; i += DEEP * THREADS) {
    uint4 w[DEEP];
#pragma unroll
    for (int k = 0; k < DEEP; ++k) w[k] = load_chunk_any(z + (int64_t)(i + k * THREADS) * EPL);
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      float v[EPL];
      Chunk<T>::unpack(w[k], v);
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = exp2_hw((v[e] - top) * c) * scale;
      store_chunk<STREAM>(dz + (int64_t)(i + k * THREADS) * EPL, Chunk<T>::pack(v));
    }
  }
  for (; i < chunks; i += THREADS) {
    float v[EPL];
    Chunk<T>::unpack(load_chunk_any(z + (int64_t)i * EPL), v);
#pragma unroll
    for (int e = 0; e < EPL; ++e) v[e] = exp2_hw((v[e] - top) * c) * scale;
    store_chunk_any(dz + (int64_t)i * EPL, Chunk<T>::pack(v));
  }
  if ((int)threadIdx.x < rest) {
    const int64_t at = (int64_t)chunks * EPL + threadIdx.x;
    store_as(dz, at, exp2_hw((Elem<T>::load(z + at) - top) * c) * scale, Elem<T>::code);
  }
  // The teacher's entries again, with their probabilities taken off before the one rounding.  An id that comes
  // twice is written twice with the same value: every writer adds all entries of its id, in the order of k.  They
  // are found in its list, whose own order is that of the atomics: the next one up from the last, while they are few.
  // (Looking at all K for each: 4096 x 50304 with 1024 entries 609 us, this way 295; 173 with 64.)  The row's
  // stores are waited for: these overwrite some of them from other waves.
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
  for (int k = threadIdx.x; k < A.K; k += THREADS) {
    if (id[k] < 0) continue;
    int same = 0;
    for (int j = head[id[k] & mask]; j >= 0; j = next[j]) same += id[j] == id[k];
    float p = 0.f;
    if (same <= 8) {
      for (int n = 0, last = -1; n < same; ++n) {
        int least = DISTILL_MAX_K;
        for (int j = head[id[k] & mask]; j >= 0; j = next[j])
          if (id[j] == id[k] && j > last) least = min(least, j);
        p += exp2_hw((prob[least] - t_max) * c);
        last = least;
      }
    } else {
      for (int j = 0; j < A.K; ++j)
        if (id[j] == id[k]) p += exp2_hw((prob[j] - t_max) * c);
    }
    const float q = exp2_hw((Elem<T>::load(z + id[k]) - top) * c) / s;
    store_as(dz, id[k], g * (q - p / t_sum), Elem<T>::code);
  }
}

static int distill_check(const DistillArgs& A, int dtype, const char* what) {
  BGX_REQUIRE(A.rows >= 0 && A.V >= 1 && A.K >= 1, BGX_E_ARG, "%s: rows=%lld V=%d K=%d", what, (long long)A.rows, A.V,
              A.K);
  BGX_REQUIRE(A.K <= DISTILL_MAX_K, BGX_E_SHAPE, "%s: K=%d, at most %d entries per token", what, A.K, DISTILL_MAX_K);
  BGX_REQUIRE(A.rows < (1ll << 31), BGX_E_SHAPE, "%s: %lld rows", what, (long long)A.rows);
  BGX_REQUIRE(A.V <= 0x7fffffff - 64, BGX_E_SHAPE, "%s: V=%d", what, A.V);
  BGX_REQUIRE(dtype >= BGX_F32 && dtype <= BGX_BF16 && A.teacher_dtype >= BGX_F32 && A.teacher_dtype <= BGX_BF16,
              BGX_E_DTYPE, "%s: dtype %d / %d", what, dtype, A.teacher_dtype);
  BGX_REQUIRE(A.tau > 0.f && A.tau < INFINITY, BGX_E_ARG, "%s: temperature %g", what, A.tau);
  BGX_REQUIRE(A.rows == 0 || (A.logits && A.ids && A.teacher), BGX_E_ARG, "%s: null operand", what);
  BGX_REQUIRE(A.rows == 0 || A.stride >= A.V, BGX_E_ARG, "%s: row stride %lld below V=%d", what, (long long)A.stride,
              A.V);
  return 0;
}

template <typename T>
static int distill_launch(const DistillArgs& A, bool backward, hipStream_t s) {
  const dim3 grid((unsigned)A.rows);
  if (A.rows < DISTILL_FEW) {
    if (backward)
      distill_backward_kernel<T, 1024, false><<<grid, 1024, 0, s>>>(A);
    else
      distill_forward_kernel<T, 1024><<<grid, 1024, 0, s>>>(A);
  } else if (backward && A.rows * A.V * (int64_t)sizeof(T) >= STREAM_BYTES) {
    distill_backward_kernel<T, 256, true><<<grid, 256, 0, s>>>(A);
  } else if (backward) {
    distill_backward_kernel<T, 256, false><<<grid, 256, 0, s>>>(A);
  } else {
    distill_forward_kernel<T, 256><<<grid, 256, 0, s>>>(A);
  }
  BGX_HIP(hipGetLastError());
  return 0;
}

static int distill_dispatch(const DistillArgs& A, int dtype, bool backward, void* stream) {
  if (A.rows == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == BGX_F32) return distill_launch<float>(A, backward, s);
  if (dtype == BGX_F16) return distill_launch<f16_t>(A, backward, s);
  return distill_launch<bf16_t>(A, backward, s);
}

int distill_forward_impl(const void* logits, int64_t stride, int64_t rows, int V, int dtype, const int64_t* ids,
                         const void* teacher, int teacher_dtype, int K, const uint8_t* valid, float tau, float* losses,
                         float* stats, void* stream) {
  DistillArgs A{};
  A.logits = logits;
  A.stride = stride;
  A.rows = rows;
  A.V = V;
  A.ids = ids;
  A.teacher = teacher;
  A.teacher_dtype = teacher_dtype;
  A.K = K;
  A.valid = valid;
  A.tau = tau;
  A.losses = losses;
  A.stats = stats;
  if (int rc = distill_check(A, dtype, "distillation")) return rc;
  BGX_REQUIRE(rows == 0 || losses, BGX_E_ARG, "distillation: null losses");
  return distill_dispatch(A, dtype, false, stream);
}

int distill_backward_impl(const void* logits, int64_t stride, int64_t rows, int V, int dtype, const int64_t* ids,
                          const void* teacher, int teacher_dtype, int K, float tau, const float* stats,
                          const float* grad, void* dlogits, int64_t dstride, void* stream) {
  DistillArgs A{};
  A.logits = logits;
  A.stride = stride;
  A.rows = rows;
  A.V = V;
  A.ids = ids;
  A.teacher = teacher;
  A.teacher_dtype = teacher_dtype;
  A.K = K;
  A.tau = tau;
  A.stats = const_cast<float*>(stats);
  A.grad = grad;
  A.dlogits = dlogits;
  A.dstride = dstride;
  if (int rc = distill_check(A, dtype, "distillation backward")) return rc;
  BGX_REQUIRE(rows == 0 || (stats && grad && dlogits), BGX_E_ARG, "distillation backward: null operand");
  BGX_REQUIRE(rows == 0 || dstride >= V, BGX_E_ARG, "distillation backward: row stride %lld below V=%d",
              (long long)dstride, V);
  return distill_dispatch(A, dtype, true, stream);
}

}  // namespace bgx
