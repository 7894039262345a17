// Beam search's selection: over the K * V continuations of a sequence,
//   value[k, t] = score[k] + x[k, t] - logsumexp(x[k, :]),  the n largest, ties to the lowest k * V + t.
//
// One pass over the logits.  A CTA takes a stretch of one row: each thread sums exp(x - m) (m: its first maximum; fp32 over at most a few hundred
// terms, 64 bits from there on, since candidates of different rows are told apart by less than 32 bits of a long sum hold) and puts elements that can
// still be among the stretch's n largest aside.  What "can still be" means: the n-th largest of 128 group maxima of the stretch's first tile, a
// value that n elements reach.  Elements put aside beyond the buffer raise that bound and the stretch is read once more; each such pass strictly
// raises it, and the set that is left does not depend on the order of the atomics.
// A second launch, chained to the first, adds up the rows' sums, turns the sorted lists into values in 64 bits and merges them.
// Bound by the logits' bytes for many rows, by the two launches' latency for few.
#include "common.cuh"

namespace tsb {
namespace {

constexpr int kThreads = 512, kVec = 2, kMaxBest = 32, kGroups = 128, kCap = 2048;
constexpr int kMaxLists = 256, kMaxBeams = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct Part {           // of a row's stretch
  double sum;           // sum of exp(x - m)
  float m;
  int pad;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// larger value first, then the lower column
__device__ __forceinline__ bool before(float xa, int ia, float xb, int ib) { return xa > xb || (xa == xb && ia < ib); }

template <typename T>
struct Row {
  static constexpr int N = 16 / (int)sizeof(T);       // elements of a 16-byte vector
  const T* base;                                      // 16-byte boundary at or below the row's first element
  int lead;                                           // elements between them
  int V;
  // elements v * N - lead .. of the row, -infinity where that is outside of it
  __device__ __forceinline__ void load(int64_t v, float (&x)[N]) const {
    const int64_t c0 = v * N - lead;
    if (c0 >= 0 && c0 + N <= V) {
      alignas(16) T e[N];
      *reinterpret_cast<uint4*>(e) = __ldcs(reinterpret_cast<const uint4*>(base + v * N));
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = to_f32<T>(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = c0 + i >= 0 && c0 + i < V ? to_f32<T>(base[v * N + i]) : -INFINITY;
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
beam_rows_kernel(const T* __restrict__ logits, int64_t row_stride, int V, int splits, int64_t span, const float* __restrict__ scores,
                 const uint8_t* __restrict__ finished, int n, Part* __restrict__ parts, float2* __restrict__ lists) {
  constexpr int N = Row<T>::N;
  __shared__ __align__(16) float s_group[kGroups];
  __shared__ float s_x[kCap];
  __shared__ int s_i[kCap];
  __shared__ float s_bound;
  __shared__ int s_group_i[kGroups], s_bound_i, s_count;
  __shared__ double s_sum[kThreads / 32];
  __shared__ float s_m[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x / splits;
  const int split = (int)(blockIdx.x % splits), tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  // a row without a score or at its end has no candidates of its own
  if (!(scores[row] > -INFINITY) || (finished && finished[row])) return;
  Row<T> r;
  const uintptr_t at = reinterpret_cast<uintptr_t>(logits + row * row_stride);
  r.base = reinterpret_cast<const T*>(at & ~(uintptr_t)15);
  r.lead = (int)((at & 15) / sizeof(T));
  r.V = V;
  const int64_t vectors = (r.lead + (int64_t)V + N - 1) / N;
  const int64_t v0 = split * span, v1 = min(vectors, v0 + span);
  float m = -INFINITY, sum = 0.f;
  if (tid == 0) { s_count = 0; s_bound = -INFINITY; }
  float bound = -INFINITY;
  auto put_aside = [&](float x, int64_t col) {
    const int slot = atomicAdd(&s_count, 1);
    if (slot < kCap) { s_x[slot] = x; s_i[slot] = (int)col; }
  };
  bool first = true;
  for (int64_t t0 = v0; t0 < v1; t0 += kThreads * kVec) {
    float x[kVec][N];
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      const int64_t v = t0 + u * kThreads + tid;
      if (v < v1) r.load(v, x[u]);
      else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[u][i] = -INFINITY;
      }
    }
    float top[kVec];
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      top[u] = x[u][0];
#pragma unroll
      for (int i = 1; i < N; ++i) top[u] = fmaxf(top[u], x[u][i]);
    }
    float most = top[0];
#pragma unroll
    for (int u = 1; u < kVec; ++u) most = fmaxf(most, top[u]);
    if (most > m + 32.f) {                             // the first tile; later ones only where terms could leave fp32's range
      sum *= m == -INFINITY ? 0.f : ex2((m - most) * kLog2e);
      m = most;
    }
    if (m > -INFINITY) {
#pragma unroll
      for (int u = 0; u < kVec; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) sum += ex2((x[u][i] - m) * kLog2e);
    } else {                                           // nothing but -infinity and NaN so far
#pragma unroll
      for (int u = 0; u < kVec; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) sum += x[u][i] == -INFINITY ? 0.f : x[u][i];
    }
    if (first) {
      first = false;
      float gm = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
      if ((lane & 3) == 0) s_group[tid >> 2] = gm;
      __syncthreads();
      if (tid < kGroups) {
        const float own = s_group[tid];
        int rank = 0;
        for (int j = 0; j < kGroups; j += 4) {
          const float4 o = *reinterpret_cast<const float4*>(&s_group[j]);
          rank += (o.x > own || (o.x == own && j < tid)) + (o.y > own || (o.y == own && j + 1 < tid)) + (o.z > own || (o.z == own && j + 2 < tid)) +
                  (o.w > own || (o.w == own && j + 3 < tid));
        }
        if (rank == n - 1) s_bound = own;
      }
      __syncthreads();
      bound = s_bound;
    }
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      if (top[u] >= bound) {
        const int64_t c0 = (t0 + u * kThreads + tid) * N - r.lead;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (x[u][i] >= bound && x[u][i] > -INFINITY) put_aside(x[u][i], c0 + i);
      }
    }
  }
  // ---- the stretch's sum
  const float mw = warp_max(m);
  double part = m == -INFINITY ? (double)sum : (double)sum * exp((double)m - (double)mw);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (lane == 0) { s_m[w] = mw; s_sum[w] = part; }
  __syncthreads();
  if (tid == 0) {
    float mm = -INFINITY;
    for (int i = 0; i < kThreads / 32; ++i) mm = fmaxf(mm, s_m[i]);
    double all = 0.0;
    for (int i = 0; i < kThreads / 32; ++i) all += s_m[i] == -INFINITY ? s_sum[i] : s_sum[i] * exp((double)s_m[i] - (double)mm);
    parts[row * splits + split] = Part{all, mm, 0};
  }
  // ---- too many put aside: the n-th best of 128 groups of those kept is a higher bound.  At least 96 groups are below it, so that every
  // pass leaves 1536 elements fewer; rows of one value or of a few allowed tokens take one, ascending ones as many as that says.
  int count = s_count;
  while (count > kCap) {
    __syncthreads();
    float gx = -INFINITY;
    int gi = 0x7fffffff;
    if (tid < kGroups) {
      for (int j = tid; j < kCap; j += kGroups)
        if (before(s_x[j], s_i[j], gx, gi)) { gx = s_x[j]; gi = s_i[j]; }
      s_group[tid] = gx;
      s_group_i[tid] = gi;
    }
    __syncthreads();
    if (tid < kGroups) {
      int rank = 0;
      for (int j = 0; j < kGroups; ++j) rank += before(s_group[j], s_group_i[j], gx, gi);
      if (rank == n - 1) { s_bound = gx; s_bound_i = gi; }
    }
    if (tid == 0) s_count = 0;
    __syncthreads();
    const float bx = s_bound;
    const int bi = s_bound_i;
    for (int64_t v = v0 + tid; v < v1; v += kThreads) {
      float x[N];
      r.load(v, x);
      const int64_t c0 = v * N - r.lead;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (x[i] > bx || (x[i] == bx && c0 + i <= bi)) put_aside(x[i], c0 + i);
    }
    __syncthreads();
    count = s_count;
  }
  // ---- the n best, sorted
  float2* list = lists + (row * splits + split) * n;
  for (int c = tid; c < count; c += kThreads) {
    const float xc = s_x[c];
    const int ic = s_i[c];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += before(s_x[j], s_i[j], xc, ic);
    if (rank < n) list[rank] = make_float2(xc, __int_as_float(ic));
  }
  if (tid >= count && tid < n) list[tid] = make_float2(-INFINITY, __int_as_float(-1));      // fewer elements than that
}

// One CTA a sequence.  The n-th best of the lists' first entries bounds what can be among the n best of all; the few entries that reach it are ranked.
// -infinity is nobody's list entry: where fewer than n candidates are above it, all of them have been selected, and the places left go
// to the lowest k * V + t that have not.
__global__ void __launch_bounds__(kThreads)
beam_merge_kernel(int K, int V, int splits, const float* __restrict__ scores, const uint8_t* __restrict__ finished, int64_t pad, int n,
                  const Part* __restrict__ parts, const float2* __restrict__ lists, float* __restrict__ out_scores, int32_t* __restrict__ out_parents,
                  int64_t* __restrict__ out_tokens) {
  constexpr int kMost = kMaxBest * (kMaxBest + 1);            // entries that can reach the bound
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ double s_val[kMost], s_bound;
  __shared__ int64_t s_at[kMost], s_bound_at, s_taken[kMaxBest];
  __shared__ int s_count;
  double* lse = reinterpret_cast<double*>(smem);              // [K]
  float2* s_list = reinterpret_cast<float2*>(lse + K);        // [K][splits][n]
  pdl_launch_dependents();
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, count = K * splits;
  const float* score = scores + b * K;
  const uint8_t* fin = finished ? finished + b * K : nullptr;
  pdl_wait();
  if (tid == 0) { s_count = 0; s_bound = -INFINITY; s_bound_at = INT64_MAX; }
  for (int i = tid; i < count * n; i += kThreads) s_list[i] = __ldcg(&lists[b * count * n + i]);
  for (int k = tid; k < K; k += kThreads) {
    double l = __longlong_as_double(0x7ff8000000000000LL);    // not a number: the row has no candidates of its own
    if (score[k] > -INFINITY && !(fin && fin[k])) {
      const Part* p = parts + (b * K + k) * splits;
      float mm = -INFINITY;
      for (int i = 0; i < splits; ++i) mm = fmaxf(mm, p[i].m);
      double all = 0.0;
      for (int i = 0; i < splits; ++i) all += p[i].m == -INFINITY ? p[i].sum : p[i].sum * exp((double)p[i].m - (double)mm);
      if (mm > -INFINITY && mm < INFINITY && all > 0.0) l = (double)mm + log(all);
    }
    lse[k] = l;
  }
  __syncthreads();
  auto entry = [&](int l, int pos, double& value, int64_t& at) {
    const int k = l / splits;
    value = -INFINITY;
    at = INT64_MAX;
    if (lse[k] == lse[k]) {
      const float2 c = s_list[l * n + pos];
      const int col = __float_as_int(c.y);
      if (col >= 0) { value = (double)score[k] + ((double)c.x - lse[k]); at = (int64_t)k * V + col; }
    } else if (fin && fin[k] && score[k] > -INFINITY && l % splits == 0 && pos == 0) {
      value = score[k];
      at = (int64_t)k * V + pad;
    }
  };
  auto first = [](double va, int64_t aa, double vb, int64_t ab) { return va > vb || (va == vb && aa < ab); };
  const int depth = min(n, (n + count - 1) / count), heads = count * depth;      // heads <= max(count, 2 n): fits s_val
  for (int i = tid; i < heads; i += kThreads) entry(i / depth, i % depth, s_val[i], s_at[i]);
  __syncthreads();
  for (int i = tid; i < heads; i += kThreads) {
    const double v = s_val[i];
    const int64_t at = s_at[i];
    if (at == INT64_MAX) continue;
    int rank = 0;
    for (int j = 0; j < heads; ++j) rank += first(s_val[j], s_at[j], v, at);
    if (rank == n - 1) { s_bound = v; s_bound_at = at; }
  }
  __syncthreads();
  const double bound = s_bound;
  const int64_t bound_at = s_bound_at;
  for (int i = tid; i < count * n; i += kThreads) {
    double v;
    int64_t at;
    entry(i / n, i % n, v, at);
    if (at != INT64_MAX && !first(bound, bound_at, v, at)) {
      const int slot = atomicAdd(&s_count, 1);
      if (slot < kMost) { s_val[slot] = v; s_at[slot] = at; }
    }
  }
  __syncthreads();
  const int total = min(s_count, kMost);
  for (int i = tid; i < total; i += kThreads) {
    const double v = s_val[i];
    const int64_t at = s_at[i];
    int rank = 0;
    for (int j = 0; j < total; ++j) rank += first(s_val[j], s_at[j], v, at);
    if (rank < n) {
      out_scores[b * n + rank] = (float)v;
      out_parents[b * n + rank] = (int32_t)(b * K + at / V);
      out_tokens[b * n + rank] = at % V;
      s_taken[rank] = at;
    }
  }
  if (total >= n) return;
  __syncthreads();
  if (tid == 0) {
    int64_t at = 0;
    for (int i = total; i < n; ++i, ++at) {
      for (bool again = true; again;) {
        again = false;
        for (int j = 0; j < total; ++j)
          if (s_taken[j] == at) { ++at; again = true; }
      }
      out_scores[b * n + i] = -INFINITY;
      out_parents[b * n + i] = (int32_t)(b * K + at / V);
      out_tokens[b * n + i] = at % V;
    }
  }
}

// Stretches of a row: enough CTAs for four an SM, whole tiles of a CTA, and no more lists than the merge ranks in a microsecond or two.
int row_splits(int64_t rows, int K, int64_t V, int dtype) {
  const int64_t tile = kThreads * kVec * (dtype == TSB200_F32 ? 4 : 8);
  int64_t s = (592 + rows - 1) / rows;
  const int64_t cap = (V + tile - 1) / tile, room = kMaxLists / K;
  if (s > cap) s = cap;
  if (s > room) s = room;
  return (int)(s < 1 ? 1 : s);
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" {

size_t tsb200_beam_select_workspace_bytes(int64_t B, int K, int64_t V, int dtype, int n) {
  if (B <= 0 || K <= 0 || V <= 0 || n <= 0) return 0;
  const int64_t lists = B * K * row_splits(B * K, K, V, dtype);
  return (size_t)(lists * (int64_t)(sizeof(Part) + n * sizeof(float2)) + 256);
}

int tsb200_beam_select(const void* logits, int dtype, int64_t row_stride, int64_t B, int K, int64_t V, const float* scores, const uint8_t* finished,
                       int64_t pad_token, int n, float* out_scores, int32_t* out_parents, int64_t* out_tokens, void* workspace, size_t workspace_bytes,
                       void* stream) {
  TSB_REQUIRE_DEVICE();
  if (B < 0 || K <= 0 || V <= 0 || n <= 0) return TSB200_ERR_ARG;
  if (dtype != TSB200_F32 && dtype != TSB200_BF16) return TSB200_ERR_UNSUPPORTED;
  if (n > kMaxBest || K > kMaxBeams || V > 0x7fffffffLL - 64 || (int64_t)n > (int64_t)K * V) return TSB200_ERR_UNSUPPORTED;
  const int64_t stride = row_stride ? row_stride : V;
  if (stride < V) return TSB200_ERR_ARG;
  if (finished && (pad_token < 0 || pad_token >= V)) return TSB200_ERR_ARG;
  if (B == 0) return TSB200_OK;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !workspace || !aligned(workspace, 16)) return TSB200_ERR_ARG;
  if (!aligned(logits, dtype == TSB200_F32 ? 4 : 2)) return TSB200_ERR_ARG;
  if (workspace_bytes < tsb200_beam_select_workspace_bytes(B, K, V, dtype, n)) return TSB200_ERR_WORKSPACE;
  const int splits = row_splits(B * K, K, V, dtype);
  if (B * K > 0x7fffffffLL / splits || B > 0x7fffffffLL) return TSB200_ERR_UNSUPPORTED;
  const int per = dtype == TSB200_F32 ? 4 : 8;
  const int64_t vectors = (V + 2 * per - 2) / per;                 // a row may start inside a vector
  const int64_t span = (vectors + splits - 1) / splits;
  Part* parts = (Part*)workspace;
  float2* lists = (float2*)(parts + B * K * splits);
  cudaStream_t s = as_stream(stream);
  const dim3 grid((unsigned)(B * K * splits));
  if (dtype == TSB200_F32)
    TSB_CUDA(launch_kernel(beam_rows_kernel<float>, grid, dim3(kThreads), 0, s, (const float*)logits, stride, (int)V, splits, span, scores, finished, n, parts,
                           lists));
  else
    TSB_CUDA(launch_kernel(beam_rows_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, s, (const __nv_bfloat16*)logits, stride, (int)V, splits, span, scores,
                           finished, n, parts, lists));
  const size_t smem = (size_t)K * 8 + (size_t)K * splits * n * 8;
  static bool configured[64] = {false};
  int dev = 0;
  TSB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TSB200_ERR_DEVICE;
  if (!configured[dev]) {
    TSB_CUDA(cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBeams * 8 + kMaxLists * kMaxBest * 8));
    configured[dev] = true;
  }
  TSB_CUDA(launch_kernel_if(true, beam_merge_kernel, dim3((unsigned)B), dim3(kThreads), smem, s, K, (int)V, splits, scores, finished, pad_token, n, parts,
                            lists, out_scores, out_parents, out_tokens));
  return TSB200_OK;
}

}  // extern "C"
