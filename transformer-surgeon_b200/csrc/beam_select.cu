// Beam search's selection: over the K * V continuations of a sequence,
//   value[k, t] = score[k] + x[k, t] - logsumexp(x[k, :]),  the n largest, ties to the lowest k * V + t.
//
// One pass over the logits.  A CTA takes a stretch of one row, in vectors of 16 bytes: it sums 2^(x log2 e - R) (R: a whole number near the first
// tile's maximum, raised with the elements, so that sums are put together by exact shifts; fp32 over the few hundred terms of a thread, 64 bits from there on, since candidates of
// different rows are told apart by less than 32 bits of a long sum hold) and notes vectors whose largest element can still be among the
// stretch's n best.  What "can still be" means: the n-th largest of 64 group maxima of the first tile, a value that n elements reach.  At the end the n
// best of the noted vectors hold the n best elements; those alone are looked at one by one.  More noted vectors than there is room for raise the
// bound, and the stretch is read once more; each such pass strictly raises it, and what is left does not depend on the order of the atomics.
// The last CTA of a sequence to be done adds up the rows' sums, turns the sorted lists into values in 64 bits and merges them (as a second launch, chained to
// the first, about as long on the device and 4 us more of the host's time a call).
// Many rows: 32 x 8 beams of 152064 30.9 us, of which the bytes alone take 12; without the merge 25.5, without all that is behind the loop 22.7, without
// exponentials 27.7.  No unit is full (exponentials 47 %, issue slots 46 %, memory 29 %): a tile's loads, the wait for them and its arithmetic follow one
// another in a CTA (tiles requested ahead into registers 31, into shared memory 34; the bound raised again after 2, 4, 8 tiles 32).  Few: the chain of steps behind the logits.
#include "common.cuh"

namespace tsb {
namespace {

constexpr int kThreads = 256, kVec = 4, kMaxBest = 32, kGroups = 64, kCap = 1024, kFew = 64;
constexpr int kSlots = 592, kEntries = 4 * kThreads, kMaxBeams = 256;
constexpr int kCounters = 4096;         // sequences of a launch; their counters are the workspace's head
constexpr int kMost = kMaxBest * (kMaxBest + 1);            // entries that can reach the merge's bound
constexpr float kLog2e = 1.4426950408889634f;
// Up to this |x log2 e| a whole number R refers to its neighbours exactly, and x log2 e - R is rounded once.  Beyond (masks of -1e9 and the like, the
// type's lowest value: x log2 e may be off by more than the range of exponents) sums refer to a logit m.
constexpr float kFar = 4194304.f;
// A thread's R follows its elements when they are this far above it: the sum's larger terms then have arguments of 4 at most, rounded to 2^-23 (an argument
// near 100: 2^-18, eleven times the exponential's own error).
constexpr float kAbove = 4.f;

struct Part {           // of a row's stretch
  double sum;           // sum of 2^(x log2 e - R), or, with R = -infinity, of 2^((x - m) log2 e); m = -infinity too: of nothing
  float R;
  float m;
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
  static constexpr int N = 16 / (int)sizeof(T);       // elements of a vector
  const T* base;                                      // 16-byte boundary at or below the row's first element
  int lead;                                           // elements between them
  int V;
  // elements v * N - lead .. of the row, -infinity where that is outside of it
  __device__ __forceinline__ uint4 load(int v) const {
    const int c0 = v * N - lead;
    if (c0 >= 0 && c0 <= V - N) return __ldcs(reinterpret_cast<const uint4*>(base) + v);
    alignas(16) T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = c0 + i >= 0 && c0 + i < V ? base[(int64_t)v * N + i] : from_f32<T>(-INFINITY);
    return *reinterpret_cast<const uint4*>(e);
  }
};
// Largest element, NaN passed over (-infinity if there is none).
template <typename T>
__device__ __forceinline__ float top_of(const uint4& r) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m = __hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3]));
    return fmaxf(-INFINITY, fmaxf(__low2float(m), __high2float(m)));
  } else {
    const float* e = reinterpret_cast<const float*>(&r);
    return fmaxf(fmaxf(fmaxf(-INFINITY, e[0]), e[1]), fmaxf(e[2], e[3]));
  }
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
// sums (a pair) += 2^(x log2 e - R) over a vector; c = (log2 e, log2 e), r = (-R, -R).
template <typename T>
__device__ __forceinline__ void add_exps(uint64_t& sums, const uint4& v, uint64_t c, uint64_t r) {
  const unsigned e[4] = {v.x, v.y, v.z, v.w};
  constexpr int PAIRS = Row<T>::N / 2;
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const uint64_t x = sizeof(T) == 2 ? pair_of(__uint_as_float(e[i] << 16), __uint_as_float(e[i] & 0xffff0000u))
                                      : pair_of(__uint_as_float(e[2 * i % 4]), __uint_as_float(e[(2 * i + 1) % 4]));
    uint64_t y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(y) : "l"(x), "l"(c), "l"(r));
    float y0, y1;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(y0), "=f"(y1) : "l"(y));
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(sums) : "l"(sums), "l"(pair_of(ex2(y0), ex2(y1))));
  }
}
__device__ __forceinline__ float sum_of(uint64_t p) {
  float a, b;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(p));
  return a + b;
}
__device__ __forceinline__ double pow2(float e) {              // of a whole number from -1000 to 0, or less: zero
  return e < -1000.f ? 0.0 : __hiloint2double((1023 + (int)e) << 20, 0);
}
__device__ __forceinline__ float pow2f(float e) { return e < -126.f ? 0.f : __int_as_float((127 + (int)e) << 23); }     // of a whole number up to 0
// What a sum of reference (R, m) is multiplied by to have the reference (Rn, mn), which is no lower.  m log2 e has 48 bits: exact.
__device__ __noinline__ double to_reference(float R, float m, float Rn, float mn) {
  const double a = R > -INFINITY ? (double)R : (double)m * (double)kLog2e, b = Rn > -INFINITY ? (double)Rn : (double)mn * (double)kLog2e;
  return exp2(a - b);
}
// Of two references (R, -infinity) and (-infinity, m), the higher one.
__device__ __forceinline__ void higher(float& R, float& m) {
  if ((double)m * (double)kLog2e > (double)R) R = -INFINITY;
  else m = -INFINITY;
}

// A value that the n-th largest of 64 groups' maxima reaches (x: this thread's maximum; a group: kThreads / 64 neighbours); -infinity where fewer than n
// groups have one.  *most: the largest of all.  Groups are compared as whole numbers of the same order whose last six bits, taken off the
// value, tell equal ones apart.  For all threads of the CTA; s: 64 words.
__device__ __noinline__ float nth_group(float x, int n, int* s, float* s_bound, float* most) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int o = 1; o < kThreads / kGroups; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  const int group = tid / (kThreads / kGroups), part = tid % (kThreads / kGroups);
  const int bits = __float_as_int(x), order = bits ^ ((bits >> 31) & 0x7fffffff);
  const int key = (order & ~(kGroups - 1)) | (kGroups - 1 - group);
  if (part == 0) s[group] = key;
  __syncthreads();
  int rank = 0;
  constexpr int PER = kGroups / (kThreads / kGroups);
#pragma unroll
  for (int j = 0; j < PER; j += 4) {
    const int4 o = *reinterpret_cast<const int4*>(&s[part * PER + j]);
    rank += (o.x > key) + (o.y > key) + (o.z > key) + (o.w > key);
  }
#pragma unroll
  for (int o = 1; o < kThreads / kGroups; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
  const int down = order & ~(kGroups - 1);
  if (rank == n - 1) s_bound[0] = x == -INFINITY ? -INFINITY : __int_as_float(down ^ ((down >> 31) & 0x7fffffff));
  if (rank == 0) s_bound[1] = x;
  __syncthreads();
  *most = s_bound[1];
  return s_bound[0];
}

// How many of s_x[0 .. count) (s_i: their places) come before entry e, counted by `per` neighbouring threads (a power of two up to 32).
__device__ __noinline__ int rank_of(const float* s_x, const int* s_i, int count, int e, int per) {
  const float x = s_x[e];
  const int at = s_i[e];
  int rank = 0;
  for (int j = threadIdx.x & (per - 1); j < count; j += per) rank += before(s_x[j], s_i[j], x, at);
  for (int o = 1; o < per; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
  return rank;
}
// Threads per entry: as many as there are for all entries at once.
__device__ __forceinline__ int threads_per(int count, int threads) {
  int per = 1;
  while (per < 32 && 2 * per * count <= threads) per *= 2;
  return per;
}

struct RowsSmem {
  float x[kCap];                                              // noted vectors: largest element, number; later the best ones' elements, columns
  int i[kCap];
  float y[kCap];                                              // those of them that reach a second bound
  int j[kCap];
};
struct MergeSmem {
  int64_t val[kMost], at[kMost], bound, bound_at, taken[kMaxBest];
  float least[kMaxBeams];                                     // logit below which a row's entries are below the bound
  double base[kMaxBeams];                                     // score - logsumexp + ref; not a number where the row has no candidates of its own
  float ref[kMaxBeams];
  int count;
};

// Of one sequence, by the CTA that is done last: parts, list and what is behind them are this sequence's.  The lists' first entries bound what can be
// among the n best of all; the few entries that reach the bound are ranked.  -infinity is nobody's list entry: where fewer than n
// candidates are above it, all of them have been selected, and the places left go to the lowest k * V + t that have not.
__device__ __forceinline__ void merge(MergeSmem& s, int* group, float* bound2, int64_t b, int first_row, int K, int V, int splits, const float* __restrict__ score, const uint8_t* __restrict__ fin, int64_t pad,
                                      int n, const Part* parts, const float2* list, float* __restrict__ out_scores,
                                      int32_t* __restrict__ out_parents, int64_t* __restrict__ out_tokens) {
  const int tid = threadIdx.x, lane = tid & 31, count = K * splits;
  if (tid == 0) { s.count = 0; s.bound = INT64_MIN; s.bound_at = INT64_MAX; }
  // entries, if they are few: neighbours in groups of their own; on their way while the rows' sums are made
  constexpr int U = kEntries / kThreads, PER = kThreads / kGroups;
  const int t0 = tid / PER + kGroups * (tid % PER);
  float2 c[U];
  if (count * n <= kEntries) {
#pragma unroll
    for (int u = 0; u < U; ++u) c[u] = t0 + u * kThreads < count * n ? __ldcg(&list[t0 + u * kThreads]) : make_float2(-INFINITY, __int_as_float(-1));
  }
  for (int k = tid >> 5; k < K; k += kThreads / 32) {             // a warp per row
    double l = __longlong_as_double(0x7ff8000000000000LL);
    float at = 0.f;
    if (score[k] > -INFINITY && !(fin && fin[k])) {
      const Part* p = parts + k * splits;
      constexpr int U = 2;                                    // up to 64 parts on their way at once
      float R = -INFINITY, m = -INFINITY;
      double all = 0.0;
      for (int i0 = 0; i0 < splits; i0 += 32 * U) {
        int4 raw[U];
        float Rn = R, mn = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + 32 * u + lane;
          raw[u] = i < splits ? __ldcg(reinterpret_cast<const int4*>(p + i)) : make_int4(0, 0, __float_as_int(-INFINITY), __float_as_int(-INFINITY));
          Rn = fmaxf(Rn, __int_as_float(raw[u].z));
          mn = fmaxf(mn, __int_as_float(raw[u].w));
        }
        Rn = warp_max(Rn);
        mn = warp_max(mn);
        // to the greatest R: by a power of two
        const bool shifts = mn == -INFINITY;
        if (!shifts) higher(Rn, mn);
        auto scaled = [&](double sum, float Ri, float mi) { return sum * (shifts ? (Ri > -INFINITY ? pow2(Ri - Rn) : 0.0) : to_reference(Ri, mi, Rn, mn)); };
        all = i0 ? scaled(all, R, m) : 0.0;
#pragma unroll
        for (int u = 0; u < U; ++u) all += scaled(__hiloint2double(raw[u].y, raw[u].x), __int_as_float(raw[u].z), __int_as_float(raw[u].w));
        R = Rn;
        m = mn;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      if (all > 0.0) {                                        // NaN where the row has one, or +infinity
        l = log(all) + (R > -INFINITY ? (double)R * (1.0 / (double)kLog2e) : 0.0);      // the log2 e that the sums were made with
        at = R > -INFINITY ? 0.f : m;
      }
    }
    if (lane == 0) { s.base[k] = (double)score[k] - l; s.ref[k] = at; }
  }
  __syncthreads();
  const float per_list = 1.f / n, per_row = 1.f / splits;      // quotients of at most 8192 by them, exact
  // (value, beam << 32 | column); values as whole numbers of the same order: comparisons in 64-bit floating point take several times as long
  auto entry = [&](float2 c, int l, int pos, int64_t& order, int64_t& at) {
    const int k = (int)((l + 0.5f) * per_row);
    const double base = s.base[k];
    double value = -INFINITY;
    at = INT64_MAX;
    if (base == base) {
      const int col = __float_as_int(c.y);
      if (col >= 0) { value = base + ((double)c.x - (double)s.ref[k]); at = (int64_t)k << 32 | col; }
    } else if (fin && fin[k] && score[k] > -INFINITY && l == k * splits && pos == 0) {
      value = score[k];
      at = (int64_t)k << 32 | pad;
    }
    const int64_t bits = __double_as_longlong(value + 0.0);   // one zero
    order = bits ^ ((bits >> 63) & INT64_MAX);
  };
  auto first = [](int64_t va, int64_t aa, int64_t vb, int64_t ab) { return va > vb || (va == vb && aa < ab); };
  auto value_of = [](int64_t order) { return __longlong_as_double(order ^ ((order >> 63) & INT64_MAX)); };
  auto rank_at = [&](int entries, int e, int per) {
    const int64_t v = s.val[e], at = s.at[e];
    int rank = 0;
    for (int j = tid & (per - 1); j < entries; j += per) rank += first(s.val[j], s.at[j], v, at);
    for (int o = 1; o < per; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    return rank;
  };
  auto keep = [&](int64_t v, int64_t at) {
    const int slot = atomicAdd(&s.count, 1);
    if (slot < kMost) { s.val[slot] = v; s.at[slot] = at; }
  };
  // ---- a bound, the n-th largest of 64 groups, and the entries that reach it
  float top = -INFINITY, all;
  if (count * n <= kEntries) {                                // every entry
    int64_t v[U], at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = t0 + u * kThreads, l = (int)((i + 0.5f) * per_list);
      at[u] = INT64_MAX;
      if (i < count * n) entry(c[u], l, i - l * n, v[u], at[u]);
      if (at[u] != INT64_MAX) top = fmaxf(top, __double2float_rd(value_of(v[u])));
    }
    const double bound = nth_group(top, n, group, bound2, &all);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at[u] != INT64_MAX && value_of(v[u]) >= bound) keep(v[u], at[u]);
  } else {                                                    // the lists' first ones; they are more than n
    for (int l = t0; l < count; l += kThreads) {
      int64_t v, at;
      entry(__ldcg(&list[l * n]), l, 0, v, at);
      if (at != INT64_MAX) top = fmaxf(top, __double2float_rd(value_of(v)));
    }
    const float bound = nth_group(top, n, group, bound2, &all);
    // the logit at which a row's entries reach it (within rounding: a few entries more do no harm)
    if (tid < K) s.least[tid] = s.base[tid] == s.base[tid] ? __double2float_rd((double)bound - s.base[tid] + (double)s.ref[tid]) : -INFINITY;
    __syncthreads();
    for (int i0 = tid; i0 < count * n; i0 += U * kThreads) {
#pragma unroll
      for (int u = 0; u < U; ++u) c[u] = i0 + u * kThreads < count * n ? __ldcg(&list[i0 + u * kThreads]) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kThreads, l = (int)((i + 0.5f) * per_list), k = (int)((l + 0.5f) * per_row);
        if (i < count * n && (s.base[k] == s.base[k] ? c[u].x >= s.least[k] : l == k * splits && i == l * n)) {
          int64_t v, at;
          entry(c[u], l, i - l * n, v, at);
          if (at != INT64_MAX) keep(v, at);
        }
      }
    }
  }
  __syncthreads();
  if (s.count > kMost) {
    // many equal values: the n-th best of the lists' first entries, lower columns first, leaves no more than n in each of n lists
    __syncthreads();
    if (tid == 0) s.count = 0;
    const int depth = min(n, (n + count - 1) / count), heads = count * depth;    // heads <= max(count, 2 n): fits s.val
    for (int i = tid; i < heads; i += kThreads) entry(__ldcg(&list[i / depth * n + i % depth]), i / depth, i % depth, s.val[i], s.at[i]);
    __syncthreads();
    for (int e = tid; e - tid < heads; e += kThreads) {
      const int rank = rank_at(heads, min(e, heads - 1), 1);
      if (e < heads && rank == n - 1 && s.at[e] != INT64_MAX) { s.bound = s.val[e]; s.bound_at = s.at[e]; }
    }
    __syncthreads();
    const int64_t bound = s.bound, bound_at = s.bound_at;
    for (int i = tid; i < count * n; i += kThreads) {
      int64_t v, at;
      entry(__ldcg(&list[i]), i / n, i % n, v, at);
      if (at != INT64_MAX && !first(bound, bound_at, v, at)) keep(v, at);
    }
    __syncthreads();
  }
  const int total = min(s.count, kMost);
  const int per = threads_per(total, kThreads);
  for (int e0 = 0; e0 < total; e0 += kThreads / per) {
    const int e = e0 + tid / per, rank = rank_at(total, min(e, total - 1), per);
    if (e < total && rank < n && (tid & (per - 1)) == 0) {
      const int64_t at = s.at[e];
      out_scores[b * n + rank] = (float)value_of(s.val[e]);
      out_parents[b * n + rank] = first_row + (int32_t)(at >> 32);
      out_tokens[b * n + rank] = at & 0xffffffffLL;
      s.taken[rank] = at;
    }
  }
  if (total >= n) return;
  __syncthreads();
  if (tid == 0) {
    int k = 0, col = 0;
    for (int i = total; i < n;) {
      bool taken = false;
      for (int j = 0; j < total; ++j) taken = taken || s.taken[j] == ((int64_t)k << 32 | col);
      if (!taken) {
        out_scores[b * n + i] = -INFINITY;
        out_parents[b * n + i] = first_row + k;
        out_tokens[b * n + i] = col;
        ++i;
      }
      if (++col == V) { col = 0; ++k; }                       // n <= K V: there are enough
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4)
beam_select_kernel(const T* __restrict__ logits, int64_t row_stride, int K, int V, int splits, int span, const float* __restrict__ scores,
                   const uint8_t* __restrict__ finished, int64_t pad, int n, Part* parts, float2* lists, unsigned* __restrict__ counters,
                   int first_row, float* __restrict__ out_scores, int32_t* __restrict__ out_parents, int64_t* __restrict__ out_tokens) {
  constexpr int N = Row<T>::N, TILE = kThreads * kVec;
  __shared__ __align__(16) uint8_t s_both[sizeof(RowsSmem) > sizeof(MergeSmem) ? sizeof(RowsSmem) : sizeof(MergeSmem)];
  RowsSmem& rows = *reinterpret_cast<RowsSmem*>(s_both);
  float (&s_x)[kCap] = rows.x, (&s_y)[kCap] = rows.y;
  int (&s_i)[kCap] = rows.i, (&s_j)[kCap] = rows.j;
  __shared__ bool s_mine;
  __shared__ __align__(16) int s_group[kGroups];
  __shared__ float s_bound[2], s_R[kThreads / 32], s_m[kThreads / 32], s_last;
  __shared__ int s_best[kMaxBest], s_count, s_kept, s_elements;
  __shared__ double s_sum[kThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x / splits;
  const int split = (int)(blockIdx.x % splits), tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  // a row without a score or at its end has no candidates of its own
  if (scores[row] > -INFINITY && !(finished && finished[row])) {
  Row<T> r;
  const uintptr_t at = reinterpret_cast<uintptr_t>(logits + row * row_stride);
  r.base = reinterpret_cast<const T*>(at & ~(uintptr_t)15);
  r.lead = (int)((at & 15) / sizeof(T));
  r.V = V;
  const int vectors = (r.lead + V - 1) / N + 1;
  const int v0 = split * span, v1 = min(vectors, v0 + span);
  const int in0 = r.lead ? 1 : 0, in1 = (r.lead + V) / N;      // vectors that lie in the row as a whole
  if (tid == 0) { s_count = s_kept = s_elements = 0; s_bound[0] = s_bound[1] = s_last = -INFINITY; }
  auto note = [&](float x, int v) {
    const int slot = atomicAdd(&s_count, 1);
    if (slot < kCap) { s_x[slot] = x; s_i[slot] = v; }
  };
  const uint64_t c = pair_of(kLog2e, kLog2e);
  uint64_t sums = pair_of(0.f, 0.f);
  float R = -INFINITY, m = -INFINITY, bound = -INFINITY;       // one of R and m at most is above -infinity
  auto load_tile = [&](int t0, uint4 (&x)[kVec]) {
    if (t0 >= in0 && t0 + TILE <= min(v1, in1)) {
      const uint4* p = reinterpret_cast<const uint4*>(r.base) + t0 + tid;
#pragma unroll
      for (int u = 0; u < kVec; ++u) x[u] = __ldcs(p + u * kThreads);
    } else {
      const unsigned word = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;         // -infinity
#pragma unroll
      for (int u = 0; u < kVec; ++u) {
        x[u] = make_uint4(word, word, word, word);
        if (t0 + u * kThreads + tid < v1) x[u] = r.load(t0 + u * kThreads + tid);
      }
    }
  };
  for (int t0 = v0; t0 < v1; t0 += TILE) {
    uint4 x[kVec];
    load_tile(t0, x);
    float top[kVec], most = -INFINITY;
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      top[u] = top_of<T>(x[u]);
      most = fmaxf(most, top[u]);
    }
    if (t0 == v0) {
      float ref;
      bound = nth_group(most, n, s_group, s_bound, &ref);
      if (fabsf(ref) * kLog2e < kFar) R = ceilf(ref * kLog2e);
    }
    if (most * kLog2e > R + kAbove) {                         // or there is no R
      const float Rn = ceilf(most * kLog2e);
      if (fabsf(Rn) <= kFar) {
        if (most > m) {
          sums = pair_of(sum_of(sums) * (R > -INFINITY ? pow2f(R - Rn) : ex2(fmaf(m, kLog2e, -Rn))), 0.f);
          R = Rn;
          m = -INFINITY;
        }
      } else if (R > -INFINITY) {
        sums = pair_of(sum_of(sums) * ex2(fmaf(most, -kLog2e, R)), 0.f);
        m = most;
        R = -INFINITY;
      }
    }
    if (R > -INFINITY) {
      const uint64_t minus = pair_of(-R, -R);
#pragma unroll
      for (int u = 0; u < kVec; ++u) add_exps<T>(sums, x[u], c, minus);
    } else {
      float count = sum_of(sums);
#pragma unroll 1
      for (int u = 0; u < kVec; ++u) {
        alignas(16) T e[N];
        *reinterpret_cast<uint4*>(e) = u == 0 ? x[0] : u == 1 ? x[1] : u == 2 ? x[2] : x[3];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float y = to_f32<T>(e[i]);
          if (y > m) { count = fmaf(count, ex2((m - y) * kLog2e), 1.f); m = y; }     // what is not a number stays so
          else if (y != -INFINITY) count += ex2((y - m) * kLog2e);
        }
      }
      sums = pair_of(count, 0.f);
    }
#pragma unroll
    for (int u = 0; u < kVec; ++u)
      if (top[u] >= bound && top[u] > -INFINITY) note(top[u], t0 + u * kThreads + tid);
  }
  // ---- the stretch's sum
  {
    const float Rw = warp_max(R), mw = warp_max(m);
    if (lane == 0) { s_R[w] = Rw; s_m[w] = mw; }
    __syncthreads();
    float Rc = -INFINITY, mc = -INFINITY;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) { Rc = fmaxf(Rc, s_R[i]); mc = fmaxf(mc, s_m[i]); }
    double part = sum_of(sums);
    if (mc == -INFINITY) {
      part *= R > -INFINITY ? pow2(R - Rc) : 0.0;
    } else {
      higher(Rc, mc);
      part *= to_reference(R, m, Rc, mc);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (lane == 0) s_sum[w] = part;
    __syncthreads();
    if (tid == 0) {
      double all = 0.0;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) all += s_sum[i];
      parts[row * splits + split] = Part{all, Rc, mc};
    }
  }
  // ---- too many noted: the n-th of the threads' best among those kept (the larger element, then the lower number) is a higher bound.  n vectors reach it,
  // and whatever the threads that come behind have kept, four vectors each, is left behind: the loop ends.
  int count = s_count;
  while (count > kCap) {
    float bx = -INFINITY;
    int bi = 0x7fffffff;
    for (int j = tid; j < kCap; j += kThreads)
      if (before(s_x[j], s_i[j], bx, bi)) { bx = s_x[j]; bi = s_i[j]; }
    s_y[tid] = bx;
    s_j[tid] = bi;
    __syncthreads();
    if (rank_of(s_y, s_j, kThreads, tid, 1) == n - 1) s_best[0] = tid;
    if (tid == 0) s_count = 0;
    __syncthreads();
    bx = bound = s_y[s_best[0]];
    bi = s_j[s_best[0]];
    for (int v = v0 + tid; v < v1; v += kThreads) {
      const float top = top_of<T>(r.load(v));
      if (top > bx || (top == bx && v <= bi)) note(top, v);
    }
    __syncthreads();
    count = s_count;
    __syncthreads();
  }
  // ---- a second bound on the noted vectors, if they are many; if it leaves many, the n best of them
  const int* best = s_i;
  if (count > kFew) {
    float most = -INFINITY, all;
    for (int j = tid; j < count; j += kThreads) most = fmaxf(most, s_x[j]);
    bound = nth_group(most, n, s_group, s_bound, &all);
    for (int j = tid; j < count; j += kThreads)
      if (s_x[j] >= bound) {
        const int slot = atomicAdd(&s_kept, 1);
        s_y[slot] = s_x[j];
        s_j[slot] = s_i[j];
      }
    __syncthreads();
    count = s_kept;
    best = s_j;
    if (count > kFew) {
      for (int e = tid; e - tid < count; e += kThreads) {
        const int rank = rank_of(s_y, s_j, count, min(e, count - 1), 1);
        if (e < count && rank < n) {
          s_best[rank] = s_j[e];
          if (rank == n - 1) s_last = s_y[e];
        }
      }
      __syncthreads();
      count = n;
      best = s_best;
      bound = s_last;
    }
  }
  // ---- their elements that reach the bound, and the n best of those, sorted
  float y[2];
  int col[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {                               // kFew vectors of 8 elements, at most
    const int e = tid + u * kThreads;
    y[u] = -INFINITY;
    if (e < count * N) {
      col[u] = best[e / N] * N - r.lead + e % N;
      if (col[u] >= 0 && col[u] < V) y[u] = to_f32<T>(r.base[r.lead + col[u]]);
    }
  }
  __syncthreads();                                            // the noted vectors are done with
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (y[u] >= bound && y[u] > -INFINITY) {
      const int slot = atomicAdd(&s_elements, 1);
      s_x[slot] = y[u];
      s_i[slot] = col[u];
    }
  __syncthreads();
  count = s_elements;
  float2* list = lists + (row * splits + split) * n;
  const int per = threads_per(count, kThreads);
  for (int e0 = 0; e0 < count; e0 += kThreads / per) {
    const int e = e0 + tid / per, rank = rank_of(s_x, s_i, count, min(e, count - 1), per);
    if (e < count && rank < n && (tid & (per - 1)) == 0) list[rank] = make_float2(s_x[e], __int_as_float(s_i[e]));
  }
  if (tid >= count && tid < n) list[tid] = make_float2(-INFINITY, __int_as_float(-1));      // fewer elements than that
  }
  // ---- the sequence's last CTA merges
  __syncthreads();
  const int64_t b = row / K;
  if (tid == 0) {
    __threadfence();
    const unsigned all = (unsigned)(K * splits);
    s_mine = atomicInc(&counters[b], all - 1u) == all - 1u;   // back to zero with the last
    __threadfence();
  }
  __syncthreads();
  if (s_mine)
    merge(*reinterpret_cast<MergeSmem*>(s_both), s_group, s_bound, b, first_row + (int)(b * K), K, V, splits, scores + b * K, finished ? finished + b * K : nullptr, pad, n, parts + b * K * splits,
          lists + b * K * splits * n, out_scores, out_parents, out_tokens);
}

// Stretches of a row: as many CTAs as the device holds (four an SM), whole tiles of a CTA, and lists whose entries the merge takes in one step where that
// leaves any choice (7 x 11 beams of 128256, n = 29: 9 stretches 30.9 us, 3 23.5).
int row_splits(int64_t rows, int K, int64_t V, int dtype, int n) {
  const int64_t tile = kThreads * kVec * (dtype == TSB200_F32 ? 4 : 8);
  int64_t s = kSlots / rows;
  const int64_t cap = (V + tile - 1) / tile, room = kEntries / ((int64_t)K * n);
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
  const int64_t rows = (B < kCounters ? B : kCounters) * K, lists = rows * row_splits(rows, K, V, dtype, n);
  return (size_t)(kCounters * sizeof(unsigned) + lists * (int64_t)(sizeof(Part) + n * sizeof(float2)));
}

int tsb200_beam_select(const void* logits, int dtype, int64_t row_stride, int64_t B, int K, int64_t V, const float* scores, const uint8_t* finished,
                       int64_t pad_token, int n, float* out_scores, int32_t* out_parents, int64_t* out_tokens, void* workspace, size_t workspace_bytes,
                       void* stream) {
  TSB_REQUIRE_DEVICE();
  if (B < 0 || K <= 0 || V <= 0 || n <= 0) return TSB200_ERR_ARG;
  if (dtype != TSB200_F32 && dtype != TSB200_BF16) return TSB200_ERR_UNSUPPORTED;
  if (n > kMaxBest || K > kMaxBeams || B * K > 0x7fffffffLL || V > 0x7fffffffLL - 65536 || (int64_t)n > (int64_t)K * V) return TSB200_ERR_UNSUPPORTED;
  const int64_t stride = row_stride ? row_stride : V;
  if (stride < V) return TSB200_ERR_ARG;
  if (finished && (pad_token < 0 || pad_token >= V)) return TSB200_ERR_ARG;
  if (B == 0) return TSB200_OK;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !workspace || !aligned(workspace, 16)) return TSB200_ERR_ARG;
  if (!aligned(logits, dtype == TSB200_F32 ? 4 : 2)) return TSB200_ERR_ARG;
  if (workspace_bytes < tsb200_beam_select_workspace_bytes(B, K, V, dtype, n)) return TSB200_ERR_WORKSPACE;
  const int64_t step = B < kCounters ? B : kCounters;              // sequences of a launch
  const int splits = row_splits(step * K, K, V, dtype, n);
  if (step * K > 0x7fffffffLL / splits) return TSB200_ERR_UNSUPPORTED;
  const int per = dtype == TSB200_F32 ? 4 : 8;
  const int64_t vectors = (V + 2 * per - 2) / per;                 // a row may start inside a vector
  const int span = (int)((vectors + splits - 1) / splits);
  unsigned* counters = (unsigned*)workspace;
  Part* parts = (Part*)(counters + kCounters);
  float2* lists = (float2*)(parts + step * K * splits);
  for (int64_t b = 0; b < B; b += step) {
    const dim3 grid((unsigned)((B - b < step ? B - b : step) * K * splits));
    const uint8_t* fin = finished ? finished + b * K : nullptr;
    if (dtype == TSB200_F32)
      TSB_CUDA(launch_kernel(beam_select_kernel<float>, grid, dim3(kThreads), 0, as_stream(stream), (const float*)logits + b * K * stride, stride, K, (int)V, splits, span,
                             scores + b * K, fin, pad_token, n, parts, lists, counters, (int)(b * K), out_scores + b * n, out_parents + b * n, out_tokens + b * n));
    else
      TSB_CUDA(launch_kernel(beam_select_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, as_stream(stream), (const __nv_bfloat16*)logits + b * K * stride, stride, K,
                             (int)V, splits, span, scores + b * K, fin, pad_token, n, parts, lists, counters, (int)(b * K), out_scores + b * n, out_parents + b * n,
                             out_tokens + b * n));
  }
  return TSB200_OK;
}

}  // extern "C"
