// Rotate, quantize and append to pages that carry their own scale (kv_page.cuh).
//
//   y_t = rope(k_t) (fp32, each product and sum rounded once), v_t as given; per page and head, over the new tokens' finite elements,
//   e_new = smallest e with amax <= 448 * 2^e;  e = max(e_new, e_old) where the page held tokens before, else e_new;
//   code = e4m3(y / 2^e), old codes re-encoded where e > e_old (exact but for e4m3's subnormals).
// Slots behind the new tokens become zero.  Queries are rotated in place, rounded once to their type.
//
// Bytes: per token (2 H + 2 hkv) d sizeof(act) + 2 hkv d.  Chunks: a CTA owns a page, its warps take the records of K and V and the queries of
// 16 heads of a token in turn, each task's elements on their way into shared memory (cp.async) while the ones before are encoded.  One token
// per sequence: a warp per record, which touches of the page only what changes, bound by the chain length -> table -> page.
#include "kv_page.cuh"

namespace tsb {
namespace {

constexpr int kWarps = 8, kTaskHeads = 16;

struct AppendArgs {
  int64_t qs, ks, vs, T, rope_rows;
  int qheads, pages, zs;          // pages a sequence may touch, CTAs per page
  bool qvec, kvec, vvec;          // rows of the three are aligned for 16-byte accesses
};

__device__ __forceinline__ unsigned code2(float a, float b) {
  return (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ unsigned code4(float a, float b, float c, float d) { return code2(a, b) | (code2(c, d) << 16); }
// The four codes of a word times `ratio` (old scale over new: a power of two), encoded again.
__device__ __forceinline__ unsigned recode4(unsigned w, float ratio) {
  const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3)));
  const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
  return code4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}
// Bits of a word's bytes [from, to), its first byte being byte `at` of a row.
__device__ __forceinline__ unsigned byte_mask(int at, int from, int to) {
  const int a = min(max(from - at, 0), 4), b = min(max(to - at, 0), 4);
  const unsigned below_b = b == 4 ? 0xffffffffu : (1u << (8 * b)) - 1u, below_a = a == 4 ? 0xffffffffu : (1u << (8 * a)) - 1u;
  return below_b & ~below_a;
}
// x with what is infinite or not a number taken as zero: such elements do not set a scale.
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }

// N consecutive elements as fp32; vec: one access of up to 16 bytes.
template <typename T, int N>
__device__ __forceinline__ void load_elems(const T* __restrict__ p, bool vec, float* x) {
  constexpr int BYTES = N * (int)sizeof(T);
  alignas(16) T e[N];
  if (vec) {
    if constexpr (BYTES == 2) *reinterpret_cast<uint16_t*>(e) = *reinterpret_cast<const uint16_t*>(p);
    else if constexpr (BYTES == 4) *reinterpret_cast<unsigned*>(e) = *reinterpret_cast<const unsigned*>(p);
    else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
    else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = to_f32<T>(e[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_elems(T* __restrict__ p, bool vec, const float* x) {
  constexpr int BYTES = N * (int)sizeof(T);
  alignas(16) T e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = from_f32<T>(x[i]);
  if (vec) {
    if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
    else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = e[i];
  }
}
// N entries of a table's row (rows of d/2 floats, the tables 16-byte aligned).
template <int N>
__device__ __forceinline__ void load_table(float* x, const float* __restrict__ p) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) reinterpret_cast<float4*>(x)[i] = __ldg(reinterpret_cast<const float4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __ldg(p + i);
  }
}
// (a, b) -> (a cos - b sin, b cos + a sin) for N pairs: x[0 .. N) and x[N .. 2 N).
template <int N>
__device__ __forceinline__ void rotate(float* x, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float a = x[i], b = x[N + i];
    x[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
    x[N + i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
  }
}

// A chunk's page.  Tasks: the records of K, those of V, then 16 query heads of each of the page's tokens.
template <typename T, int D, int STAGES>
__global__ void __launch_bounds__(kWarps * 32, 2)
kv_append_page_kernel(tsb200_kv_desc kv, T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                      const int32_t* __restrict__ new_lens, const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, AppendArgs a) {
  // P: elements of a half that a lane of K and Q holds (its partners: the same of the other half); E: elements of V.
  constexpr int P = D / 16, HALF = D / 2, E = D / 32, REC = page_record_bytes(D);
  constexpr int ROW = D * (int)sizeof(T), STAGE = 16 * ROW;
  static_assert(kTaskHeads == 16, "a task's queries fill a stage");
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, piece = lane & 7, quad = lane >> 3;
  const int z = (int)(blockIdx.x % a.zs);
  const int64_t bn = blockIdx.x / a.zs;
  const int n = (int)(bn % a.pages);
  const int64_t b = bn / a.pages;
  const int64_t len = kv.seq_lens[b];
  int64_t count = a.T;
  if (new_lens) count = min(count, (int64_t)new_lens[b]);
  const int c = (int)(max(len, (int64_t)0) & 15);
  const int64_t j0 = (int64_t)n * 16 - c;                    // token of this page's slot 0
  if (count <= 0 || j0 >= count) return;
  const int64_t logical = (max(len, (int64_t)0) >> 4) + n;
  int64_t page = -1;
  if (len >= 0 && logical < kv.bt_stride) page = kv.block_table[b * kv.bt_stride + logical];
  const bool have = page >= 0 && page < kv.num_pages;
  const int first = n == 0 ? c : 0;                           // slots below hold older tokens
  const int last = (int)min((int64_t)16, count - j0);         // first slot without a token
  const int records = have ? 2 * kv.hkv : 0, per_token = q ? (a.qheads + kTaskHeads - 1) / kTaskHeads : 0;
  const int tasks = records + (last - first) * per_token;
  uint8_t* ring = smem + w * STAGES * STAGE;
  pdl_wait();
  // rows of task -> stage: tokens of K or V, heads of Q
  auto stage = [&](int task, int slot) {
    if (task < tasks) {
      const T* src;
      int64_t stride;
      int lo, hi;
      bool vec;
      if (task < records) {
        const bool is_v = task >= kv.hkv;
        stride = is_v ? a.vs : a.ks;
        vec = is_v ? a.vvec : a.kvec;
        src = (is_v ? v : k) + (b * a.T + j0) * stride + (int64_t)(is_v ? task - kv.hkv : task) * D;
        lo = first;
        hi = last;
      } else {
        const int t = task - records, h0 = t % per_token * kTaskHeads;
        src = q + (b * a.T + j0 + first + t / per_token) * a.qs + (int64_t)h0 * D;
        stride = D;
        vec = a.qvec;
        lo = 0;
        hi = min(kTaskHeads, a.qheads - h0);
      }
      uint8_t* dst = ring + slot * STAGE;
      if (vec) {
        constexpr int PER = ROW / 16;                         // 16-byte pieces of a row
#pragma unroll
        for (int i = 0; i < 16 * PER / 32; ++i) {
          const int idx = lane + i * 32, r = idx / PER;
          if (r >= lo && r < hi)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"((unsigned)__cvta_generic_to_shared(dst + idx * 16)),
                         "l"(reinterpret_cast<const uint8_t*>(src + r * stride) + idx % PER * 16)
                         : "memory");
        }
      } else {
        for (int i = lane; i < 16 * D; i += 32) {
          const int r = i / D;
          if (r >= lo && r < hi) reinterpret_cast<T*>(dst)[i] = src[r * stride + i % D];
        }
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  const int t0 = z * kWarps + w, step = a.zs * kWarps;
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) stage(t0 + i * step, i);
  int slot = 0;
  for (int task = t0; task < tasks; task += step) {
    stage(task + (STAGES - 1) * step, slot == 0 ? STAGES - 1 : slot - 1);
    asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 1) : "memory");
    __syncwarp();
    const T* rows = reinterpret_cast<const T*>(ring + slot * STAGE);
    if (task >= records) {
      const int t = task - records, h0 = t % per_token * kTaskHeads;
      const int64_t j = j0 + first + t / per_token, at = min(max(len + j, (int64_t)0), a.rope_rows - 1);
      float cs[P], sn[P];
      load_table<P>(cs, rope_cos + at * HALF + piece * P);
      load_table<P>(sn, rope_sin + at * HALF + piece * P);
      T* dst = q + (b * a.T + j) * a.qs + (int64_t)h0 * D + piece * P;
#pragma unroll
      for (int u = 0; u < kTaskHeads / 4; ++u) {
        const int h = quad + 4 * u;
        if (h0 + h < a.qheads) {
          float x[2 * P];
          load_elems<T, P>(rows + h * D + piece * P, true, x);
          load_elems<T, P>(rows + h * D + HALF + piece * P, true, x + P);
          rotate<P>(x, cs, sn);
          store_elems<T, P>(dst + h * D, a.qvec, x);
          store_elems<T, P>(dst + h * D + HALF, a.qvec, x + P);
        }
      }
    } else if (task < kv.hkv) {
      // ---- K: a lane holds 4 tokens x P elements of each half
      uint8_t* rec = kv.k_pool + (page * kv.hkv + task) * REC;
      const float old_scale = first ? *reinterpret_cast<const float*>(rec + 16 * D) : 0.f;
      float x[4][2 * P], m = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int r = 4 * quad + t;
        if (r >= first && r < last) {
          load_elems<T, P>(rows + r * D + piece * P, true, x[t]);
          load_elems<T, P>(rows + r * D + HALF + piece * P, true, x[t] + P);
          if (rope_cos) {
            const int64_t at = min(max(len + j0 + r, (int64_t)0), a.rope_rows - 1);
            float cs[P], sn[P];
            load_table<P>(cs, rope_cos + at * HALF + piece * P);
            load_table<P>(sn, rope_sin + at * HALF + piece * P);
            rotate<P>(x[t], cs, sn);
          }
#pragma unroll
          for (int i = 0; i < 2 * P; ++i) m = fmaxf(m, fabsf(x[t][i]));      // passes over NaN
        } else {
#pragma unroll
          for (int i = 0; i < 2 * P; ++i) x[t][i] = 0.f;
        }
      }
      m = warp_max(m);
      if (m == INFINITY) {
        m = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 2 * P; ++i) m = fmaxf(m, finite_abs(x[t][i]));
        m = warp_max(m);
      }
      int e = page_exponent(m);
      const int e_old = scale_exponent(old_scale);
      const bool grows = !first || e > e_old;
      if (!grows) e = e_old;
      const float inv = exp2_int(-e), ratio = exp2_int(max(e_old - e, -126));
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int r = 4 * quad + t;
        if (r < first && !grows) continue;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          unsigned* dst = reinterpret_cast<unsigned*>(rec + r * D + half * HALF + piece * P);
          const float* y = x[t] + half * P;
          unsigned word[P / 4];
#pragma unroll
          for (int i = 0; i < P / 4; ++i)
            word[i] = r < first ? recode4(dst[i], ratio) : code4(y[4 * i] * inv, y[4 * i + 1] * inv, y[4 * i + 2] * inv, y[4 * i + 3] * inv);
          if constexpr (P == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(word[0], word[1]);
          else *dst = word[0];
        }
      }
      if (grows && lane == 0) *reinterpret_cast<float*>(rec + 16 * D) = exp2_int(e);
    } else {
      // ---- V: a lane holds all 16 tokens of E elements, whole rows of the record
      uint8_t* rec = kv.v_pool + (page * kv.hkv + task - kv.hkv) * REC;
      const float old_scale = first ? *reinterpret_cast<const float*>(rec + 16 * D) : 0.f;
      uint4* dst = reinterpret_cast<uint4*>(rec + lane * E * 16);
      uint4 old[E];
#pragma unroll
      for (int i = 0; i < E; ++i) old[i] = first ? dst[i] : make_uint4(0u, 0u, 0u, 0u);
      float x[16][E], m = 0.f;
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        if (t >= first && t < last) {
          load_elems<T, E>(rows + t * D + lane * E, true, x[t]);
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) x[t][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) m = fmaxf(m, fabsf(x[t][i]));
      }
      m = warp_max(m);
      if (m == INFINITY) {
        m = 0.f;
#pragma unroll
        for (int t = 0; t < 16; ++t)
#pragma unroll
          for (int i = 0; i < E; ++i) m = fmaxf(m, finite_abs(x[t][i]));
        m = warp_max(m);
      }
      int e = page_exponent(m);
      const int e_old = scale_exponent(old_scale);
      const bool grows = !first || e > e_old;
      if (!grows) e = e_old;
      const float inv = exp2_int(-e), ratio = exp2_int(max(e_old - e, -126));
#pragma unroll
      for (int i = 0; i < E; ++i) {
        unsigned* o = reinterpret_cast<unsigned*>(&old[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned word = code4(x[4 * j][i] * inv, x[4 * j + 1][i] * inv, x[4 * j + 2][i] * inv, x[4 * j + 3][i] * inv);
          if (first) {
            const unsigned keep = byte_mask(4 * j, 0, first);
            o[j] = (word & ~keep) | ((grows ? recode4(o[j], ratio) : o[j]) & keep);
          } else {
            o[j] = word;
          }
        }
        dst[i] = old[i];
      }
      if (grows && lane == 0) *reinterpret_cast<float*>(rec + 16 * D) = exp2_int(e);
    }
    __syncwarp();                                             // the stage may be filled again
    slot = slot == STAGES - 1 ? 0 : slot + 1;
  }
}

// One token per sequence: a warp per record or four query heads.
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32)
kv_append_token_kernel(tsb200_kv_desc kv, T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const int32_t* __restrict__ new_lens,
                       const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, AppendArgs a) {
  constexpr int P = D / 16, HALF = D / 2, E = D / 32, REC = page_record_bytes(D);
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int records = 2 * kv.hkv, tasks = records + (q ? (a.qheads + 3) / 4 : 0);
  const int64_t task_b = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t b = task_b / tasks;
  const int task = (int)(task_b % tasks);
  if (b >= a.pages) return;                                   // one page a sequence: pages = sequences
  if (new_lens && new_lens[b] <= 0) return;
  const int64_t len = kv.seq_lens[b], at = min(max(len, (int64_t)0), a.rope_rows - 1);
  if (task >= records) {
    const int h = (task - records) * 4 + (lane >> 3), piece = lane & 7;
    if (h >= a.qheads) return;
    T* p = q + b * a.qs + (int64_t)h * D + piece * P;
    float cs[P], sn[P], x[2 * P];
    load_table<P>(cs, rope_cos + at * HALF + piece * P);
    load_table<P>(sn, rope_sin + at * HALF + piece * P);
    pdl_wait();
    load_elems<T, P>(p, a.qvec, x);
    load_elems<T, P>(p + HALF, a.qvec, x + P);
    rotate<P>(x, cs, sn);
    store_elems<T, P>(p, a.qvec, x);
    store_elems<T, P>(p + HALF, a.qvec, x + P);
    return;
  }
  if (len < 0 || (len >> 4) >= kv.bt_stride) return;
  const int64_t page = kv.block_table[b * kv.bt_stride + (len >> 4)];
  if (page < 0 || page >= kv.num_pages) return;
  const int c = (int)(len & 15);
  const bool is_v = task >= kv.hkv;
  const int h = is_v ? task - kv.hkv : task;
  uint8_t* rec = (is_v ? kv.v_pool : kv.k_pool) + (page * kv.hkv + h) * REC;
  // K: E / 2 elements of each half; V: E consecutive ones, whose rows of the record this lane rewrites
  float x[E], cs[E / 2], sn[E / 2];
  const bool rope = !is_v && rope_cos;
  if (rope) {
    load_table<E / 2>(cs, rope_cos + at * HALF + lane * (E / 2));
    load_table<E / 2>(sn, rope_sin + at * HALF + lane * (E / 2));
  }
  pdl_wait();
  const float old_scale = c ? *reinterpret_cast<const float*>(rec + 16 * D) : 0.f;
  unsigned old[E][4];
  if (is_v) {
    load_elems<T, E>(v + b * a.vs + (int64_t)h * D + lane * E, a.vvec, x);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const uint4 o = c ? reinterpret_cast<const uint4*>(rec)[lane * E + i] : make_uint4(0u, 0u, 0u, 0u);
      old[i][0] = o.x; old[i][1] = o.y; old[i][2] = o.z; old[i][3] = o.w;
    }
  } else {
    const T* p = k + b * a.ks + (int64_t)h * D + lane * (E / 2);
    load_elems<T, E / 2>(p, a.kvec, x);
    load_elems<T, E / 2>(p + HALF, a.kvec, x + E / 2);
    if (rope) rotate<E / 2>(x, cs, sn);
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) m = fmaxf(m, finite_abs(x[i]));
  m = warp_max(m);
  int e = page_exponent(m);
  const int e_old = scale_exponent(old_scale);
  const bool grows = !c || e > e_old;
  if (!grows) e = e_old;
  const float inv = exp2_int(-e), ratio = exp2_int(max(e_old - e, -126));
  if (is_v) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const unsigned code = code2(x[i] * inv, 0.f) & 0xffu;
      unsigned (&o)[4] = old[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (grows && 4 * j < c) o[j] = recode4(o[j], ratio);
        o[j] &= byte_mask(4 * j, 0, c);                        // what is behind becomes zero
        if (j == c >> 2) o[j] |= code << (8 * (c & 3));
      }
      reinterpret_cast<uint4*>(rec)[lane * E + i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else {
    if (grows)
      for (int i = lane; i < c * D / 16; i += 32) {            // the older tokens' rows
        uint4 o = reinterpret_cast<const uint4*>(rec)[i];
        o.x = recode4(o.x, ratio); o.y = recode4(o.y, ratio); o.z = recode4(o.z, ratio); o.w = recode4(o.w, ratio);
        reinterpret_cast<uint4*>(rec)[i] = o;
      }
    for (int i = (c + 1) * D / 16 + lane; i < D; i += 32) reinterpret_cast<uint4*>(rec)[i] = make_uint4(0u, 0u, 0u, 0u);
    uint8_t* row = rec + c * D + lane * (E / 2);
    if constexpr (E == 4) {
      *reinterpret_cast<uint16_t*>(row) = (uint16_t)code2(x[0] * inv, x[1] * inv);
      *reinterpret_cast<uint16_t*>(row + HALF) = (uint16_t)code2(x[2] * inv, x[3] * inv);
    } else {
      const unsigned w = code2(x[0] * inv, x[1] * inv);
      row[0] = (uint8_t)w;
      row[HALF] = (uint8_t)(w >> 8);
    }
  }
  if (grows && lane == 0) *reinterpret_cast<float*>(rec + 16 * D) = exp2_int(e);
}

}  // namespace

template <typename T, int D>
int launch_append_page(const tsb200_kv_desc& kv, void* q, int64_t qs, int qheads, const void* k, const void* v, int64_t ks, int64_t vs, int64_t B,
                       int64_t Tn, const int32_t* new_lens, const float* rc, const float* rs, int64_t rr, cudaStream_t s) {
  if (rc && (!aligned(rc, 16) || !aligned(rs, 16))) return TSB200_ERR_ARG;
  AppendArgs a;
  a.qs = qs; a.ks = ks; a.vs = vs; a.T = Tn; a.rope_rows = rr; a.qheads = qheads;
  auto rows_aligned = [](const void* p, int64_t stride) { return aligned(p, 16) && stride * sizeof(T) % 16 == 0; };
  a.qvec = rows_aligned(q, qs);
  a.kvec = rows_aligned(k, ks);
  a.vvec = rows_aligned(v, vs);
  if (Tn == 1) {
    const int64_t warps = B * (2 * (int64_t)kv.hkv + (q ? (qheads + 3) / 4 : 0)), blocks = (warps + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffffLL || B > 0x7fffffffLL) return TSB200_ERR_UNSUPPORTED;
    a.pages = (int)B;
    a.zs = 1;
    TSB_CUDA(launch_kernel(kv_append_token_kernel<T, D>, dim3((unsigned)blocks), dim3(kWarps * 32), 0, s, kv, (T*)q, (const T*)k, (const T*)v, new_lens, rc,
                           rs, a));
    return TSB200_OK;
  }
  constexpr int STAGES = sizeof(T) == 2 ? 3 : 2;
  constexpr size_t smem = (size_t)kWarps * STAGES * 16 * D * sizeof(T);
  static bool configured[64] = {false};
  int dev = 0;
  TSB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TSB200_ERR_DEVICE;
  if (!configured[dev]) {
    TSB_CUDA(cudaFuncSetAttribute(kv_append_page_kernel<T, D, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured[dev] = true;
  }
  const int64_t pages = (Tn + 14) / 16 + 1;
  const int64_t tasks = 2 * (int64_t)kv.hkv + (q ? (Tn < 16 ? Tn : 16) * ((qheads + kTaskHeads - 1) / kTaskHeads) : 0);
  int64_t zs = 592 / (pages * B);                              // short chunks: a page's tasks over several CTAs
  if (zs > (tasks + kWarps - 1) / kWarps) zs = (tasks + kWarps - 1) / kWarps;
  if (zs < 1) zs = 1;
  if (pages > 0x7fffffffLL || pages * B * zs > 0x7fffffffLL) return TSB200_ERR_UNSUPPORTED;
  a.pages = (int)pages;
  a.zs = (int)zs;
  TSB_CUDA(launch_kernel(kv_append_page_kernel<T, D, STAGES>, dim3((unsigned)(pages * B * zs)), dim3(kWarps * 32), smem, s, kv, (T*)q, (const T*)k,
                         (const T*)v, new_lens, rc, rs, a));
  return TSB200_OK;
}
#define TSB_INST(TT, DD)                                                                                                                              \
  template int launch_append_page<TT, DD>(const tsb200_kv_desc&, void*, int64_t, int, const void*, const void*, int64_t, int64_t, int64_t, int64_t, \
                                          const int32_t*, const float*, const float*, int64_t, cudaStream_t);
TSB_INST(float, 64)
TSB_INST(float, 128)
TSB_INST(__nv_bfloat16, 64)
TSB_INST(__nv_bfloat16, 128)
#undef TSB_INST

}  // namespace tsb
