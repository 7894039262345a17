// Rotate, quantize and append to pages that carry their own scale (kv_page.cuh).
//
//   y_t = rope(k_t) (fp32, each product and sum rounded once), v_t as given; per page and head, over the new tokens' finite elements,
//   e_new = smallest e with amax <= 448 * 2^e;  e = max(e_new, e_old) where the page held tokens before, else e_new;
//   code = e4m3(y / 2^e), old codes re-encoded where e > e_old (exact but for e4m3's subnormals).
// Slots behind the new tokens become zero.  Queries are rotated in place, rounded once to their type.
//
// Bytes: per token (2 H + 2 hkv) d sizeof(act) + 2 hkv d.  One warp owns one (page, head) record of K or V or the queries of one token.
// A lane holds 4 tokens x (d/16 elements of the first half + their partners of the second), so that a rotation needs no other lane and
// four tokens of an element are one word of the token-minor V record.
#include "kv_page.cuh"

namespace tsb {
namespace {

// PIECE consecutive elements as fp32; `vec`: the address is aligned for one 8-, 16- or 2 x 16-byte access.
template <typename T, int PIECE>
__device__ __forceinline__ void load_piece(const T* __restrict__ p, bool vec, float* x) {
  constexpr int BYTES = PIECE * (int)sizeof(T);
  if (vec) {
    alignas(16) T e[PIECE];
    if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
    }
#pragma unroll
    for (int i = 0; i < PIECE; ++i) x[i] = to_f32<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < PIECE; ++i) x[i] = to_f32<T>(p[i]);
  }
}
template <typename T, int PIECE>
__device__ __forceinline__ void store_piece(T* __restrict__ p, bool vec, const float* x) {
  constexpr int BYTES = PIECE * (int)sizeof(T);
  alignas(16) T e[PIECE];
#pragma unroll
  for (int i = 0; i < PIECE; ++i) e[i] = from_f32<T>(x[i]);
  if (vec) {
    if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
    } else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < PIECE; ++i) p[i] = e[i];
  }
}
// (a, b) -> (a cos - b sin, b cos + a sin) for PIECE pairs: x[0 .. PIECE) and x[PIECE .. 2 PIECE).
template <int PIECE>
__device__ __forceinline__ void rotate(float* x, const float* __restrict__ cosr, const float* __restrict__ sinr) {
  float c[PIECE], s[PIECE];
#pragma unroll
  for (int i = 0; i < PIECE / 4; ++i) {      // tables are fp32 rows of d/2, checked for 16-byte alignment on the host
    reinterpret_cast<float4*>(c)[i] = __ldg(reinterpret_cast<const float4*>(cosr) + i);
    reinterpret_cast<float4*>(s)[i] = __ldg(reinterpret_cast<const float4*>(sinr) + i);
  }
#pragma unroll
  for (int i = 0; i < PIECE; ++i) {
    const float a = x[i], b = x[PIECE + i];
    x[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
    x[PIECE + i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
  }
}
__device__ __forceinline__ unsigned code4(float a, float b, float c, float d) {
  const unsigned lo = (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const unsigned hi = (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float code_value(unsigned c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3);
  return __half2float(__half(h));
}

struct AppendArgs {
  int64_t qs, ks, vs, T, rope_rows;
  int qheads, pages, zs;          // pages a sequence may touch, CTAs per page
  bool qvec, kvec, vvec;
};

template <typename T, int D>
__global__ void __launch_bounds__(256)
kv_append_page_kernel(tsb200_kv_desc kv, T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                      const int32_t* __restrict__ new_lens, const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, AppendArgs a) {
  constexpr int P = D / 16, HALF = D / 2, REC = page_record_bytes(D);
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, piece = lane & 7, quad = lane >> 3;     // elements [piece * P, +P) of each half, tokens 4 quad ..
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
  const int records = 2 * kv.hkv, tasks = records + (q ? last - first : 0);
  pdl_wait();
  for (int task = z * 8 + (threadIdx.x >> 5); task < tasks; task += a.zs * 8) {
    if (task >= records) {                                    // the queries of one token, four heads at a time
      const int64_t j = j0 + first + (task - records);
      const int64_t at = min(max(len + j, (int64_t)0), a.rope_rows - 1);
      T* row = q + (b * a.T + j) * a.qs;
      for (int h = quad; h < a.qheads; h += 4) {
        T* p = row + (int64_t)h * D + piece * P;
        float x[2 * P];
        load_piece<T, P>(p, a.qvec, x);
        load_piece<T, P>(p + HALF, a.qvec, x + P);
        rotate<P>(x, rope_cos + at * HALF + piece * P, rope_sin + at * HALF + piece * P);
        store_piece<T, P>(p, a.qvec, x);
        store_piece<T, P>(p + HALF, a.qvec, x + P);
      }
      continue;
    }
    if (!have) continue;
    const bool is_v = task >= kv.hkv;
    const int h = is_v ? task - kv.hkv : task;
    const T* src = (is_v ? v : k) + (int64_t)h * D + piece * P;
    const int64_t stride = is_v ? a.vs : a.ks;
    const bool vec = is_v ? a.vvec : a.kvec;
    uint8_t* rec = (is_v ? kv.v_pool : kv.k_pool) + (page * kv.hkv + h) * REC;
    const float old_scale = first ? *reinterpret_cast<const float*>(rec + 16 * D) : 0.f;
    float x[4][2 * P];                                        // [token 4 quad + t][element]
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int slot = 4 * quad + t;
      if (slot >= first && slot < last) {
        const T* p = src + (b * a.T + j0 + slot) * stride;
        load_piece<T, P>(p, vec, x[t]);
        load_piece<T, P>(p + HALF, vec, x[t] + P);
      } else {
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) x[t][i] = 0.f;
      }
    }
    if (!is_v && rope_cos) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int64_t at = min(max(len + j0 + 4 * quad + t, (int64_t)0), a.rope_rows - 1);
        rotate<P>(x[t], rope_cos + at * HALF + piece * P, rope_sin + at * HALF + piece * P);
      }
    }
    float m = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 2 * P; ++i) m = fmaxf(m, fabsf(x[t][i]));          // passes over NaN
    m = warp_max(m);
    if (m == INFINITY) {                                      // infinite elements saturate and do not set the scale
      m = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) m = fmaxf(m, fabsf(x[t][i]) == INFINITY ? 0.f : fabsf(x[t][i]));
      m = warp_max(m);
    }
    int e = page_exponent(m);
    const int e_old = scale_exponent(old_scale);
    const bool keep = first && e <= e_old;                    // older codes stay as they are: the new tokens' alone are written
    if (keep) e = e_old;
    const float inv = exp2_int(-e);
    if (first && !keep) {                                     // the scale grew: the older tokens' values join the new ones
      const float s_old = exp2_int(e_old);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int slot = 4 * quad + t;
        if (slot < first) {
#pragma unroll
          for (int i = 0; i < 2 * P; ++i) {
            const int el = (i < P ? piece * P + i : HALF + piece * P + i - P);
            x[t][i] = code_value(is_v ? rec[el * 16 + slot] : rec[slot * D + el]) * s_old;
          }
        }
      }
    }
    __syncwarp();                                             // every lane has read what others are about to write
    if (!is_v) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int slot = 4 * quad + t;
        if (keep && slot < first) continue;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float* y = x[t] + half * P;
          uint8_t* dst = rec + slot * D + half * HALF + piece * P;
#pragma unroll
          for (int i = 0; i < P; i += 4)
            reinterpret_cast<unsigned*>(dst)[i / 4] = code4(y[i] * inv, y[i + 1] * inv, y[i + 2] * inv, y[i + 3] * inv);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2 * P; ++i) {
        const int el = (i < P ? piece * P + i : HALF + piece * P + i - P);
        const unsigned w = code4(x[0][i] * inv, x[1][i] * inv, x[2][i] * inv, x[3][i] * inv);
        uint8_t* dst = rec + el * 16 + 4 * quad;
        if (!keep || 4 * quad >= first) {
          *reinterpret_cast<unsigned*>(dst) = w;
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (4 * quad + t >= first) dst[t] = (uint8_t)(w >> (8 * t));
        }
      }
    }
    if (!keep && lane == 0) *reinterpret_cast<float*>(rec + 16 * D) = exp2_int(e);
  }
}

}  // namespace

template <typename T, int D>
int launch_append_page(const tsb200_kv_desc& kv, void* q, int64_t qs, int qheads, const void* k, const void* v, int64_t ks, int64_t vs, int64_t B,
                       int64_t Tn, const int32_t* new_lens, const float* rc, const float* rs, int64_t rr, cudaStream_t s) {
  if (rc && (!aligned(rc, 16) || !aligned(rs, 16))) return TSB200_ERR_ARG;
  constexpr int piece_bytes = D / 16 * (int)sizeof(T);
  constexpr size_t al = piece_bytes < 16 ? piece_bytes : 16;
  AppendArgs a;
  a.qs = qs; a.ks = ks; a.vs = vs; a.T = Tn; a.rope_rows = rr; a.qheads = qheads;
  a.qvec = aligned(q, al) && qs * sizeof(T) % al == 0;
  a.kvec = aligned(k, al) && ks * sizeof(T) % al == 0;
  a.vvec = aligned(v, al) && vs * sizeof(T) % al == 0;
  const int64_t pages = (Tn + 14) / 16 + 1;
  const int64_t tasks = 2 * (int64_t)kv.hkv + (q ? (Tn < 16 ? Tn : 16) : 0);
  int64_t zs = 592 / (pages * B);
  if (zs > (tasks + 7) / 8) zs = (tasks + 7) / 8;
  if (zs < 1) zs = 1;
  if (pages > 0x7fffffffLL || pages * B * zs > 0x7fffffffLL) return TSB200_ERR_UNSUPPORTED;
  a.pages = (int)pages;
  a.zs = (int)zs;
  TSB_CUDA(launch_kernel(kv_append_page_kernel<T, D>, dim3((unsigned)(pages * B * zs)), dim3(256), 0, s, kv, (T*)q, (const T*)k, (const T*)v, new_lens, rc,
                         rs, a));
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
