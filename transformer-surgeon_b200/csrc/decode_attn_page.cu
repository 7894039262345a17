// Split-K paged decode attention over e4m3 pages that carry their own scales (kv_page.cuh):
//   out[h] = sum_t p_t V_t / sum_t p_t,  p_t = exp(sm_scale q_h . K_t),  K_t = 2^eK code, V_t = 2^eV code,  e per page.
// The codes go to the tensor cores as they are (mma.sync m16n8k32 e4m3).  The scale of V joins the exponent:
//   w_t = 2^(s_t + eV - M) <= 1,  numerator sum w_t code_t,  denominator sum w_t 2^-eV   (s_t in bits, M the running maximum of s_t + eV),
// so that pages of any scales share one accumulator.
// q and w are fed as sums of e4m3 terms, each 16 times finer than the one before (term t stands for code / 16^t): bf16 queries are two terms
// exactly and weights keep 8 bits, fp32 takes four terms, 16 bits.  The 16 rows of an MMA are 8 heads x 2 terms or 4 heads x 4 terms, the tokens
// of K and the elements of V its columns: a softmax row stays in the four lanes that feed the second product, and its weights are that
// product's operand as they are.
#include "tc_common.cuh"
#include "decode_attn_common.cuh"
#include "kv_page.cuh"

namespace tsb {
namespace {

using tc::mbar_expect_tx;
using tc::mbar_init;
using tc::mbar_try_wait;
using tc::smem_u32;

constexpr int kWarps = 6;
constexpr int kStages = 2;                  // page pairs in a warp's ring
constexpr unsigned kWaitLimit = 1u << 22;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void bulk_g2s(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void mma_e4m3(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(unsigned (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// Nearest e4m3 codes of four values, in one word; on return y holds 16 times what they leave over.
__device__ __forceinline__ unsigned take_term(float (&y)[4]) {
  const unsigned short lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
  const unsigned short hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
  const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(lo, __NV_E4M3)));
  const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(hi, __NV_E4M3)));
  y[0] = (y[0] - a.x) * 16.f;
  y[1] = (y[1] - a.y) * 16.f;
  y[2] = (y[2] - b.x) * 16.f;
  y[3] = (y[3] - b.y) * 16.f;
  return (unsigned)lo | ((unsigned)hi << 16);
}
// The words of rows gid and gid + 8: terms 0 and 1, or (four terms) 0 and 1 in even rows, 2 and 3 in odd ones.
template <int TERMS>
__device__ __forceinline__ void terms_of_rows(float (&y)[4], bool odd, unsigned& row, unsigned& row8) {
  row = take_term(y);
  row8 = take_term(y);
  if constexpr (TERMS == 4) {
    const unsigned t2 = take_term(y), t3 = take_term(y);
    if (odd) { row = t2; row8 = t3; }
  }
}
// Sum over a head's terms of an accumulator's rows gid (hi) and gid + 8 (lo).
template <int TERMS>
__device__ __forceinline__ float add_terms(float hi, float lo, bool odd) {
  float v = fmaf(lo, 1.f / 16.f, hi);
  if constexpr (TERMS == 4) {
    if (odd) v *= 1.f / 256.f;
    v += __shfl_xor_sync(0xffffffffu, v, 4);
  }
  return v;
}

template <typename T, int D>
struct Cfg {
  static constexpr int TERMS = sizeof(T) == 2 ? 2 : 4, HEADS = 16 / TERMS;
  static constexpr int REC = page_record_bytes(D), STAGE = 4 * REC;            // K_A, V_A, K_B, V_B
  static constexpr int RING = kStages * STAGE;
  static constexpr size_t SMEM = (size_t)kWarps * RING + kWarps * kStages * 8;
  static_assert((size_t)kWarps * HEADS * (2 + D) * sizeof(float) <= (size_t)kWarps * RING, "the merge stays clear of the barriers");
};

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32, 2)
decode_attn_page_kernel(tsb200_kv_desc kv, const T* __restrict__ q, int64_t qs, int H, int chunks, float sm_scale, int64_t max_seq_len, int S,
                        float* __restrict__ ws, T* __restrict__ out, int* __restrict__ status) {
  using C = Cfg<T, D>;
  constexpr int TERMS = C::TERMS, HEADS = C::HEADS, REC = C::REC;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int gid = lane >> 2, tid = lane & 3;
  const bool odd = gid & 1;
  const int ch = (int)(blockIdx.x % chunks), s = blockIdx.y;
  const int64_t bh = blockIdx.x / chunks;
  const int hk = (int)(bh % kv.hkv);
  const int64_t b = bh / kv.hkv;
  const int g = H / kv.hkv, g0 = ch * HEADS, gn = min(HEADS, g - g0);

  uint8_t* ring = smem + (size_t)w * C::RING;
  unsigned long long* bars = reinterpret_cast<unsigned long long*>(smem + (size_t)kWarps * C::RING) + w * kStages;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();
  // Lanes 0 .. 3 copy one record each: K and V of a pair's first page, K and V of its second.
  const int64_t rec_stride = (int64_t)kv.hkv * REC;
  const uint8_t* pool = ((lane & 1) ? kv.v_pool : kv.k_pool) + (int64_t)hk * REC;
  auto copy = [&](int stage, int records, int page) {
    if (lane == 0) mbar_expect_tx(&bars[stage], (unsigned)(records * REC));
    __syncwarp();
    if (lane < records) {
      const int64_t at = page < 0 ? 0 : (page >= kv.num_pages ? kv.num_pages - 1 : page);
      bulk_g2s(ring + stage * C::STAGE + lane * REC, pool + at * rec_stride, REC, &bars[stage]);
    }
  };
  pdl_wait();
  int len = kv.seq_lens[b];
  len = len < 0 ? 0 : (len > max_seq_len ? (int)max_seq_len : len);
  int pb, pe;
  split_range(len, s, S, pb, pe);
  // this warp's pages: pb + w, pb + w + kWarps, ...; consecutive two form a pair (one ring stage)
  const int n_pages = pe - pb - w > 0 ? (pe - pb - w + kWarps - 1) / kWarps : 0;
  const int n_pairs = (n_pages + 1) / 2;
  const int32_t* table = kv.block_table + b * kv.bt_stride + pb + w;
  auto look_up = [&](int pair) {
    const int idx = 2 * pair + (lane >> 1);
    return lane < 4 && idx < n_pages ? table[idx * kWarps] : 0;
  };
  auto issue = [&](int pair, int page) {
    if (pair < n_pairs) copy(pair % kStages, 2 * pair + 1 < n_pages ? 4 : 2, page);
  };
  issue(0, look_up(0));
  int next_page = look_up(1);

  // ---- the query as the first product's operand: k-step 2 c + u of a lane covers elements 16 (tid + 4 c) + 8 u + [0, 8)
  unsigned qf[D / 32][4];
  float scf;                                                 // raw sum -> score in bits
  {
    const int head = TERMS == 2 ? gid : gid >> 1;
    float x[D / 64][16];
    const T* qp = q + b * qs + (int64_t)(hk * g + g0 + head) * D;
    const bool vec = ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(qs * (int64_t)sizeof(T))) & 15) == 0;
    float amax = 0.f;
    bool finite = true;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const T* p = qp + 16 * (tid + 4 * c);
      if (head < gn && vec) {
        alignas(16) T e[16];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[c][i] = to_f32<T>(e[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[c][i] = head < gn ? to_f32<T>(p[i]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        amax = fmaxf(amax, fabsf(x[c][i]));
        finite = finite && fabsf(x[c][i]) < INFINITY;
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // the largest element to [128, 256): a power of two, so that no bit is lost
    const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 126);
    const float up = exp2_int(min(7 - e, 127));
    scf = finite ? exp2_int(max(e - 7, -126)) * sm_scale * kLog2e : __int_as_float(0x7fc00000);
    scf += __shfl_xor_sync(0xffffffffu, scf, 1) * 0.f;       // not a number in one lane: in the whole row
    scf += __shfl_xor_sync(0xffffffffu, scf, 2) * 0.f;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = x[c][8 * u + 4 * r + i] * up;
          terms_of_rows<TERMS>(y, odd, qf[2 * c + u][2 * r], qf[2 * c + u][2 * r + 1]);
        }
  }

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  bool ok = true;
  for (int pair = 0; pair < n_pairs; ++pair) {
    issue(pair + 1, next_page);
    next_page = look_up(pair + 2);
    {
      unsigned spins = 0;
      while (!mbar_try_wait(&bars[pair % kStages], (pair / kStages) & 1)) {
        if (++spins > kWaitLimit) { ok = false; break; }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
    }
    const uint8_t* st = ring + (pair % kStages) * C::STAGE;
    const bool two = 2 * pair + 1 < n_pages;
    // ---- scores of tokens 4 tid .. + 3 of both pages, in bits, with the exponent of the page's V scale
    float sv[2][4], iv[2] = {0.f, 0.f};
    float mx = -INFINITY;
#pragma unroll
    for (int X = 0; X < 2; ++X) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sv[X][i] = -INFINITY;
      if (X == 0 || two) {
        const uint8_t* sK = st + X * 2 * REC;
        const int nt = len - (pb + w + (2 * pair + X) * kWarps) * 16;       // tokens left from this page on
        float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // column n of n-tile j: token 4 (n / 2) + 2 j + n % 2, so that a lane's four columns are consecutive tokens
          const uint8_t* row = sK + (4 * (gid >> 1) + 2 * j + (gid & 1)) * D;
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            const uint4 kk = *reinterpret_cast<const uint4*>(row + 16 * (tid + 4 * h));
            mma_e4m3(c[j], qf[2 * h], kk.x, kk.y);
            mma_e4m3(c[j], qf[2 * h + 1], kk.z, kk.w);
          }
        }
        const float ks = scf * *reinterpret_cast<const float*>(sK + 16 * D);
        const int ev = scale_exponent(*reinterpret_cast<const float*>(sK + REC + 16 * D));
        iv[X] = exp2_int(-ev);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = add_terms<TERMS>(c[i >> 1][i & 1], c[i >> 1][2 + (i & 1)], odd);
          if (4 * tid + i < nt) sv[X][i] = fmaf(v, ks, (float)ev);
          mx = fmaxf(mx, sv[X][i]);
        }
      }
    }
    // ---- online softmax: a row's maximum over its four lanes
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float mn = fmaxf(m_run, mx), ref = mn == -INFINITY ? 0.f : mn;
    const float corr = ex2(m_run - ref);
    const bool rescale = __any_sync(0xffffffffu, mn != m_run);
    m_run = mn;
    l_run *= corr;
    unsigned pf[4];
#pragma unroll
    for (int X = 0; X < 2; ++X) {
      float y[4], sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = ex2(sv[X][i] - ref);
        sum += y[i];
      }
      l_run = fmaf(sum, iv[X], l_run);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] *= 256.f;
      terms_of_rows<TERMS>(y, odd, pf[2 * X], pf[2 * X + 1]);
    }
    // ---- O += w V: k-slots 4 tid .. + 3 are tokens 4 tid .. + 3 of the first page, the upper sixteen those of the second
    if (rescale) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) { o[i][0] *= corr; o[i][1] *= corr; o[i][2] *= corr; o[i][3] *= corr; }
    }
    const uint8_t* sV = st + REC + lane * 16;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      unsigned va[4], vb[4] = {0u, 0u, 0u, 0u};
      ldmatrix4(va, sV + i * 512);
      if (two) ldmatrix4(vb, sV + 2 * REC + i * 512);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_e4m3(o[4 * i + j], pf, va[j], vb[j]);
    }
    __syncwarp();     // all lanes are done with this stage before it is refilled
  }
  if (!ok) {
    // a wait ran out: give the copies in flight a bounded time to land before shared memory is reused, and record it
    if (lane == 0 && status) atomicMax(status, 8);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }

  // ---- the warps' results meet in shared memory
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
  __syncthreads();
  float* sm_m = reinterpret_cast<float*>(smem);              // [warps][HEADS]
  float* sm_l = sm_m + kWarps * HEADS;
  float* sm_acc = sm_l + kWarps * HEADS;                     // [warps][HEADS][D]
  const int head = TERMS == 2 ? gid : gid >> 1;
  if (tid == 0 && (TERMS == 2 || !odd)) {
    sm_m[w * HEADS + head] = m_run;
    sm_l[w * HEADS + head] = l_run;
  }
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const float a0 = add_terms<TERMS>(o[i][0], o[i][2], odd), a1 = add_terms<TERMS>(o[i][1], o[i][3], odd);
    if (TERMS == 2 || !odd) *reinterpret_cast<float2*>(sm_acc + (size_t)(w * HEADS + head) * D + 8 * i + 2 * tid) = make_float2(a0, a1);
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < gn * D; idx += blockDim.x) {
    const int i = idx / D, e = idx % D;
    float mm = -INFINITY;
#pragma unroll
    for (int ww = 0; ww < kWarps; ++ww) mm = fmaxf(mm, sm_m[ww * HEADS + i]);
    float ll = 0.f, acc = 0.f;
#pragma unroll
    for (int ww = 0; ww < kWarps; ++ww) {
      const float mw = sm_m[ww * HEADS + i];
      const float c = mw == -INFINITY ? 0.f : exp2f(mw - mm);
      ll = fmaf(sm_l[ww * HEADS + i], c, ll);
      acc = fmaf(sm_acc[(size_t)(ww * HEADS + i) * D + e], c, acc);
    }
    acc *= 1.f / 256.f;
    const int64_t oh = b * H + hk * g + g0 + i;
    if (S == 1) {
      out[oh * D + e] = from_f32<T>(len > 0 ? acc / ll : 0.f);
    } else {
      float* p = ws + (oh * S + s) * (2 + D);
      if (e == 0) { p[0] = mm * 0.6931471805599453f; p[1] = ll; }
      p[2 + e] = acc;
    }
  }
}

template <typename T, int D>
int launch(const tsb200_kv_desc& kv, const void* q, int64_t qs, int H, float sm_scale, int64_t max_seq_len, int S, int64_t B, float* ws, void* out,
           int* status, cudaStream_t st) {
  using C = Cfg<T, D>;
  static bool configured[64] = {false};
  int dev = 0;
  TSB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TSB200_ERR_DEVICE;
  if (!configured[dev]) {
    TSB_CUDA(cudaFuncSetAttribute(decode_attn_page_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
    configured[dev] = true;
  }
  const int g = H / kv.hkv, chunks = (g + C::HEADS - 1) / C::HEADS;
  if (B * kv.hkv * chunks > 0x7fffffffLL) return TSB200_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)(B * kv.hkv * chunks), (unsigned)S);
  TSB_CUDA(launch_kernel_if(attn_overlaps(kv), decode_attn_page_kernel<T, D>, grid, dim3(kWarps * 32), C::SMEM, st, kv, (const T*)q, qs, H, chunks, sm_scale,
                            max_seq_len, S, ws, (T*)out, status));
  return S == 1 ? TSB200_OK : launch_reduce<T, D>(ws, B * H, S, out, st);
}

}  // namespace

int choose_splits_page(int64_t B, int hkv, int64_t max_seq_len) {
  const int64_t base = B * hkv, pages = (max_seq_len + 15) / 16;
  int64_t s = base > 0 ? (2 * 296 + base - 1) / base : 1;
  const int64_t cap = pages / 24 > 0 ? pages / 24 : 1;
  if (s > cap) s = cap;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

int launch_attn_page(const tsb200_kv_desc& kv, const void* q, void* out, int dtype, int64_t qs, int64_t B, int H, float sm_scale, int64_t max_seq_len,
                     float* ws, int* status, cudaStream_t st) {
  const int S = choose_splits_page(B, kv.hkv, max_seq_len);
  if (dtype == TSB200_F32)
    return kv.head_dim == 64 ? launch<float, 64>(kv, q, qs, H, sm_scale, max_seq_len, S, B, ws, out, status, st)
                             : launch<float, 128>(kv, q, qs, H, sm_scale, max_seq_len, S, B, ws, out, status, st);
  return kv.head_dim == 64 ? launch<__nv_bfloat16, 64>(kv, q, qs, H, sm_scale, max_seq_len, S, B, ws, out, status, st)
                           : launch<__nv_bfloat16, 128>(kv, q, qs, H, sm_scale, max_seq_len, S, B, ws, out, status, st);
}

}  // namespace tsb
