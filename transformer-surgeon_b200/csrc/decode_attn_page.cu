// Split-K paged decode attention over e4m3 pages that carry their own scales (kv_page.cuh):
//   out[h] = sum_t p_t V_t / sum_t p_t,  p_t = exp(sm_scale q_h . K_t),  K_t = 2^eK code, V_t = 2^eV code,  e per page.
// The scale of V joins the exponent:
//   w_t = 2^(s_t + eV - M + 8),  numerator sum w_t code_t,  denominator sum w_t 2^-eV   (s_t in bits; M is at most 6 below the largest s_t + eV so far),
// so that pages of any scales share one accumulator and the maximum moves rarely.  The largest w of a head lies between 2^8 and 2^14; a w keeps the bits that
// are said below down to 2^-14, 22 bits under it at least, and is nothing below 2^-25 (two terms: 2^-36).  So an element's error is that share of the head's largest
// w code, also where the pages of large w hold zeros in that element.
// Products run on warp-level f16 MMAs (m16n8k16), whose 16 rows are a page's tokens (elements of V) and whose 8 columns are query heads: 8 of bf16
// (a query scaled by a power of two is an f16 number, weights keep 11 bits), 4 of fp32 in two f16 terms, code and rest * 2^11 (22 bits).  The
// codes are widened to f16 pairs, one conversion for two; the e4m3 form of the MMA does the same in every instruction, to both operands: 425
// instructions for a page of 128, 305 here.  A word of four codes is a k-step of the first product and half a row of the second, with the
// tokens of both in the order that makes the transposed weights (movmatrix) the second one's operand.
//
// Work: the pages of all sequences in one row, cut into equal ranges, each for as many CTAs as there are kv heads, together as many as the device holds,
// and each of those into equal ranges of its warps.  A warp streams its pages through a private ring (cp.async.bulk, K and V record) that does not
// drain between sequences; a sequence that lies in one warp's range is done there, one that crosses warps is put together in shared memory
// at the CTA's end, one that crosses ranges by a second launch (by the last of its CTAs: 5 us longer, one CTA then waits for every step of that alone).
// So, where sequences are cut (whole_is_faster), lengths of any mixture keep every SM busy to the end, and the heads of a page, neighbours in memory, are read
// at about the same time (64 x 8192 tokens, 8 heads, pages in random order: 5.5 TB/s where they were not).
#include "tc_common.cuh"
#include "decode_attn_common.cuh"
#include "kv_page.cuh"

namespace tsb {
namespace {

using tc::mbar_expect_tx;
using tc::mbar_init;
using tc::mbar_try_wait;
using tc::smem_u32;

// Two CTAs of six warps with three pages each an SM (64 x 8192 tokens, 32 / 8 heads, 139 us; five warps and four pages 141, six and four, which
// leaves the larger parts of more than four heads one CTA, 147, seven and three 146, eight and three 166).
constexpr int NW = 6;
constexpr int kStages = 3;                  // pages in a warp's ring
constexpr int kSlots = 296;                 // CTAs that the device holds: two an SM
constexpr int kMaxRows = 1024;              // sequences of a launch
constexpr unsigned kMinPages = 6;           // of a range: one for every warp
constexpr unsigned kWaitLimit = 1u << 22;
constexpr float kAhead = 6.f, kUp = 8.f;    // bits a score may be above M; bits weights are scaled up by (2^14 at most in f16)
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void bulk_g2s(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transposed(unsigned x) {     // of an 8 x 8 matrix of f16, a pair a lane
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
// Four e4m3 codes -> f16 pairs (first, second) and (third, fourth).
__device__ __forceinline__ void widen(unsigned w, unsigned& a, unsigned& b) {
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.rn.f16x2.e4m3x2 %0, lo;\ncvt.rn.f16x2.e4m3x2 %1, hi;\n}\n" : "=r"(a), "=r"(b) : "r"(w));
}
__device__ __forceinline__ void ldmatrix4(unsigned (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// x = hi + lo * 2^-11 in f16.
__device__ __forceinline__ unsigned two_terms(float x) {
  const float hi = __half2float(__float2half_rn(x));
  return pack_f16(hi, (x - hi) * 2048.f);
}

// Pages of sequence b.
__device__ __forceinline__ int pages_of(const tsb200_kv_desc& kv, int64_t b, int64_t max_seq_len) {
  const int64_t len = min((int64_t)kv.seq_lens[b], max_seq_len);
  return len <= 0 ? 0 : (int)((len + 15) >> 4);
}
// Pages of a range.  per_min bounds the number of ranges that a sequence can lie in.  (The launch's pages fit 31 bits.)
__device__ __forceinline__ unsigned range_pages(unsigned total, unsigned ranges, unsigned per_min) { return max((total + ranges - 1) / ranges, per_min); }

struct PageArgs {
  int64_t qs, max_seq_len;
  unsigned per_min;
  int B, H, chunks, heads;        // heads: query heads that a CTA takes of a kv head's, in so many chunks (the last may have fewer)
  int S;                          // partials of a (sequence, head) in the workspace; 0: ranges end where sequences end
  float sm_scale;
};

// Position in the row: page p of n of sequence b, `left` pages to go (this one among them).
struct Cursor {
  int b, p, n, left;
};

template <typename T, int D>
struct Cfg {
  static constexpr int HEADS = sizeof(T) == 2 ? 8 : 4;
  static constexpr int REC = page_record_bytes(D), STAGE = 2 * REC;            // K, V
  static constexpr int RING = kStages * STAGE;
  static size_t smem(int heads, int B) {
    return (size_t)NW * (RING + heads * (2 + D) * sizeof(float) + kStages * 8) + (size_t)B * sizeof(int);
  }
  static_assert(HEADS * (2 + D) * (int)sizeof(float) <= RING, "a warp's last partial fits its ring");
};

template <typename T, int D>
__global__ void __launch_bounds__(NW * 32, 2)
decode_attn_page_kernel(tsb200_kv_desc kv, const T* __restrict__ q, PageArgs a, float* __restrict__ ws, T* __restrict__ out, int* __restrict__ status) {
  using C = Cfg<T, D>;
  constexpr int HEADS = C::HEADS, REC = C::REC;
  constexpr bool kTwo = HEADS == 4;                          // columns are two terms of a head
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_scan[NW];
  // parts of a warp: of a sequence that began before its range (0), of one that goes on behind it (1): the sequence (or -1), and the place of
  // this CTA's part among the sequence's
  __shared__ int2 s_part[2][NW];
  __shared__ unsigned s_ends;                                // warps in whose range the sequence of part 0 ends
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int gid = lane >> 2, tid = lane & 3;
  const int column_head = kTwo ? gid >> 1 : gid;             // of the CTA's, as the columns of both products' operands
  const int g = a.H / kv.hkv, HU = kv.hkv * a.chunks;
  const int range = (int)blockIdx.x / HU, ranges = (int)gridDim.x / HU, uh = (int)blockIdx.x % HU;
  const int hk = uh / a.chunks, h0 = uh % a.chunks * HEADS, gn = min(HEADS, g - h0);       // this CTA's heads: gn from hk g + h0 on
  const int PART = a.heads * (2 + D);                        // floats of a partial: (m, l) per head, then the sums

  uint8_t* ring = smem + (size_t)w * C::RING;
  float* parts = reinterpret_cast<float*>(smem + (size_t)NW * C::RING);           // [warps][PART]: of a sequence that began before the warp's range
  unsigned long long* bars = reinterpret_cast<unsigned long long*>(parts + NW * PART) + w * kStages;
  int* cum = reinterpret_cast<int*>(reinterpret_cast<unsigned long long*>(parts + NW * PART) + NW * kStages);   // pages of the sequences up to and with b
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    s_part[0][w].x = s_part[1][w].x = -1;
    if (w == 0) s_ends = 0u;
  }
  // Lengths and block table are inputs that the launch directly before this one does not write (see the header): looked up ahead of the wait.
  // Where ranges end with sequences, a CTA counts its own alone.
  const int each = (a.B + ranges - 1) / ranges, s0 = a.S ? 0 : min(range * each, a.B), s1 = a.S ? a.B : min(s0 + each, a.B);
  int before = 0;
  for (int b0 = s0; b0 < s1; b0 += NW * 32) {
    const int b = b0 + (int)threadIdx.x;
    int v = b < s1 ? pages_of(kv, b, a.max_seq_len) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) s_scan[w] = v;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if (i < w) v += s_scan[i];
      total += s_scan[i];
    }
    if (b < s1) cum[b] = before + v;
    before += total;
    __syncthreads();
  }
  const unsigned P = (unsigned)before;
  auto start_of = [&](int b) { return (unsigned)(b > s0 ? cum[b - 1] : 0); };
  unsigned c0, c1, per = 0;
  if (a.S) {
    per = range_pages(P, ranges, a.per_min);
    c0 = min((uint64_t)P, (uint64_t)range * per);
    c1 = min((uint64_t)P, (uint64_t)c0 + per);
  } else {
    c0 = 0;
    c1 = P;
  }
  Cursor at;
  {
    const unsigned each = (c1 - c0) / NW, rest = (c1 - c0) % NW;
    const unsigned x0 = c0 + w * each + min((unsigned)w, rest);
    at.left = (int)(each + ((unsigned)w < rest));
    at.b = at.p = at.n = 0;
    if (at.left > 0) {
      // first sequence that ends behind x0: which 32, which of them
      const int i0 = min(s0 + 32 * lane + 31, s1 - 1);
      int lo = s0 + 32 * (__ffs(__ballot_sync(0xffffffffu, (unsigned)cum[i0] > x0)) - 1);
      lo += __ffs(__ballot_sync(0xffffffffu, (unsigned)cum[min(lo + lane, s1 - 1)] > x0)) - 1;
      at.b = lo;
      at.p = (int)(x0 - start_of(lo));
      at.n = cum[lo] - (int)start_of(lo);
    }
  }
  auto advance = [&](Cursor& c) {
    --c.left;
    if (++c.p == c.n && c.left > 0) {
      c.p = 0;
      do ++c.b; while (cum[c.b] == cum[c.b - 1]);             // left > 0: there is one with pages
      c.n = cum[c.b] - cum[c.b - 1];
    }
  };

  // Lanes 0 and 1 copy K and V.  Page numbers are looked up 32 at a time, one a lane.
  Cursor ahead = at;
  int next_stage = 0, numbers = 0, first_number = 0, numbered = -1;       // of pages first_number .. of sequence `numbered`
  const int64_t rec_stride = (int64_t)kv.hkv * REC;
  const uint8_t* pool = (lane ? kv.v_pool : kv.k_pool) + (int64_t)hk * REC;
  auto look_up = [&]() {
    if (ahead.left > 0 && (ahead.b != numbered || ahead.p - first_number >= 32)) {
      numbered = ahead.b;
      first_number = ahead.p;
      numbers = lane < ahead.n - ahead.p ? kv.block_table[ahead.b * kv.bt_stride + ahead.p + lane] : 0;
    }
  };
  auto issue = [&]() {
    if (ahead.left > 0) {
      const int page = __shfl_sync(0xffffffffu, numbers, ahead.p - first_number);
      if (lane == 0) mbar_expect_tx(&bars[next_stage], 2 * REC);
      __syncwarp();
      if (lane < 2) {
        const int64_t pg = page < 0 ? 0 : (page >= kv.num_pages ? kv.num_pages - 1 : page);
        bulk_g2s(ring + next_stage * C::STAGE + lane * REC, pool + pg * rec_stride, REC, &bars[next_stage]);
      }
      next_stage = next_stage == kStages - 1 ? 0 : next_stage + 1;
      advance(ahead);
      look_up();
    }
  };
  // Elements of the column's query: 16 (tid + 4 c) + [0, 16)
  T qraw[D / 64][16];
  const bool qvec = ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(a.qs * (int64_t)sizeof(T))) & 15) == 0;
  auto load_query = [&](int b) {
    const bool there = column_head < gn;
    const T* qp = q + b * a.qs + (int64_t)(hk * g + h0 + column_head) * D + 16 * tid;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (there && qvec) {
          v = *reinterpret_cast<const uint4*>(qp + 64 * c + i * (16 / (int)sizeof(T)));
        } else if (there) {
          alignas(16) T e[16 / sizeof(T)];
#pragma unroll
          for (int j = 0; j < 16 / (int)sizeof(T); ++j) e[j] = qp[64 * c + i * (16 / (int)sizeof(T)) + j];
          v = *reinterpret_cast<const uint4*>(e);
        }
        *reinterpret_cast<uint4*>(&qraw[c][i * (16 / (int)sizeof(T))]) = v;
      }
  };
  look_up();
  // Pages strictly older than a sequence's newest are written by no append before this launch: their copies leave while those launches finish.
  int started = 0;
  for (; started < kStages - 1 && ahead.left > 0 && ahead.p + 1 < ahead.n; ++started) issue();
  pdl_wait();     // q and the newest token's pages come from the launches before
  if (at.left > 0) load_query(at.b);
  for (; started < kStages - 1; ++started) issue();

  unsigned qf[D / 16][2];         // k-step 4 c + r: elements 16 (tid + 4 c) + 4 r + {0, 1}, {2, 3}
  float scf[2];                   // raw sum -> score in bits, of the heads whose scores this lane holds: 2 tid and 2 tid + 1, or tid
  float o[D / 16][4];
  float m_run[2], l_run[2];
  int p_first = 0, len = 0;
  bool fresh = true, loaded = true, ok = true;
  int stage = 0;
  unsigned parity = 0;

  while (at.left > 0) {
    issue();
    if (fresh) {
      if (!loaded) load_query(at.b);
      fresh = loaded = false;
      p_first = at.p;
      len = (int)min((int64_t)kv.seq_lens[at.b], a.max_seq_len);
      float amax = 0.f;
      bool finite = true;
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = fabsf(to_f32<T>(qraw[c][i]));
          amax = fmaxf(amax, x);
          finite = finite && x < INFINITY;
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // the largest element to [128, 256), by a power of two
      const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 126);
      const float up = exp2_int(min(7 - e, 127));
      float sc = finite ? exp2_int(max(e - 7, -126)) * a.sm_scale * kLog2e : __int_as_float(0x7fc00000);
      sc += __shfl_xor_sync(0xffffffffu, sc, 1) * 0.f;       // not a number in one lane: in the whole column
      sc += __shfl_xor_sync(0xffffffffu, sc, 2) * 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        scf[i] = __shfl_sync(0xffffffffu, sc, 4 * (2 * tid + (kTwo ? 0 : i)));
        m_run[i] = -INFINITY;
        l_run[i] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float x0 = to_f32<T>(qraw[c][4 * r + 2 * i]) * up, x1 = to_f32<T>(qraw[c][4 * r + 2 * i + 1]) * up;
            if constexpr (kTwo) {
              const unsigned t0 = two_terms(x0), t1 = two_terms(x1);
              qf[4 * c + r][i] = __byte_perm(t0, t1, gid & 1 ? 0x7632 : 0x5410);
            } else {
              qf[4 * c + r][i] = pack_f16(x0, x1);
            }
          }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    }
    {
      unsigned spins = 0;
      while (!mbar_try_wait(&bars[stage], parity)) {
        if (++spins > kWaitLimit) { ok = false; break; }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
    }
    const uint8_t* sK = ring + stage * C::STAGE;
    const uint8_t* sV = sK + REC;
    const int nt = len - at.p * 16;                           // tokens from this page on
    if (nt < 16) {
      // codes behind the sequence's end may be anything, and a weight of zero does not take a NaN away (32 x 2100 tokens 26.0 -> 26.3 us; masks on the
      // second product's operands 27.5)
      uint4* rows = reinterpret_cast<uint4*>(ring + stage * C::STAGE + REC);
      unsigned m[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) m[j] = nt >= 4 * j + 4 ? ~0u : nt <= 4 * j ? 0u : (1u << (8 * (nt - 4 * j))) - 1u;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint4 x = rows[lane + 32 * i];
        x.x &= m[0]; x.y &= m[1]; x.z &= m[2]; x.w &= m[3];
        rows[lane + 32 * i] = x;
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
    }
    // ---- scores: row r of the tile's upper half is token 4 (r / 2) + r % 2, of its lower half the one two behind
    float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
    const int token = 4 * (gid >> 1) + (gid & 1);
    {
      const uint8_t* row = sK + token * D + 16 * tid;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const uint4 ka = *reinterpret_cast<const uint4*>(row + 64 * c);
        const uint4 kb = *reinterpret_cast<const uint4*>(row + 2 * D + 64 * c);
        const unsigned wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          unsigned a0, a1, a2, a3;
          widen(wa[r], a0, a2);
          widen(wb[r], a1, a3);
          mma_f16(r & 1 ? c1 : c0, a0, a1, a2, a3, qf[4 * c + r][0], qf[4 * c + r][1]);
        }
      }
    }
    const float ks = *reinterpret_cast<const float*>(sK + 16 * D);
    const int ev = scale_exponent(*reinterpret_cast<const float*>(sV + 16 * D));
    const bool in0 = token < nt, in1 = token + 2 < nt;
    // sv[half][head]: of the lane's two heads, or (two terms) the one
    constexpr int N = kTwo ? 1 : 2;
    float sv[2][N];
    bool above = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float f = scf[i] * ks;
      const float lo = kTwo ? fmaf(c0[1] + c1[1], 1.f / 2048.f, c0[0] + c1[0]) : c0[i] + c1[i];
      const float hi = kTwo ? fmaf(c0[3] + c1[3], 1.f / 2048.f, c0[2] + c1[2]) : c0[2 + i] + c1[2 + i];
      sv[0][i] = in0 ? fmaf(lo, f, (float)ev) : -INFINITY;
      sv[1][i] = in1 ? fmaf(hi, f, (float)ev) : -INFINITY;
      above = above || fmaxf(sv[0][i], sv[1][i]) > m_run[i] + kAhead;
    }
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float mx = fmaxf(sv[0][i], sv[1][i]);
#pragma unroll
        for (int of = 4; of < 32; of <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, of));
        mx = fmaxf(mx, m_run[i]);
        const float corr = mx == -INFINITY ? 1.f : ex2(m_run[i] - mx);
        m_run[i] = mx;
        l_run[i] *= corr;
        // accumulators of this lane: columns 2 tid and 2 tid + 1 (two terms: both of head tid)
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[j][i] *= corr;
          o[j][2 + i] *= corr;
          if (kTwo) { o[j][1] *= corr; o[j][3] *= corr; }
        }
      }
    }
    const float iv = exp2_int(-ev);
    float w0[N], w1[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float ref = (m_run[i] == -INFINITY ? 0.f : m_run[i]) - kUp;
      w0[i] = ex2(sv[0][i] - ref);
      w1[i] = ex2(sv[1][i] - ref);
      l_run[i] = fmaf(w0[i] + w1[i], iv, l_run[i]);
    }
    const unsigned b0 = transposed(kTwo ? two_terms(w0[0]) : pack_f16(w0[0], w0[N - 1]));
    const unsigned b1 = transposed(kTwo ? two_terms(w1[0]) : pack_f16(w1[0], w1[N - 1]));
    // ---- sums over the page's tokens: k-slots 2 tid, 2 tid + 1, 2 tid + 8, 2 tid + 9 are tokens 4 tid .. + 3
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      unsigned va[4];
      ldmatrix4(va, sV + lane * 16 + i * 512);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        unsigned a0, a1, a2, a3;
        widen(va[2 * j], a0, a2);
        widen(va[2 * j + 1], a1, a3);
        mma_f16(o[2 * i + j], a0, a1, a2, a3, b0, b1);
      }
    }
    __syncwarp();     // all lanes are done with this stage before it is refilled
    if (++stage == kStages) { stage = 0; parity ^= 1; }
    // ---- the sequence's last page in this range
    if (at.left == 1 || at.p + 1 == at.n) {
      fresh = true;
      const bool begins = p_first == 0, ends = at.p + 1 == at.n;
      float* part = begins ? reinterpret_cast<float*>(ring) : parts + w * PART;   // one that goes on is the range's last: its ring is empty
      if (!(begins && ends) && lane == 0) {
        s_part[begins][w] = make_int2(at.b, a.S ? range - (int)(start_of(at.b) / per) : 0);
        if (ends) atomicOr(&s_ends, 1u << w);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int of = 4; of < 32; of <<= 1) l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], of);
      }
      T* dst = out + ((int64_t)at.b * a.H + hk * g + h0) * D;
      // accumulators of head tid (two terms), or of heads 2 tid and 2 tid + 1; rows are elements 16 j + gid and + 8
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int h = kTwo ? tid : 2 * tid + i;
        if (h >= gn) continue;
        const float inv = 1.f / l_run[i];
        if (!(begins && ends) && gid == 0) *reinterpret_cast<float2*>(part + 2 * h) = make_float2(m_run[i], l_run[i]);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          const float x0 = kTwo ? fmaf(o[j][1], 1.f / 2048.f, o[j][0]) : o[j][i], x1 = kTwo ? fmaf(o[j][3], 1.f / 2048.f, o[j][2]) : o[j][2 + i];
          if (begins && ends) {
            dst[h * D + 16 * j + gid] = from_f32<T>(x0 * inv);
            dst[h * D + 16 * j + 8 + gid] = from_f32<T>(x1 * inv);
          } else {
            part[2 * a.heads + h * D + (16 * j + gid + 8 * tid) % D] = x0;        // turned by 8 elements a lane of the quad: no bank twice
            part[2 * a.heads + h * D + (16 * j + 8 + gid + 8 * tid) % D] = x1;
          }
        }
      }
    }
    advance(at);
  }
  if (!ok) {
    // a wait ran out: give the copies in flight a bounded time to land before shared memory is reused, and record it
    if (lane == 0 && status) atomicMax(status, 8);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  __syncthreads();

  // ---- sequences that cross warps.  A chain starts with a part of the second kind, or with the CTA's first part if that is of the first kind.
  const int unit0 = lane < NW ? s_part[0][lane].x : -1, unit1 = lane < NW ? s_part[1][lane].x : -1;
  const unsigned with0 = __ballot_sync(0xffffffffu, unit0 >= 0), with1 = __ballot_sync(0xffffffffu, unit1 >= 0), ending = s_ends;
  const int lead = with0 && !(with1 & ((with0 & -with0) - 1u)) ? __ffs(with0) - 1 : -1;
  int task = 0;
#pragma unroll 1
  for (unsigned starts = with1 << 1 | (lead >= 0); starts; starts &= starts - 1) {
    const int f = __ffs(starts) - 2;                         // -1: the lead
    const int fw = f < 0 ? lead : f;
    const int2 info = s_part[f >= 0][fw];
    unsigned members = f < 0 && (ending >> fw & 1) ? 0u : __ballot_sync(0xffffffffu, unit0 == info.x && lane > fw);
    const unsigned last = members & ending;                  // the sequence's last part
    if (last) members &= (last << 1) - 1u;
    const bool done = f >= 0 && last;
    const float* first = f < 0 ? parts + fw * PART : reinterpret_cast<const float*>(smem + (size_t)fw * C::RING);
#pragma unroll 1
    for (int h = 0; h < gn; ++h) {
      if (task++ % NW != w) continue;
      // lane i: the part of warp i, lane NW: the first
      float2 ml = make_float2(-INFINITY, 0.f);
      if (lane == NW || (members >> lane & 1)) ml = *reinterpret_cast<const float2*>((lane == NW ? first : parts + lane * PART) + 2 * h);
      const float mm = warp_max(ml.x);
      const float c = ml.x == -INFINITY ? 0.f : ex2(ml.x - mm);
      const float ll = warp_sum(ml.y * c);
      const int turn = 8 * (kTwo ? h : h >> 1);
      float acc[D / 32];
      const float cf = __shfl_sync(0xffffffffu, c, NW);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = first[2 * a.heads + h * D + (lane + 32 * i + turn) % D] * cf;
#pragma unroll
      for (int j = 1; j < NW; ++j) {
        const float cj = __shfl_sync(0xffffffffu, c, j);
        if (members >> j & 1) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(parts[j * PART + 2 * a.heads + h * D + (lane + 32 * i + turn) % D], cj, acc[i]);
        }
      }
      const int64_t oh = (int64_t)info.x * a.H + hk * g + h0 + h;
      if (done) {
        const float inv = 1.f / ll;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) out[oh * D + lane + 32 * i] = from_f32<T>(acc[i] * inv);
      } else {
        float* p = ws + (oh * a.S + info.y) * (2 + D);
        if (lane == 0) *reinterpret_cast<float2*>(p) = make_float2(mm, ll);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) p[2 + lane + 32 * i] = acc[i];
      }
    }
  }
  // ---- sequences without tokens
  for (int b = s0 + (a.S ? (int)blockIdx.x : 0); b < s1; b += a.S ? (int)gridDim.x : 1)
    if (cum[b] == (int)start_of(b)) {
      if (a.S) {                                             // of all heads; where ranges end with sequences, of the CTA's own
        for (int i = threadIdx.x; i < a.H * D; i += NW * 32) out[(int64_t)b * a.H * D + i] = from_f32<T>(0.f);
      } else {
        for (int i = threadIdx.x; i < gn * D; i += NW * 32) out[((int64_t)b * a.H + hk * g + h0) * D + i] = from_f32<T>(0.f);
      }
    }
}

// One CTA per (sequence, head), one thread per element: adds up the parts of a sequence that crosses ranges, in order.  Chained to the attention.
template <typename T, int D>
__global__ void __launch_bounds__(D)
decode_attn_page_join_kernel(tsb200_kv_desc kv, PageArgs a, int ranges, const float* __restrict__ ws, T* __restrict__ out) {
  __shared__ int s_sum[2][D / 32];
  __shared__ float s_c[64], s_l;
  pdl_launch_dependents();
  const int t = threadIdx.x;
  const int64_t oh = blockIdx.x;
  const int b = (int)(oh / a.H);
  int before = 0, all = 0;
  for (int i = t; i < a.B; i += D) {
    const int n = pages_of(kv, i, a.max_seq_len);
    all += n;
    before += i < b ? n : 0;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  all = __reduce_add_sync(0xffffffffu, all);
  if ((t & 31) == 0) { s_sum[0][t >> 5] = before; s_sum[1][t >> 5] = all; }
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) { before += s_sum[0][i]; all += s_sum[1][i]; }
  const int n = pages_of(kv, b, a.max_seq_len);
  const unsigned per = range_pages((unsigned)all, ranges, a.per_min), start = (unsigned)before;
  const int count = n == 0 ? 0 : (int)((start + n - 1) / per - start / per) + 1;
  pdl_wait();
  if (count < 2) return;
  // all parts' sums on their way while the coefficients are made
  const float* p = ws + oh * a.S * (2 + D);
  constexpr int kFly = 16;
  float v[kFly];
#pragma unroll
  for (int i = 0; i < kFly; ++i)
    if (i < count) v[i] = __ldcg(p + (int64_t)i * (2 + D) + 2 + t);
  if (t < 32) {
    float2 ml[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      if (t + 32 * i < count) ml[i] = __ldcg(reinterpret_cast<const float2*>(p + (int64_t)(t + 32 * i) * (2 + D)));
    }
    const float mm = warp_max(fmaxf(ml[0].x, ml[1].x));
    float ll = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float c = ml[i].x == -INFINITY ? 0.f : ex2(ml[i].x - mm);
      s_c[t + 32 * i] = c;
      ll = fmaf(ml[i].y, c, ll);
    }
    ll = warp_sum(ll);
    if (t == 0) s_l = ll;
  }
  __syncthreads();
  float acc = 0.f;
  for (int i0 = 0; i0 < count; i0 += kFly) {
#pragma unroll
    for (int i = 0; i < kFly; ++i)
      if (i0 + i < count) acc = fmaf(v[i], s_c[i0 + i], acc);
#pragma unroll
    for (int i = 0; i < kFly; ++i)
      if (i0 + kFly + i < count) v[i] = __ldcg(p + (int64_t)(i0 + kFly + i) * (2 + D) + 2 + t);
  }
  out[oh * D + t] = from_f32<T>(acc / s_l);
}

template <typename T, int D>
int launch(tsb200_kv_desc kv, const T* q, PageArgs a, int64_t B, float* ws, T* out, int* status, cudaStream_t st) {
  using C = Cfg<T, D>;
  static bool configured[64] = {false};
  int dev = 0;
  TSB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TSB200_ERR_DEVICE;
  if (!configured[dev]) {
    TSB_CUDA(cudaFuncSetAttribute(decode_attn_page_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::smem(C::HEADS, kMaxRows)));
    configured[dev] = true;
  }
  const int64_t units = (int64_t)kv.hkv * a.chunks, pages = (a.max_seq_len + 15) / 16;
  const int64_t rows = pages > 0 && 0x7fffffffLL / pages < kMaxRows ? 0x7fffffffLL / pages : kMaxRows;
  if (rows < 1) return TSB200_ERR_UNSUPPORTED;
  for (int64_t b = 0; b < B; b += rows) {
    a.B = (int)(B - b < rows ? B - b : rows);
    // two CTAs an SM, and no more than there can be ranges
    const int64_t most = a.S ? (pages * a.B + a.per_min - 1) / a.per_min : a.B;
    int64_t ranges = kSlots / units;
    if (ranges > most) ranges = most;
    if (ranges < 1) ranges = 1;
    TSB_CUDA(launch_kernel_if(attn_overlaps(kv), decode_attn_page_kernel<T, D>, dim3((unsigned)(ranges * units)), dim3(NW * 32), C::smem(a.heads, a.B), st, kv, q, a, ws,
                              out, status));
    if (a.S)
      TSB_CUDA(launch_kernel_if(true, decode_attn_page_join_kernel<T, D>, dim3((unsigned)(a.B * a.H)), dim3(D), 0, st, kv, a, (int)ranges, (const float*)ws, out));
    kv.block_table += a.B * kv.bt_stride;
    kv.seq_lens += a.B;
    q += a.B * a.qs;
    out += (int64_t)a.B * a.H * D;
  }
  return TSB200_OK;
}

// Whole sequences, if the most pages that a warp then gets are not many more than in equal ranges: the parts of cut ones cost a launch, about as long as
// a warp takes for five pages (whole / cut, us: 58 sequences x 575 tokens, 8 kv heads, 3 pages more: 19.1 / 21.3; 68 x 2076, 4 heads, 3: 30.7 / 32.6; 4 x 519,
// 2 heads, 6: 8.1 / 7.4; 92 x 1660, 2 heads, 8: 22.0 / 18.7; 5 x 1491, 2 heads, 16: 17.7 / 8.5; two chunks of fp32 heads: 40 x 600, 14 / 2, 4: 9.4 / 11.0;
// 74 x 1500, 14 / 2, 1: 16.9 / 17.7; 64 x 2080, 28 / 4, 7: 46.2 / 45.3; 50 x 900, 28 / 4, 8: 24.4 / 23.4).  Lengths are known to the device alone: all count
// as the longest.  Where the others are far shorter, whole is the wrong choice (37 x 4096 at most, 8 heads, one of them that long and the rest 100
// tokens: 38.9 / 13.7; 32 x 2100, half to all: 26.5 / 27.5).  units: CTAs that share a range.
bool whole_is_faster(int64_t B, int64_t units, int64_t pages) {
  const int64_t ranges = units < kSlots ? kSlots / units : 1;
  const int64_t whole = (B + ranges - 1) / ranges * ((pages + NW - 1) / NW), cut = B * pages / (ranges * NW);
  return whole - cut <= 5;
}

template <typename T, int D>
int launch_for(const tsb200_kv_desc& kv, const void* q, PageArgs a, int64_t B, float* ws, void* out, int* status, cudaStream_t st) {
  constexpr int HEADS = Cfg<T, D>::HEADS;
  const int g = a.H / kv.hkv;
  a.chunks = (g + HEADS - 1) / HEADS;
  a.heads = g < HEADS ? g : HEADS;
  if ((int64_t)kMaxRows * a.H > 0x7fffffffLL) return TSB200_ERR_UNSUPPORTED;
  const int64_t pages = (a.max_seq_len + 15) / 16;
  if (whole_is_faster(B, (int64_t)kv.hkv * a.chunks, pages)) a.S = 0;
  if (a.S) {
    a.per_min = (unsigned)((pages + a.S - 3) / (a.S - 2));
    if (a.per_min < kMinPages) a.per_min = kMinPages;
  }
  return launch<T, D>(kv, (const T*)q, a, B, ws, (T*)out, status, st);
}

}  // namespace

int launch_attn_page(const tsb200_kv_desc& kv, const void* q, void* out, int dtype, int64_t qs, int64_t B, int H, float sm_scale, int64_t max_seq_len,
                     float* ws, size_t ws_bytes, int* status, cudaStream_t st) {
  PageArgs a = {};
  a.qs = qs;
  a.max_seq_len = max_seq_len;
  a.H = H;
  a.sm_scale = sm_scale;
  // A sequence lies in at most S ranges: no more than the workspace has room for.  Sequences of a few pages stay whole.
  const int64_t pages = (max_seq_len + 15) / 16, room = (int64_t)(ws_bytes / ((size_t)(B * H) * (2 + kv.head_dim) * sizeof(float)));
  int64_t S = pages / 4 < 64 ? pages / 4 : 64;
  if (S > room) S = room;
  a.S = S < 3 ? 0 : (int)S;
  if (dtype == TSB200_F32)
    return kv.head_dim == 64 ? launch_for<float, 64>(kv, q, a, B, ws, out, status, st) : launch_for<float, 128>(kv, q, a, B, ws, out, status, st);
  return kv.head_dim == 64 ? launch_for<__nv_bfloat16, 64>(kv, q, a, B, ws, out, status, st)
                           : launch_for<__nv_bfloat16, 128>(kv, q, a, B, ws, out, status, st);
}

}  // namespace tsb
