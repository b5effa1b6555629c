// Attention with a decay for each head in chunks of 128 steps on the tensor
// cores (formulas: decay_attention.cuh). One CTA walks the chunks of one
// (batch row, head, segment); with S the carry, per chunk
//
//   P = (Q K^T) * g^|r-j| on the causal side      O  = P V + W_out Q S
//   D = (W_kv K)^T V                               S <- g^n S + c D
//
// Four matrix products on tcgen05 (M = 128), everything else on the way between
// tensor memory and shared memory:
//
//   warp 0     copies: Q (one buffer), K and V (two each), 128-byte swizzle
//   warp 1     issues the products, one thread
//   warps 2-5  scores (TMEM) -> P (16 bits, back into TMEM as an A operand);
//              K -> W_kv K in place, and what rounding left of it into a second
//              buffer, so that D is good to 2^-16 of its terms
//   warps 6-9  outputs; the carry in fp32 registers (thread = row of S), rounded
//              into shared memory as the next chunk's operand
//
// What bounds it: the bytes of q, k, v and o (one read, one write) while there
// are enough (row, head) pairs for the SMs; per chunk of 128 x 128 heads that is
// 128 KB or 5.6 thousand cycles of one SM's share of the copy bandwidth, against
// about 2.6 thousand for the products and 2 thousand for either group of warps.
#include <cuda.h>
#include <math.h>

#include <cstring>
#include <type_traits>

#include "async_copy.cuh"
#include "decay_attention.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace mb {
namespace {

constexpr int kC = 128;  // steps per chunk: the M of one product
constexpr int kTcThreads = 320;
constexpr int kBlockBytes = kC * 128;  // 64 columns x 128 steps of 16 bits
constexpr int64_t kTcMinSteps = 16;    // below: the recurrent kernel

struct TcArgs {
  mb_decay_attention_args a;
  AttnSplit split;
  // whether a dimension's coordinate counts (0: the tensor is broadcast along it)
  int32_t q_b, q_h, k_b, k_h, v_b, v_h;
};

template <int DK, int DV>
struct TcLayout {
  static constexpr int kQBytes = kC * DK * 2;
  static constexpr int kVBytes = kC * DV * 2;
  static constexpr int kSBytes = DK * DV * 2;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kQBytes;       // two stages
  static constexpr int kLo = kK + 2 * kQBytes;  // rounding remainders of W_kv K
  static constexpr int kV = kLo + kQBytes;      // two stages
  static constexpr int kS = kV + 2 * kVBytes;
  static constexpr int kTables = kS + kSBytes;
  static constexpr int kPow = kTables;                  // g^n, n = 0..128
  static constexpr int kWeights = kPow + 132 * 4;       // weights of the scores by distance
  static constexpr int kRowScale = kWeights + 256 * 4;  // fp16: 1 / scale of P's rows, two chunks
  static constexpr int kMax = kRowScale + 2 * kC * 4;    // fp16: largest carry of each warp
  static constexpr int kBars = kMax + 32;
  static constexpr int kNumBars = 15;
  static constexpr size_t kSmem = kBars + kNumBars * 8 + 16;
  static_assert(kBars % 8 == 0 && kSmem <= 232448, "shared memory");
  // TMEM columns
  static constexpr uint32_t kScores = 0;
  static constexpr uint32_t kIntra = 128;
  static constexpr uint32_t kInter = kIntra + DV;
  static constexpr uint32_t kDelta = kInter + DV;
  static constexpr uint32_t kTmemCols = 512;
};

template <typename T>
__device__ __forceinline__ uint32_t tc_idesc(int n, bool a_mn, bool b_mn) {
  constexpr uint32_t ab = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (ab << 7) | (ab << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         (uint32_t(n >> 3) << 17) | (uint32_t(kC >> 4) << 24);
}

// MN-major operand: 64-element blocks `block` bytes apart, K rows of 128 bytes.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr, uint32_t block) {
  uint64_t d = 0;
  d |= uint64_t((saddr >> 4) & 0x3fffu);
  d |= uint64_t(block >> 4) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}

// D += A B with A (16-bit, K-major) in tensor memory.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// One box (64 columns x 128 steps of one row and head) of a [d, t, h, b] map.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int d, int t, int h,
                                            int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(d), "r"(t), "r"(h), "r"(b), "r"(smem_addr(bar))
      : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  } else {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

// Byte offset of 16-byte piece `q` (8 columns) of row r in a 128-byte-swizzled
// tile of `rows` rows whose 64-column blocks follow one another.
__device__ __forceinline__ int piece_at(int r, int q, int rows) {
  return (q >> 3) * rows * 128 + r * 128 + (((q & 7) ^ (r & 7)) << 4);
}

// The power of two that brings `top` to [2^13, 2^14): fp16 operands keep their
// full precision and range whatever their magnitude. 1 for zero and non-finite.
__device__ __forceinline__ float fp16_scale(float top) {
  const int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xff);
  if (e == 0 || e == 0xff) return 1.0f;
  int s = 127 + 13 - (e - 127);  // biased exponent of the scale
  s = s < 67 ? 67 : (s > 187 ? 187 : s);  // 2^-60 .. 2^60
  return __uint_as_float(static_cast<uint32_t>(s) << 23);
}

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// A warp's threads have done their part: one arrival.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

template <typename T, int DK, int DV, bool STATES_ONLY>
__global__ void __launch_bounds__(kTcThreads, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap map_q,
                      const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ TcArgs args) {
  using L = TcLayout<DK, DV>;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* pow_t = reinterpret_cast<float*>(smem + L::kPow);
  float* weights = reinterpret_cast<float*>(smem + L::kWeights);
  float* row_scale = reinterpret_cast<float*>(smem + L::kRowScale);
  float* warp_max = reinterpret_cast<float*>(smem + L::kMax);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* full_q = bars;
  uint64_t* full_k = bars + 1;   // [2]
  uint64_t* full_v = bars + 3;   // [2]
  uint64_t* empty_q = bars + 5;
  uint64_t* empty_kv = bars + 6;  // [2]
  uint64_t* scores_done = bars + 8;
  uint64_t* p_ready = bars + 9;
  uint64_t* kw_ready = bars + 10;
  uint64_t* out_done = bars + 11;
  uint64_t* delta_done = bars + 12;
  uint64_t* carry_ready = bars + 13;
  uint64_t* drained = bars + 14;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kNumBars);

  const mb_decay_attention_args& a = args.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t u = blockIdx.x;
  const int h = static_cast<int>(u % a.H);
  u /= a.H;
  const int b = static_cast<int>(u % a.B);
  const int64_t seg = u / a.B;
  const int64_t len = attn_row_length(a.lengths, b, a.T);
  const int64_t lo = seg * args.split.len;
  const int64_t hi = imin64(a.T, lo + args.split.len);
  const int64_t end = imin64(hi, len);
  const int chunks = end > lo ? static_cast<int>((end - lo + kC - 1) / kC) : 0;
  const bool reverse = a.reverse != 0;
  const float log2g = log2f(a.decay[h]);

  auto chunk_t0 = [&](int i) {  // first step of the i-th chunk in processing order
    return lo + int64_t(reverse ? chunks - 1 - i : i) * kC;
  };
  auto chunk_steps = [&](int64_t t0) { return static_cast<int>(imin64(kC, end - t0)); };

  for (int i = threadIdx.x; i <= kC; i += kTcThreads) {
    pow_t[i] = decay_pow(log2g, i);
  }
  // weights[128 + r - j]: scale * g^|r - j| of the causal side, 0 of the other
  for (int i = threadIdx.x; i < 256; i += kTcThreads) {
    const int d = reverse ? 128 - i : i - 128;
    weights[i] = d >= 0 ? decay_pow(log2g, d) * (a.out_scale * a.kv_scale) : 0.0f;
  }
  if (threadIdx.x == 0) {
    mbar_init(full_q, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&full_k[s], 1);
      mbar_init(&full_v[s], 1);
      mbar_init(&empty_kv[s], 1);
    }
    mbar_init(empty_q, 1);
    mbar_init(scores_done, 1);
    mbar_init(p_ready, 4);
    mbar_init(kw_ready, 4);
    mbar_init(out_done, 2);  // the product's completion, and what its operand's makers wrote
    mbar_init(delta_done, 1);
    mbar_init(carry_ready, 4);
    mbar_init(drained, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(tmem_slot)),
                 "r"(L::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      const int qh = h * args.q_h, qb = b * args.q_b, kh = h * args.k_h, kb = b * args.k_b;
      const int vh = h * args.v_h, vb = b * args.v_b;
      int issued = 0;
      for (int i = 0; i < chunks; ++i) {
        const int s = i & 1;
        const int t = static_cast<int>(chunk_t0(i));
        if (i >= 2 && !mbar_wait_bounded(&empty_kv[s], ((i >> 1) - 1) & 1)) break;
        mbar_arrive_expect_tx(&full_k[s], L::kQBytes);
        for (int x = 0; x < DK / 64; ++x) {
          tma_load_4d(smem + L::kK + s * L::kQBytes + x * kBlockBytes, &map_k, x * 64, t, kh, kb,
                      &full_k[s]);
        }
        mbar_arrive_expect_tx(&full_v[s], L::kVBytes);
        for (int x = 0; x < DV / 64; ++x) {
          tma_load_4d(smem + L::kV + s * L::kVBytes + x * kBlockBytes, &map_v, x * 64, t, vh, vb,
                      &full_v[s]);
        }
        issued = i + 1;
        if constexpr (!STATES_ONLY) {
          if (i >= 1 && !mbar_wait_bounded(empty_q, (i - 1) & 1)) break;
          mbar_arrive_expect_tx(full_q, L::kQBytes);
          for (int x = 0; x < DK / 64; ++x) {
            tma_load_4d(smem + L::kQ + x * kBlockBytes, &map_q, x * 64, t, qh, qb, full_q);
          }
        }
      }
      // every issued copy has landed before the CTA can retire
      for (int i = issued > 2 ? issued - 2 : 0; i < issued; ++i) {
        (void)mbar_wait_bounded(&full_k[i & 1], (i >> 1) & 1);
        (void)mbar_wait_bounded(&full_v[i & 1], (i >> 1) & 1);
      }
      if (!STATES_ONLY && issued == chunks && chunks > 0) {
        (void)mbar_wait_bounded(full_q, (chunks - 1) & 1);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t i_scores = tc_idesc<T>(kC, false, false);
      const uint32_t i_out = tc_idesc<T>(DV, false, true);
      const uint32_t i_delta = tc_idesc<T>(DV, true, true);
      const uint32_t sq = smem_addr(smem + L::kQ), sk = smem_addr(smem + L::kK);
      const uint32_t slo = smem_addr(smem + L::kLo), sv = smem_addr(smem + L::kV);
      const uint32_t ss = smem_addr(smem + L::kS);
      auto scores = [&](int i) {
        if (!mbar_wait_bounded(full_q, i & 1) ||
            !mbar_wait_bounded(&full_k[i & 1], (i >> 1) & 1)) {
          return false;
        }
        tc_fence_after();
        const uint32_t k0 = sk + (i & 1) * L::kQBytes;
#pragma unroll
        for (int k = 0; k < DK / 16; ++k) {
          const uint32_t at = (k >> 2) * kBlockBytes + (k & 3) * 32;
          mma_f16(tmem + L::kScores, sw128_kmajor_desc(sq + at), sw128_kmajor_desc(k0 + at),
                  i_scores, k != 0);
        }
        mma_commit(scores_done);
        return true;
      };
      bool ok = true;
      if (!STATES_ONLY && chunks > 0) ok = scores(0);
      for (int i = 0; i < chunks && ok; ++i) {
        const int s = i & 1;
        const uint32_t v0 = sv + s * L::kVBytes;
        // the carry's operand is written, and what the accumulators held has been read
        if (!mbar_wait_bounded(carry_ready, i & 1)) break;
        tc_fence_after();
        if constexpr (!STATES_ONLY) {
#pragma unroll
          for (int k = 0; k < DK / 16; ++k) {
            mma_f16(tmem + L::kInter,
                    sw128_kmajor_desc(sq + (k >> 2) * kBlockBytes + (k & 3) * 32),
                    mn_desc(ss + k * 2048, DK * 128), i_out, k != 0);
          }
          mma_commit(empty_q);
          if (!mbar_wait_bounded(p_ready, i & 1)) break;
          if (!mbar_wait_bounded(&full_v[s], (i >> 1) & 1)) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kC / 16; ++k) {
            mma_f16_ts(tmem + L::kIntra, tmem + L::kScores + k * 8,
                       mn_desc(v0 + k * 2048, kBlockBytes), i_out, k != 0);
          }
          mma_commit(out_done);
          mbar_arrive(out_done);
          if (i + 1 < chunks) {
            // the next scores overwrite P: its product has to be complete
            if (!mbar_wait_bounded(out_done, i & 1)) break;
            if (!scores(i + 1)) break;
          }
        } else {
          if (!mbar_wait_bounded(&full_v[s], (i >> 1) & 1)) break;
        }
        if (!mbar_wait_bounded(kw_ready, i & 1)) break;
        tc_fence_after();
        const uint32_t k0 = sk + s * L::kQBytes;
#pragma unroll
        for (int k = 0; k < kC / 16; ++k) {
          mma_f16(tmem + L::kDelta, mn_desc(slo + k * 2048, kBlockBytes),
                  mn_desc(v0 + k * 2048, kBlockBytes), i_delta, k != 0);
        }
#pragma unroll
        for (int k = 0; k < kC / 16; ++k) {
          mma_f16(tmem + L::kDelta, mn_desc(k0 + k * 2048, kBlockBytes),
                  mn_desc(v0 + k * 2048, kBlockBytes), i_delta, 1u);
        }
        mma_commit(delta_done);
        mma_commit(&empty_kv[s]);
      }
      // all products and commits are complete before TMEM is released
      mma_commit(drained);
      (void)mbar_wait_bounded(drained, 0);
    }
  } else if (warp < 6) {
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t t_scores = tmem + L::kScores + (uint32_t(quarter * 32) << 16);
    const float* w_row = weights + 128 + r;  // w_row[-j]: weight of step j for this row
    for (int i = 0; i < chunks; ++i) {
      const int s = i & 1;
      const int n = chunk_steps(chunk_t0(i));
      uint8_t* ks = smem + L::kK + s * L::kQBytes;
      uint8_t* vs = smem + L::kV + s * L::kVBytes;
      if (!mbar_wait_bounded(&full_k[s], (i >> 1) & 1)) break;
      if (n < kC) {
        // values past the row's end may hold anything: 0 * NaN must not reach a sum
        if (!mbar_wait_bounded(&full_v[s], (i >> 1) & 1)) break;
        if (r >= n) {
#pragma unroll
          for (int q = 0; q < DV / 8; ++q) {
            *reinterpret_cast<uint4*>(vs + piece_at(r, q, kC)) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
      }
      if constexpr (!STATES_ONLY) {
        if (!mbar_wait_bounded(scores_done, i & 1)) break;
        tc_fence_after();
        // column blocks wholly on the other side of the diagonal are zero
        auto empty = [&](int jb) { return reverse ? jb < quarter : jb > quarter; };
        // in reverse, steps past the row's end lie on the causal side
        const int last = reverse ? n : kC;
        float scale = 1.0f;
        if constexpr (kHalf) {
          // fp16: P's rows are brought to a common magnitude by a power of two
          float top = 0.0f;
#pragma unroll
          for (int jb = 0; jb < 4; ++jb) {
            if (empty(jb)) continue;
            uint32_t x[32];
            tmem_ld32_issue(t_scores + jb * 32, x);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float w = fabsf(__uint_as_float(x[j]) * w_row[-(jb * 32 + j)]);
              top = fmaxf(top, jb * 32 + j < last ? w : 0.0f);  // drops a NaN
            }
          }
          scale = fp16_scale(top);
          row_scale[s * kC + r] = 1.0f / scale;
        }
#pragma unroll
        for (int jb = 0; jb < 4; ++jb) {
          uint32_t p[16];
          if (empty(jb)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) p[j] = 0;
          } else {
            uint32_t x[32];
            tmem_ld32_issue(t_scores + jb * 32, x);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              // a select: what a zero weight hides may be infinite or NaN
              const float w = jb * 32 + j < last ? w_row[-(jb * 32 + j)] : 0.0f;
              const float v = __uint_as_float(x[j]) * (kHalf ? w * scale : w);
              x[j] = __float_as_uint(w != 0.0f ? v : 0.0f);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              p[j] = pack2<T>(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]));
            }
          }
          // overwrites scores of blocks that this thread has read
          tmem_st16(t_scores + jb * 16, p);
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(p_ready, lane);
      }
      // the remainders' buffer is free once the last chunk's D is complete
      if (i >= 1 && !mbar_wait_bounded(delta_done, (i - 1) & 1)) break;
      const float w = r < n ? pow_t[reverse ? r + 1 : n - 1 - r] : 0.0f;
#pragma unroll
      for (int q = 0; q < DK / 8; ++q) {
        const int at = piece_at(r, q, kC);
        const uint4 x = *reinterpret_cast<const uint4*>(ks + at);
        const uint32_t in[4] = {x.x, x.y, x.z, x.w};
        uint32_t hi16[4], lo16[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack2<T>(in[e]);
          const float f0 = r < n ? f.x * w : 0.0f, f1 = r < n ? f.y * w : 0.0f;
          hi16[e] = pack2<T>(f0, f1);
          const float2 back = unpack2<T>(hi16[e]);
          lo16[e] = pack2<T>(f0 - back.x, f1 - back.y);
        }
        *reinterpret_cast<uint4*>(ks + at) = make_uint4(hi16[0], hi16[1], hi16[2], hi16[3]);
        *reinterpret_cast<uint4*>(smem + L::kLo + at) =
            make_uint4(lo16[0], lo16[1], lo16[2], lo16[3]);
      }
      fence_proxy_async_smem();
      warp_arrive(kw_ready, lane);
    }
  } else {
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row of the carry, and step of a chunk
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const bool row_ok = r < a.Dk;
    const bool holds = quarter * 32 < DK;  // warps past DK hold no carry (uniform)
    float S[DV];
    {
      const float* from = nullptr;
      int64_t sc = 1;
      if (!STATES_ONLY && row_ok) {
        if (args.split.segments > 1) {
          from = args.split.states + (((seg * a.B + b) * a.H + h) * a.Dk + r) * a.Dv;
        } else if (a.first.data != nullptr) {
          from = a.first.data + b * a.first.stride_b + h * a.first.stride_h +
                 r * a.first.stride_row;
          sc = a.first.stride_col;
        }
      }
#pragma unroll
      for (int c = 0; c < DV; ++c) S[c] = from != nullptr && c < a.Dv ? from[c * sc] : 0.0f;
    }
    float inv_s = 1.0f;  // fp16: 1 / scale of the carry's operand
    // the carry, rounded, as the B operand of the next chunk (rows of S, MN-major)
    auto put_carry = [&]() {
      float scale = 1.0f;
      if constexpr (kHalf) {
        float top = 0.0f;
        if (holds) {
#pragma unroll
          for (int c = 0; c < DV; ++c) top = fmaxf(top, fabsf(S[c]));
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        }
        bar_sync(1, 128);  // the last maxima have been read
        if (lane == 0) warp_max[quarter] = top;
        bar_sync(1, 128);
        top = fmaxf(fmaxf(warp_max[0], warp_max[1]), fmaxf(warp_max[2], warp_max[3]));
        scale = fp16_scale(top);
        inv_s = 1.0f / scale;
      }
      if (holds) {
#pragma unroll
        for (int q = 0; q < DV / 8; ++q) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = pack2<T>(S[8 * q + 2 * e] * scale, S[8 * q + 2 * e + 1] * scale);
          }
          *reinterpret_cast<uint4*>(smem + L::kS + piece_at(r, q, DK)) =
              make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
      fence_proxy_async_smem();
    };
    if (chunks > 0) {
      if constexpr (!STATES_ONLY) put_carry();
      warp_arrive(carry_ready, lane);
    }
    T* o = static_cast<T*>(a.o.data) + b * a.o.stride_b + h * a.o.stride_h;
    for (int i = 0; i < chunks; ++i) {
      const int64_t t0 = chunk_t0(i);
      const int n = chunk_steps(t0);
      if constexpr (!STATES_ONLY) {
        if (!mbar_wait_bounded(out_done, i & 1)) break;
        tc_fence_after();
        const float w_in = kHalf ? row_scale[(i & 1) * kC + r] : 1.0f;
        const float w_out =
            r < n ? pow_t[reverse ? n - 1 - r : r + 1] * a.out_scale * inv_s : 0.0f;
        const bool store = t0 + r < hi;  // steps past the row's length get zeros
        T* row = o + (t0 + r) * a.o.stride_t;
#pragma unroll
        for (int c0 = 0; c0 < DV; c0 += 16) {
          uint32_t x[16], y[16];
          tmem_ld16_issue(tmem + L::kIntra + lanes + c0, x);
          tmem_ld16_issue(tmem + L::kInter + lanes + c0, y);
          tmem_wait_ld();
          uint32_t p[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float in = __uint_as_float(x[2 * j + e]), out = __uint_as_float(y[2 * j + e]);
              v[e] = fmaf(out, w_out, kHalf ? in * w_in : in);
            }
            p[j] = r < n ? pack2<T>(v[0], v[1]) : 0u;
          }
          if (store && c0 < a.Dv) {
            *reinterpret_cast<uint4*>(row + c0) = make_uint4(p[0], p[1], p[2], p[3]);
            if (c0 + 8 < a.Dv) {
              *reinterpret_cast<uint4*>(row + c0 + 8) = make_uint4(p[4], p[5], p[6], p[7]);
            }
          }
        }
      }
      if (!mbar_wait_bounded(delta_done, i & 1)) break;
      tc_fence_after();
      if (holds) {
        const float gn = pow_t[n];
#pragma unroll
        for (int c0 = 0; c0 < DV; c0 += 32) {
          uint32_t x[32];
          tmem_ld32_issue(tmem + L::kDelta + lanes + c0, x);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            S[c0 + j] = fmaf(gn, S[c0 + j], a.kv_scale * __uint_as_float(x[j]));
          }
        }
      }
      if (i + 1 < chunks) {
        if constexpr (!STATES_ONLY) put_carry();
        tc_fence_before();
        warp_arrive(carry_ready, lane);
      }
    }
    if (!STATES_ONLY) {  // whole chunks past the row's length: zeros
      for (int64_t t = lo + int64_t(chunks) * kC + r; t < hi; t += kC) {
        T* row = o + t * a.o.stride_t;
        for (int c = 0; c < a.Dv; c += 8) {
          *reinterpret_cast<uint4*>(row + c) = make_uint4(0, 0, 0, 0);
        }
      }
    }
    if (row_ok) {
      float* to = nullptr;
      int64_t sc = 1;
      if (STATES_ONLY) {
        to = args.split.states + (((seg * a.B + b) * a.H + h) * a.Dk + r) * a.Dv;
      } else if (args.split.segments == 1 && a.last.data != nullptr) {
        to = a.last.data + b * a.last.stride_b + h * a.last.stride_h + r * a.last.stride_row;
        sc = a.last.stride_col;
      }
      if (to != nullptr) {
#pragma unroll
        for (int c = 0; c < DV; ++c) {
          if (c < a.Dv) to[c * sc] = S[c];
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(L::kTmemCols));
  }
}

// A [d, t, h, b] map of 64 x 128 boxes; a dimension of stride 0 or size 1 has
// extent 1 and its coordinate multiplied by 0.
bool make_attn_map(CUtensorMap* map, const mb_steps& x, int64_t T, int64_t H, int64_t B, int64_t D,
                   bool bf16, int32_t* h_on, int32_t* b_on) {
  auto fn = tma_encode_fn();
  if (fn == nullptr) return false;
  *h_on = H > 1 && x.stride_h != 0;
  *b_on = B > 1 && x.stride_b != 0;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(T),
                        static_cast<cuuint64_t>(*h_on ? H : 1),
                        static_cast<cuuint64_t>(*b_on ? B : 1)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(T > 1 ? x.stride_t * 2 : 16),
                           static_cast<cuuint64_t>(*h_on ? x.stride_h * 2 : 16),
                           static_cast<cuuint64_t>(*b_on ? x.stride_b * 2 : 16)};
  cuuint32_t box[4] = {64, kC, 1, 1};
  cuuint32_t estride[4] = {1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            x.data, dims, strides, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DK, int DV, bool STATES_ONLY>
int launch_chunks(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                  const TcArgs& args, cudaStream_t s) {
  auto kern = attn_chunk_kernel<T, DK, DV, STATES_ONLY>;
  constexpr size_t smem = TcLayout<DK, DV>::kSmem;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  const int64_t blocks = args.split.segments * args.a.B * args.a.H;
  MB_CHECK_ARG(blocks <= 0x7fffffff, "mb_decay_attention: too many (batch, head) rows");
  kern<<<static_cast<unsigned>(blocks), kTcThreads, smem, s>>>(mq, mk, mv, args);
  MB_CHECK_LAUNCH("mb_decay_attention (chunks)");
  return 0;
}

template <typename T, int DK, int DV>
int launch_mode(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                const TcArgs& args, bool states_only, cudaStream_t s) {
  return states_only ? launch_chunks<T, DK, DV, true>(mq, mk, mv, args, s)
                     : launch_chunks<T, DK, DV, false>(mq, mk, mv, args, s);
}

template <typename T>
int launch_type(const mb_decay_attention_args& a, const AttnSplit& split, bool states_only,
                cudaStream_t s) {
  TcArgs args;
  args.a = a;
  args.split = split;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap mq, mk, mv;
  MB_CHECK_ARG(make_attn_map(&mq, a.q, a.T, a.H, a.B, a.Dk, bf16, &args.q_h, &args.q_b) &&
                   make_attn_map(&mk, a.k, a.T, a.H, a.B, a.Dk, bf16, &args.k_h, &args.k_b) &&
                   make_attn_map(&mv, a.v, a.T, a.H, a.B, a.Dv, bf16, &args.v_h, &args.v_b),
               "mb_decay_attention: cuTensorMapEncodeTiled failed (shape or alignment)");
  const bool k64 = a.Dk <= 64, v64 = a.Dv <= 64;
  if (k64 && v64) return launch_mode<T, 64, 64>(mq, mk, mv, args, states_only, s);
  if (k64) return launch_mode<T, 64, 128>(mq, mk, mv, args, states_only, s);
  if (v64) return launch_mode<T, 128, 64>(mq, mk, mv, args, states_only, s);
  return launch_mode<T, 128, 128>(mq, mk, mv, args, states_only, s);
}

// Rows that the tensor-map copies and 16-byte stores take: 16-byte base and strides.
bool steps_ok(const mb_steps& x, int64_t T, bool broadcast_ok) {
  const int64_t limit = int64_t(1) << 38;  // strides below 2^40 bytes
  return aligned_to(x.data, 16) && x.stride_t % 8 == 0 && x.stride_h % 8 == 0 &&
         x.stride_b % 8 == 0 && x.stride_t >= 0 && x.stride_h >= 0 && x.stride_b >= 0 &&
         x.stride_t < limit && x.stride_h < limit && x.stride_b < limit &&
         (T <= 1 || x.stride_t > 0) && broadcast_ok;
}

}  // namespace

bool attn_tc_supported(const mb_decay_attention_args& a) {
  if (a.dtype == MB_F32 || a.Dk > 128 || a.Dv > 128 || a.T < kTcMinSteps) return false;
  return a.Dv % 8 == 0 && steps_ok(a.q, a.T, true) && steps_ok(a.k, a.T, true) &&
         steps_ok(a.v, a.T, true) && steps_ok(a.o, a.T, true);
}

// Segments of the time axis, in whole chunks: the count whose waves of CTAs (one
// per SM) take the fewest chunk times, where a split costs a second pass over k
// and v (about six tenths of a chunk) and, per segment, a read and a write of its
// memory (about one chunk each).
AttnSplit attn_tc_split(const mb_decay_attention_args& a) {
  const int64_t chunks = ceil_div(a.T, kC), rows = a.B * a.H;
  int64_t best = 1;
  double best_cost = 0;
  for (int64_t want = 1; want <= chunks && want <= 64; ++want) {
    const int64_t per = ceil_div(chunks, want), segments = ceil_div(chunks, per);
    if (segments != want) continue;
    const double waves = static_cast<double>(ceil_div(rows * segments, 148));
    const double cost = waves * (segments == 1 ? per + 1.0 : 1.6 * per + 4.0) +
                        (segments == 1 ? 0.0 : 3.0);
    if (want == 1 || cost < best_cost) {
      best = want;
      best_cost = cost;
    }
  }
  const int64_t per = ceil_div(chunks, best);
  return AttnSplit{static_cast<int>(best), best > 1 ? per * kC : a.T, nullptr};
}

int attn_tc_launch(const mb_decay_attention_args& a, const AttnSplit& split, bool states_only,
                   cudaStream_t stream) {
  return a.dtype == MB_BF16 ? launch_type<__nv_bfloat16>(a, split, states_only, stream)
                            : launch_type<__half>(a, split, states_only, stream);
}

int attention_unit_status(bool clear) { return read_device_status(clear); }

cudaError_t attention_unit_wait_probe(uint32_t polls, cudaStream_t stream) {
  wait_timeout_probe_kernel<<<1, 32, 0, stream>>>(polls);
  return cudaGetLastError();
}

}  // namespace mb
