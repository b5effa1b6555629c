// Attention with a decay for each head in chunks of 128 steps on the tensor
// cores (formulas: decay_attention.cuh). Two kernels, both one persistent CTA per
// SM that walks whole (segment, batch row, head) units chunk by chunk; with S the
// carry, g^|r-j| and the weights W of a chunk's rows:
//
//   outputs  P = (Q K^T) * g^|r-j| on the causal side    O = P V + W_out (Q S)
//            D = (W_kv K)^T V                             S <- g^n S + c D
//   states   D and S only
//
// W_kv K goes as 16-bit parts whose sum keeps its bits: in the states kernel two of fp16
// (brought to a common magnitude by a power of two first, which leaves 2^-22) or three of
// bf16, so that the memories that leave the operator are good to fp32; in the outputs
// kernel two of either, since the carry there is rounded to 16 bits before use. That
// rounding and the one of P, one 16-bit part each, are the outputs' own error: 0.0023
// relative in bf16, 0.0017 for a result rounded once. Second parts would take 16 more
// products per chunk of 128-wide heads and a second tile in full shared memory.
//
// All products are tcgen05 (M = 128 steps or memory rows, sums in TMEM). 20 warps:
//   warp 0      copies: Q, K, V, two stages of 128-byte-swizzled tiles
//   warp 1      issues the products, one thread: the next chunk's Q K^T, then this one's
//               Q S, (W_kv K)^T V and P V
//   warps 4-11  scores -> P (16 bits, back into TMEM as an A operand) and K -> W_kv K
//               in place; two warps per 32 rows, half of the columns each
//   warps 12-19 outputs; the carry in fp32 registers (row per lane, half of the
//               columns), rounded into shared memory as the next chunk's operand
// Registers move from the first three warpgroups to the last two (setmaxnreg).
//
// Floor: the bytes of q, k, v and o (one read, one write); a chunk of 128-wide heads is
// 128 KB, 5.6 thousand cycles of one SM's share of the copy bandwidth. Measured (bf16,
// 134 M elements each of q, k, v, o): outputs 0.235 ms at T = 256 and 0.285 ms at
// T = 4096, against 0.164 ms at the copy bandwidth. What holds it there is the chain of
// one chunk's hand-overs (Q S -> D -> carry -> P V -> outputs read -> next Q S, about 7
// thousand cycles), not a unit: of the cycles, the tensor pipe is active in 18 %, the
// issue slots in 26 %, DRAM in 36 %. 65 cycles per 128 x 128 x 16 product, 32 (40) of them per
// chunk, would take 2.1 (2.6) thousand. Memories: 0.15 ms for 134 M elements each of k
// and v (0.082 at the copy bandwidth, plus the memories' own bytes).
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
constexpr int kTcThreads = 640;
constexpr int kBlockBytes = kC * 128;  // 64 columns x 128 steps of 16 bits
constexpr int64_t kTcMinSteps = 16;    // below: the recurrent kernel
constexpr int kGroup = 256;            // threads of each of the two worker groups
// Batch rows that are put in order of their lengths (T = 1000, 4 heads of 64: 128 rows
// 0.108 ms, 129 rows in batch order 0.123 ms).
constexpr int kMaxOrder = 128;

struct TcArgs {
  mb_decay_attention_args a;
  AttnSplit split;
  int64_t units;  // segments x B x H
  // whether a dimension's coordinate counts (0: the tensor is broadcast along it)
  int32_t q_b, q_h, k_b, k_h, v_b, v_h, o_b, o_h;
  int32_t m_map;  // states: memories leave by tensor stores
};

template <int DK, int DV>
struct OutLayout {
  // 128-wide heads fill shared memory: one V stage instead of two, and outputs are
  // staged where their chunk's Q was
  static constexpr bool kFull = DK == 128 && DV == 128;
  static constexpr int kVStages = kFull ? 1 : 2;
  static constexpr int kQBytes = kC * DK * 2;
  static constexpr int kVBytes = kC * DV * 2;
  static constexpr int kQ = 0;  // two stages each of Q and K
  static constexpr int kK = kQ + 2 * kQBytes;
  static constexpr int kLo = kK + 2 * kQBytes;  // what rounding leaves of W_kv K
  static constexpr int kV = kLo + kQBytes;
  static constexpr int kS = kV + kVStages * kVBytes;
  static constexpr int kO = kFull ? kQ : kS + DK * DV * 2;
  static constexpr int kRowScale = kS + DK * DV * 2 + (kFull ? 0 : kVBytes);  // fp16: 1 / scale of
                                                          // P's rows, by stage
  static constexpr int kRowTop = kRowScale + 2 * kC * 4;  // fp16: largest of the other half
  static constexpr int kMax = kRowTop + kC * 4;           // fp16: largest values of each warp
  static constexpr int kKeyTop = kMax + 2 * 8 * 4;        // fp16: largest weighed key of each warp
  static constexpr int kKeyInv = kKeyTop + 2 * 8 * 4;     // fp16: 1 / scale of the weighed keys
  static constexpr int kBars = kKeyInv + 2 * 4;
  static constexpr int kNumBars = 20;
  static constexpr int kOrder = kBars + kNumBars * 8 + 16;  // batch rows, longest first
  static constexpr size_t kSmem = kOrder + kMaxOrder * 2;
  static_assert(kBars % 8 == 0 && kSmem <= 232448, "shared memory");
  // TMEM columns: two buffers of scores (P takes the first half of its own), P V, Q S;
  // D uses P V's columns, which the carry warps have left by the time P is ready
  static constexpr uint32_t kScores = 0;
  static constexpr uint32_t kIntra = 256;
  static constexpr uint32_t kDelta = kIntra;
  static constexpr uint32_t kInter = kIntra + DV;
};

template <int DK, int DV, int PARTS>
struct StatesLayout {
  static constexpr int kKBytes = kC * DK * 2;
  static constexpr int kVBytes = kC * DV * 2;
  static constexpr int kK = 0;  // two stages each
  static constexpr int kLo = kK + 2 * kKBytes;  // the further parts of W_kv K
  static constexpr int kV = kLo + (PARTS - 1) * kKBytes;
  static constexpr int kOut = kV + 2 * kVBytes;  // 32 x 32 fp32 per carry warp, on the way out
  static constexpr int kKeyTop = kOut + 8 * 4096;      // fp16: largest weighed key of each warp
  static constexpr int kKeyInv = kKeyTop + 2 * 8 * 4;  // fp16: 1 / scale of the weighed keys
  static constexpr int kBars = kKeyInv + 2 * 4;
  static constexpr int kNumBars = 12;
  static constexpr int kOrder = kBars + kNumBars * 8 + 16;  // batch rows, longest first
  static constexpr size_t kSmem = kOrder + kMaxOrder * 2;
  static_assert(kBars % 8 == 0 && kSmem <= 232448, "shared memory");
  static constexpr uint32_t kDelta = 0;
};

// One (segment, batch row, head): its valid steps [lo, end) and their chunks.
struct Unit {
  int b, h;
  int64_t seg, lo, hi, end;
  int chunks;  // -1: no unit
  float g, log2g;
};

// Ragged rows: a CTA's units should add up to the same steps as its neighbours'. The
// batch rows are ranked by length, longest first, and dealt in turns that go up and
// down the CTAs, so that the CTA with a turn's longest unit gets the next one's
// shortest (T = 1000, 288 units of 0 to 1000 steps: 0.099 -> 0.092 ms). Every CTA ranks
// them for itself, ahead of a __syncthreads. Kernels of their own (RANKED), since the
// bookkeeping costs the others 3 to 5 %.
__device__ __forceinline__ void rank_rows(const TcArgs& args, uint16_t* order) {
  const mb_decay_attention_args& a = args.a;
  const int b = threadIdx.x;
  if (b < a.B) {
    const int64_t mine = attn_row_length(a.lengths, b, a.T);
    int rank = 0;
    for (int i = 0; i < a.B; ++i) {
      const int64_t other = attn_row_length(a.lengths, i, a.T);
      rank += other > mine || (other == mine && i < b);
    }
    order[rank] = static_cast<uint16_t>(b);
  }
}

// Turns of all CTAs, as units: whole rounds where the order of a turn may be reversed.
__device__ __forceinline__ uint32_t unit_visits(const TcArgs& args, const uint16_t* order) {
  const uint32_t g = gridDim.x, units = static_cast<uint32_t>(args.units);
  return order == nullptr ? units : (units + g - 1) / g * g;
}

__device__ __forceinline__ Unit decode_unit(const TcArgs& args, uint32_t unit,
                                            const uint16_t* order) {
  const mb_decay_attention_args& a = args.a;
  const uint32_t H = static_cast<uint32_t>(a.H), B = static_cast<uint32_t>(a.B);
  Unit u;
  if (order != nullptr) {
    const uint32_t g = gridDim.x, turn = unit / g;
    if (turn & 1) unit = turn * g + (g - 1 - unit % g);
    if (unit >= static_cast<uint32_t>(args.units)) {  // no unit in this turn
      return Unit{0, 0, 0, 0, 0, 0, -1, 0.0f, 0.0f};
    }
  }
  const uint32_t row = unit / H;
  u.h = static_cast<int>(unit % H);
  u.b = static_cast<int>(row % B);
  u.seg = row / B;
  if (order != nullptr) u.b = order[u.b];
  u.lo = u.seg * args.split.len;
  u.hi = imin64(a.T, u.lo + args.split.len);
  u.end = imin64(u.hi, attn_row_length(a.lengths, u.b, a.T));
  u.chunks = u.end > u.lo ? static_cast<int>((u.end - u.lo + kC - 1) / kC) : 0;
  u.g = a.decay[u.h];
  u.log2g = log2f(u.g);
  return u;
}

// First step of the unit's i-th chunk in processing order, and its valid steps.
__device__ __forceinline__ int64_t chunk_t0(const Unit& u, int i, bool reverse) {
  return u.lo + int64_t(reverse ? u.chunks - 1 - i : i) * kC;
}
__device__ __forceinline__ int chunk_steps(const Unit& u, int64_t t0) {
  return static_cast<int>(imin64(kC, u.end - t0));
}

// Weight of row r (< n) of a chunk of n steps in the carry that leaves it, and of
// the carry that enters it in row r's output.
__device__ __forceinline__ float kv_weight(const Unit& u, int r, int n, bool reverse) {
  return decay_pow(u.log2g, reverse ? r + 1 : n - 1 - r);
}
__device__ __forceinline__ float out_weight(const Unit& u, int r, int n, bool reverse) {
  return decay_pow(u.log2g, reverse ? n - 1 - r : r + 1);
}

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

__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int d, int t,
                                             int h, int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(d), "r"(t), "r"(h), "r"(b), "r"(smem_addr(src))
      : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
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

// Two fp32 products or sums in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
        "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}

// One lane of a converged warp, the same each time; the compiler knows that the
// code under it runs in one thread (products issue from uniform registers).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// Whether phase `parity` of a barrier is complete, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Byte offset of 16-byte piece `q` (8 columns) of row r in a 128-byte-swizzled
// tile of `rows` rows whose 64-column blocks follow one another.
__device__ __forceinline__ int piece_at(int r, int q, int rows) {
  return (q >> 3) * rows * 128 + r * 128 + (((q & 7) ^ (r & 7)) << 4);
}

// The power of two that brings `top` to [2^13, 2^14): fp16 operands keep their
// full precision and range whatever their magnitude (fp32's own range: the scale and its
// inverse are normal numbers). 1 for zero and non-finite.
__device__ __forceinline__ float fp16_scale(float top) {
  const int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xff);
  if (e == 0 || e == 0xff) return 1.0f;
  int s = 127 + 13 - (e - 127);  // biased exponent of the scale
  s = s < 14 ? 14 : (s > 240 ? 240 : s);  // 2^-113 .. 2^113
  return __uint_as_float(static_cast<uint32_t>(s) << 23);
}

// Named barriers: 2 the carry warps, 3..6 the two score warps and 7..10 the two
// output warps of one TMEM lane quarter, 11 the warps that weigh the keys.
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// A warp's threads have done their part: one arrival.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}


// This thread's half of row r of a K tile times w (zero past the chunk's n steps), as
// PARTS 16-bit parts that add up to it: the first in place, the others to `lo`.
template <typename T, int DK, int PARTS>
__device__ __forceinline__ void weigh_k_row(uint8_t* ks, uint8_t* lo, int r, int half, float w,
                                            bool valid) {
  const float2 w2 = make_float2(w, w), minus = make_float2(-1.0f, -1.0f);
#pragma unroll
  for (int q = 0; q < DK / 16; ++q) {
    const int at = piece_at(r, half * (DK / 16) + q, kC);
    const uint4 x = *reinterpret_cast<const uint4*>(ks + at);
    const uint32_t in[4] = {x.x, x.y, x.z, x.w};
    float2 f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = mul2(unpack2<T>(valid ? in[e] : 0u), w2);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      uint32_t y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = pack2<T>(f[e].x, f[e].y);
        if (part + 1 < PARTS) f[e] = fma2(unpack2<T>(y[e]), minus, f[e]);
      }
      uint8_t* to = part == 0 ? ks : lo + (part - 1) * kC * DK * 2;
      *reinterpret_cast<uint4*>(to + at) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

// fp16: the power of two that brings a chunk's largest weighed key to [2^13, 2^14), so
// that two parts leave 2^-22 of a key whatever the keys' magnitude (rounded where they
// are, keys of 1e-5 lost 0.5 %, since the second part adds nothing below 2^-24). One for
// the whole chunk, whose products are one sum. `tops` has 8 values for each of two chunks:
// who writes a chunk's has passed the barrier of the one between.
template <int DK>
__device__ __forceinline__ float key_scale(const uint8_t* ks, float* tops, int r, int half,
                                           float w, bool valid) {
  __half2 top2 = __float2half2_rn(0.0f);
#pragma unroll
  for (int q = 0; q < DK / 16; ++q) {
    const uint4 x = *reinterpret_cast<const uint4*>(ks + piece_at(r, half * (DK / 16) + q, kC));
    const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      top2 = __hmax2(top2, __habs2(*reinterpret_cast<const __half2*>(&in[e])));
    }
  }
  const float mine = valid ? w * __half2float(__hmax(__low2half(top2), __high2half(top2))) : 0.0f;
  const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(mine));
  if ((threadIdx.x & 31) == 0) tops[(threadIdx.x >> 5) - 4] = __uint_as_float(top);
  bar_sync(11, kGroup);
  float all = tops[0];
#pragma unroll
  for (int x = 1; x < 8; ++x) all = fmaxf(all, tops[x]);
  return fp16_scale(all);
}

template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ uint32_t tmem_alloc(uint32_t* slot, int warp) {
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return *slot;
}

__device__ __forceinline__ void tmem_free(uint32_t tmem, int warp) {
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// COLS values of one memory row (element c at p[c * stride], c < valid), zeros
// where p is null or past `valid`.
template <int COLS>
__device__ __forceinline__ void load_memory_row(const float* p, int64_t stride, int64_t valid,
                                                float (&S)[COLS]) {
  if (p == nullptr || valid <= 0) {
#pragma unroll
    for (int c = 0; c < COLS; ++c) S[c] = 0.0f;
  } else if (stride == 1 && valid >= COLS && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int c = 0; c < COLS; c += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + c);
      S[c] = x.x;
      S[c + 1] = x.y;
      S[c + 2] = x.z;
      S[c + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int c = 0; c < COLS; ++c) S[c] = c < valid ? p[c * stride] : 0.0f;
  }
}

template <int COLS>
__device__ __forceinline__ void store_memory_row(float* p, int64_t stride, int64_t valid,
                                                 const float (&S)[COLS]) {
  if (p == nullptr) return;
  if (stride == 1 && valid >= COLS && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int c = 0; c < COLS; c += 4) {
      *reinterpret_cast<float4*>(p + c) = make_float4(S[c], S[c + 1], S[c + 2], S[c + 3]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      if (c < valid) p[c * stride] = S[c];
    }
  }
}

// Sixteen scores of one row times c g^distance, zero on the other side of the
// diagonal: column j of the group lies at distance e0 - j (REVERSE: j - e0) from the
// row; in reverse, columns from `valid` on lie past the row's end. The weight runs
// along the columns, one product each. Selects, not products with zero: what lies
// outside may be infinite or NaN. (A second copy without the selects, for groups
// wholly inside, saved instructions but missed the instruction cache: 3 to 7 % slower.)
template <bool REVERSE>
__device__ __forceinline__ void weigh16(const uint32_t* v, int e0, int valid, float c,
                                        const Unit& u, float (&f)[16]) {
  const int d = REVERSE ? -1 - e0 : e0 - 16;  // distance one step before the first column
  float w = d >= 0 ? c * decay_pow(u.log2g, d) : 0.0f;
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const int j = REVERSE ? x : 15 - x;
    w = j == e0 ? c : w * u.g;
    const bool in = REVERSE ? j >= e0 && j < valid : j <= e0;
    f[j] = in ? __uint_as_float(v[j]) * w : 0.0f;
  }
}

// Values past the row's end may hold anything (0 * NaN must not reach a sum):
// this thread's half of row r of a V tile becomes zero.
template <int DV>
__device__ __forceinline__ void zero_v_row(uint8_t* vs, int r, int half) {
#pragma unroll
  for (int q = 0; q < DV / 16; ++q) {
    *reinterpret_cast<uint4*>(vs + piece_at(r, half * (DV / 16) + q, kC)) = make_uint4(0, 0, 0, 0);
  }
}

// ---------------------------------------------------------------------------
// Outputs
// ---------------------------------------------------------------------------
template <typename T, int DK, int DV, bool REVERSE, bool RANKED>
__global__ void __launch_bounds__(kTcThreads, 1)
    attn_out_kernel(const __grid_constant__ CUtensorMap map_q,
                    const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ CUtensorMap map_o,
                    const __grid_constant__ TcArgs args) {
  using L = OutLayout<DK, DV>;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr int kCols = DV / 2;  // memory and output columns per worker thread
  extern __shared__ __align__(1024) uint8_t smem[];
  float* row_scale = reinterpret_cast<float*>(smem + L::kRowScale);
  float* row_top = reinterpret_cast<float*>(smem + L::kRowTop);
  float* warp_max = reinterpret_cast<float*>(smem + L::kMax);
  float* key_top = reinterpret_cast<float*>(smem + L::kKeyTop);
  float* key_inv = reinterpret_cast<float*>(smem + L::kKeyInv);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* full_q = bars;            // [2]
  uint64_t* full_k = bars + 2;        // [2]
  uint64_t* full_v = bars + 4;        // [2]
  uint64_t* empty_q = bars + 6;       // [2] scores and Q S read it, outputs left it
  uint64_t* empty_kv = bars + 8;      // [2] a chunk's K and V
  uint64_t* scores_done = bars + 10;  // [2]
  uint64_t* p_ready = bars + 12;      // [2] the score warps may be a chunk ahead
  uint64_t* out_done = bars + 14;
  uint64_t* out_read = bars + 15;
  uint64_t* kw_ready = bars + 16;
  uint64_t* delta_done = bars + 17;
  uint64_t* carry_ready = bars + 18;
  uint64_t* drained = bars + 19;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kNumBars);

  const mb_decay_attention_args& a = args.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr bool reverse = REVERSE;
  constexpr int VS = L::kVStages;
  // whether units start from a memory; without one their first chunk has no Q S
  const bool carry_in = args.split.segments > 1 || a.first.data != nullptr;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&full_q[s], 1);
      mbar_init(&full_k[s], 1);
      mbar_init(&full_v[s], 1);
      mbar_init(&empty_q[s], 8);
      mbar_init(&empty_kv[s], 1);
      mbar_init(&scores_done[s], 1);
      mbar_init(&p_ready[s], 8);
    }
    mbar_init(out_done, 2);  // the products' completion, and what their operands' makers wrote
    mbar_init(out_read, 8);
    mbar_init(kw_ready, 8);
    mbar_init(delta_done, kHalf ? 2 : 1);  // fp16: with the scale that the keys' weighers wrote
    mbar_init(carry_ready, 8);
    mbar_init(drained, 1);
    fence_barrier_init();
  }
  uint16_t* order = RANKED ? reinterpret_cast<uint16_t*>(smem + L::kOrder) : nullptr;
  if constexpr (RANKED) rank_rows(args, order);
  const uint32_t tmem = tmem_alloc(tmem_slot, warp);
  const uint32_t visits = unit_visits(args, order);

  // Parities: `it` counts chunks over all of the CTA's units (stage it & 1), `hand`
  // the chunks whose carry goes on (all but each unit's last), `cin` the chunks
  // that a carry enters. All roles count alike.
  if (warp < 4) {
    reg_dec<56>();
    if (warp == 0 && elect_one()) {
      uint32_t it = 0, nq = 0, nk = 0, nv = 0;  // loads issued
      bool ok = true;
      for (uint32_t unit = blockIdx.x; unit < visits && ok; unit += gridDim.x) {
        const Unit u = decode_unit(args, unit, order);
        const int qh = u.h * args.q_h, qb = u.b * args.q_b, kh = u.h * args.k_h;
        const int kb = u.b * args.k_b, vh = u.h * args.v_h, vb = u.b * args.v_b;
        for (int i = 0; i < u.chunks; ++i, ++it) {
          const int s = it & 1;
          const int t = static_cast<int>(chunk_t0(u, i, reverse));
          ok = false;
          if (it >= 2 && !mbar_wait_bounded(&empty_kv[s], ((it >> 1) - 1) & 1)) break;
          mbar_arrive_expect_tx(&full_k[s], L::kQBytes);
#pragma unroll
          for (int x = 0; x < DK / 64; ++x) {
            tma_load_4d(smem + L::kK + s * L::kQBytes + x * kBlockBytes, &map_k, x * 64, t, kh, kb,
                        &full_k[s]);
          }
          nk = it + 1;
          if (it >= 2 && !mbar_wait_bounded(&empty_q[s], ((it >> 1) - 1) & 1)) break;
          mbar_arrive_expect_tx(&full_q[s], L::kQBytes);
#pragma unroll
          for (int x = 0; x < DK / 64; ++x) {
            tma_load_4d(smem + L::kQ + s * L::kQBytes + x * kBlockBytes, &map_q, x * 64, t, qh, qb,
                        &full_q[s]);
          }
          nq = it + 1;
          if (VS == 1 && it >= 1 && !mbar_wait_bounded(&empty_kv[s ^ 1], ((it - 1) >> 1) & 1)) break;
          mbar_arrive_expect_tx(&full_v[it % VS], L::kVBytes);
#pragma unroll
          for (int x = 0; x < DV / 64; ++x) {
            tma_load_4d(smem + L::kV + (it % VS) * L::kVBytes + x * kBlockBytes, &map_v, x * 64, t,
                        vh, vb, &full_v[it % VS]);
          }
          nv = it + 1;
          ok = true;
        }
      }
      // every issued copy has landed before the CTA can retire
      for (uint32_t j = nq > 2 ? nq - 2 : 0; j < nq; ++j) {
        (void)mbar_wait_bounded(&full_q[j & 1], (j >> 1) & 1);
      }
      for (uint32_t j = nk > 2 ? nk - 2 : 0; j < nk; ++j) {
        (void)mbar_wait_bounded(&full_k[j & 1], (j >> 1) & 1);
      }
      for (uint32_t j = nv > VS ? nv - VS : 0; j < nv; ++j) {
        (void)mbar_wait_bounded(&full_v[j % VS], (j / VS) & 1);
      }
    } else if (warp == 1 && elect_one()) {
      const uint32_t i_scores = tc_idesc<T>(kC, false, false);
      const uint32_t i_out = tc_idesc<T>(DV, false, true);
      const uint32_t i_delta = tc_idesc<T>(DV, true, true);
      // descriptors of the tiles' starts: a step along a tile adds its bytes / 16
      const uint64_t dq = sw128_kmajor_desc(smem_addr(smem + L::kQ));
      const uint64_t dk = sw128_kmajor_desc(smem_addr(smem + L::kK));
      const uint64_t dkt = mn_desc(smem_addr(smem + L::kK), kBlockBytes);
      const uint64_t dlo = mn_desc(smem_addr(smem + L::kLo), kBlockBytes);
      const uint64_t dv = mn_desc(smem_addr(smem + L::kV), kBlockBytes);
      const uint64_t ds = mn_desc(smem_addr(smem + L::kS), DK * 128);
      uint32_t it = 0, hand = 0, cin = 0;
      bool ok = true;
      // the scores of chunk j, if its Q and K are there (or after waiting for them);
      // what their buffer held has been read by then
      uint32_t scored = 0;
      auto scores = [&](uint32_t j, bool wait) {
        const int s = j & 1;
        if (!wait && !(mbar_test(&full_q[s], (j >> 1) & 1) && mbar_test(&full_k[s], (j >> 1) & 1))) {
          return true;
        }
        if (!mbar_wait_bounded(&full_q[s], (j >> 1) & 1) ||
            !mbar_wait_bounded(&full_k[s], (j >> 1) & 1)) {
          return false;
        }
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < DK / 16; ++k) {
          const uint32_t at = (s * L::kQBytes + (k >> 2) * kBlockBytes + (k & 3) * 32) >> 4;
          mma_f16(tmem + L::kScores + s * 128, dq + at, dk + at, i_scores, k != 0);
        }
        mma_commit(&scores_done[s]);
        ++scored;
        return true;
      };
      // the next chunk's scores are issued a chunk ahead, across units
      uint32_t unit = blockIdx.x;
      auto next_unit = [&](uint32_t from) {
        uint32_t x = from;
        while (x < visits && decode_unit(args, x, order).chunks <= 0) x += gridDim.x;
        return x;
      };
      unit = next_unit(unit);
      if (unit < visits) ok = scores(0, true);
      while (unit < visits && ok) {
        const Unit u = decode_unit(args, unit, order);
        const uint32_t following = next_unit(unit + gridDim.x);
        for (int i = 0; i < u.chunks; ++i, ++it) {
          const int s = it & 1;
          const uint64_t v0 = dv + (((it % VS) * L::kVBytes) >> 4);
          const bool last = i + 1 == u.chunks;
          ok = false;
          const bool more = !last || following < visits;
          // what the last chunk left in the accumulators and in P has been read
          if (it >= 1 && !mbar_wait_bounded(out_read, (it - 1) & 1)) break;
          if (more && !scores(it + 1, false)) break;
          if (i > 0 || carry_in) {
            // (later chunks' carries were waited for ahead of the last P V)
            if (i == 0) {
              if (!mbar_wait_bounded(carry_ready, cin & 1)) break;
              ++cin;
            }
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < DK / 16; ++k) {
              const uint32_t at = (s * L::kQBytes + (k >> 2) * kBlockBytes + (k & 3) * 32) >> 4;
              mma_f16(tmem + L::kInter, dq + at, ds + k * 128, i_out, k != 0);
            }
          }
          if (!last) {
            if (!mbar_wait_bounded(kw_ready, hand & 1)) break;
            ++hand;
            if (!mbar_wait_bounded(&full_v[it % VS], (it / VS) & 1)) break;
            tc_fence_after();
            const uint64_t k0 = dkt + ((s * L::kQBytes) >> 4);
#pragma unroll
            for (int k = 0; k < kC / 16; ++k) {
              mma_f16(tmem + L::kDelta, dlo + k * 128, v0 + k * 128, i_delta, k != 0);
            }
#pragma unroll
            for (int k = 0; k < kC / 16; ++k) {
              mma_f16(tmem + L::kDelta, k0 + k * 128, v0 + k * 128, i_delta, 1u);
            }
            mma_commit(delta_done);
            if (kHalf) mbar_arrive(delta_done);
            if (scored == it + 1 && !scores(it + 1, false)) break;
            // D has been read: its columns take P V
            if (!mbar_wait_bounded(carry_ready, cin & 1)) break;
            ++cin;
          }
          if (!mbar_wait_bounded(&p_ready[s], (it >> 1) & 1)) break;
          if (!mbar_wait_bounded(&full_v[it % VS], (it / VS) & 1)) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kC / 16; ++k) {
            mma_f16_ts(tmem + L::kIntra, tmem + L::kScores + s * 128 + k * 8, v0 + k * 128, i_out,
                       k != 0);
          }
          mma_commit(out_done);
          mma_commit(&empty_kv[s]);
          mbar_arrive(out_done);
          if (more && scored == it + 1 && !scores(it + 1, true)) break;
          ok = true;
        }
        unit = following;
      }
      // all products and commits are complete before TMEM is released
      mma_commit(drained);
      (void)mbar_wait_bounded(drained, 0);
    }
  } else if (warp < 12) {
    reg_dec<80>();
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;
    const float intra = a.out_scale * a.kv_scale;
    uint32_t it = 0, hand = 0;
    Waits wait;
    for (uint32_t unit = blockIdx.x; unit < visits; unit += gridDim.x) {
      const Unit u = decode_unit(args, unit, order);
      for (int i = 0; i < u.chunks; ++i, ++it) {
        const int s = it & 1;
        const int n = chunk_steps(u, chunk_t0(u, i, reverse));
        const uint32_t t_scores = tmem + L::kScores + s * 128 + (uint32_t(quarter * 32) << 16);
        wait(&full_k[s], (it >> 1) & 1);
        wait(&scores_done[s], (it >> 1) & 1);
        if (n < kC) {
          // (with one V stage these warps may be here before the last chunk left it)
          if (VS == 1 && it >= 1) wait(out_done, (it - 1) & 1);
          wait(&full_v[it % VS], (it / VS) & 1);
          if (r >= n) zero_v_row<DV>(smem + L::kV + (it % VS) * L::kVBytes, r, half);
          fence_proxy_async_smem();
        }
        tc_fence_after();
        // column blocks half and half + 2; those wholly on the other side of the
        // diagonal are zero
        auto blank = [&](int jb) { return reverse ? jb < quarter : jb > quarter; };
        auto group = [&](const uint32_t* v, int jb, int y, float (&f)[16]) {  // columns jb * 32 + y ..
          weigh16<REVERSE>(v + y, r - jb * 32 - y, n - jb * 32 - y, intra, u, f);
        };
        float scale = 1.0f;
        if constexpr (kHalf) {
          // fp16: P's rows are brought to a common magnitude by a power of two
          float top = 0.0f;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int jb = half + 2 * x;
            if (blank(jb)) continue;
            uint32_t v[32];
            tmem_ld32_issue(t_scores + jb * 32, v);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; y += 16) {
              float f[16];
              group(v, jb, y, f);
#pragma unroll
              for (int j = 0; j < 16; ++j) top = fmaxf(top, fabsf(f[j]));  // drops a NaN
            }
          }
          (half == 0 ? row_scale + s * kC : row_top)[r] = top;
          bar_sync(3 + quarter, 64);
          scale = fp16_scale(fmaxf(row_scale[s * kC + r], row_top[r]));
        }
        uint32_t p[2][16];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int jb = half + 2 * x;
          if (blank(jb)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) p[x][j] = 0;
          } else {
            uint32_t v[32];
            tmem_ld32_issue(t_scores + jb * 32, v);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; y += 16) {
              float f[16];
              group(v, jb, y, f);
#pragma unroll
              for (int j = 0; j < 16; j += 2) {
                p[x][(y + j) / 2] = kHalf ? pack2<T>(f[j] * scale, f[j + 1] * scale)
                                          : pack2<T>(f[j], f[j + 1]);
              }
            }
          }
        }
        bar_sync(3 + quarter, 64);  // both warps have read the scores that P overwrites
#pragma unroll
        for (int x = 0; x < 2; ++x) tmem_st16(t_scores + (half + 2 * x) * 16, p[x]);
        if constexpr (kHalf) {
          // for the output warps, which have read this stage's last ones (P V of
          // the chunk between waited for that)
          if (half == 0) row_scale[s * kC + r] = 1.0f / scale;
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(&p_ready[s], lane);
        if (i + 1 < u.chunks) {
          // K <- W_kv K (the scores that read K are complete), and what rounding leaves
          // of it, once the last chunk's remainders are used
          uint8_t* ks = smem + L::kK + s * L::kQBytes;
          float w = r < n ? kv_weight(u, r, n, reverse) : 0.0f;
          float k_scale = 1.0f;
          if constexpr (kHalf) k_scale = key_scale<DK>(ks, key_top + (hand & 1) * 8, r, half, w, r < n);
          if (hand >= 1) wait(delta_done, (hand - 1) & 1);
          if (kHalf && threadIdx.x == 4 * 32) key_inv[hand & 1] = 1.0f / k_scale;
          ++hand;
          weigh_k_row<T, DK, 2>(ks, smem + L::kLo, r, half, w * k_scale, r < n);
          fence_proxy_async_smem();
          warp_arrive(kw_ready, lane);
        }
      }
    }
  } else {
    reg_inc<128>();
    const int quarter = warp & 3, half = (warp - 12) >> 2;
    const int r = quarter * 32 + lane;  // row of the carry, and step of a chunk
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const int col0 = half * kCols;
    const bool holds = quarter * 32 < DK;  // warps past DK hold no carry (uniform)
    float S[kCols];
    float inv_s = 1.0f;  // fp16: 1 / scale of the carry's operand
    uint32_t put = 0;
    // the carry, rounded, as the B operand of the next chunk (rows of S, MN-major)
    auto put_carry = [&]() {
      float scale = 1.0f;
      if constexpr (kHalf) {
        float top = 0.0f;
        if (holds) {
#pragma unroll
          for (int c = 0; c < kCols; ++c) top = fmaxf(top, fabsf(S[c]));
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        }
        float* at = warp_max + (put & 1) * 8;
        ++put;
        if (lane == 0) at[warp - 12] = top;
        bar_sync(2, kGroup);
        top = at[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) top = fmaxf(top, at[w]);
        scale = fp16_scale(top);
        inv_s = 1.0f / scale;
      }
      if (holds) {
#pragma unroll
        for (int q = 0; q < kCols / 8; ++q) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = pack2<T>(S[8 * q + 2 * e] * scale, S[8 * q + 2 * e + 1] * scale);
          }
          *reinterpret_cast<uint4*>(smem + L::kS + piece_at(r, col0 / 8 + q, DK)) =
              make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      warp_arrive(carry_ready, lane);
    };
    uint32_t it = 0, hand = 0;
    Waits wait;
    for (uint32_t unit = blockIdx.x; unit < visits; unit += gridDim.x) {
      const Unit u = decode_unit(args, unit, order);
      T* o = static_cast<T*>(a.o.data) + u.b * a.o.stride_b + u.h * a.o.stride_h;
      if (u.chunks > 0) {
        const float* from = nullptr;
        int64_t sc = 1;
        if (r < a.Dk) {
          if (args.split.segments > 1) {
            from = args.split.states + (((u.seg * a.B + u.b) * a.H + u.h) * a.Dk + r) * a.Dv + col0;
          } else if (a.first.data != nullptr) {
            sc = a.first.stride_col;
            from = a.first.data + u.b * a.first.stride_b + u.h * a.first.stride_h +
                   r * a.first.stride_row + col0 * sc;
          }
        }
        load_memory_row<kCols>(from, sc, a.Dv - col0, S);
        // the last unit's operand has been read: its outputs were complete
        if (carry_in) put_carry();
      }
      bool owed = false;
      for (int i = 0; i < u.chunks; ++i, ++it) {
        const int64_t t0 = chunk_t0(u, i, reverse);
        const int n = chunk_steps(u, t0);
        const int s = it & 1;
        const float inv_now = inv_s;  // of the operand behind this chunk's Q S
        auto release = [&]() {  // the last chunk's Q stage: its outputs have left it
          if (L::kFull && owed && lane == 0) {
            tma_store_wait_read<0>();
            mbar_arrive(&empty_q[s ^ 1]);
          }
          owed = false;
        };
        if (i + 1 < u.chunks) {
          release();
          wait(delta_done, hand & 1);
          const float d_scale = kHalf ? a.kv_scale * key_inv[hand & 1] : a.kv_scale;
          ++hand;
          tc_fence_after();
          if (holds) {
            const float gn = decay_pow(u.log2g, n);
#pragma unroll
            for (int c0 = 0; c0 < kCols; c0 += 16) {
              uint32_t x[16];
              tmem_ld16_issue(tmem + L::kDelta + lanes + col0 + c0, x);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                S[c0 + j] = fmaf(gn, S[c0 + j], d_scale * __uint_as_float(x[j]));
              }
            }
          }
          put_carry();
        }
        release();
        wait(out_done, it & 1);
        tc_fence_after();
        const float w_in = kHalf ? row_scale[s * kC + r] : 1.0f;
        const bool inter = i > 0 || carry_in;
        const float w_out =
            r < n ? out_weight(u, r, n, reverse) * (a.out_scale * inv_now) : 0.0f;
        // staged as rows of 128 bytes: a block of 32 rows x 64 columns per warp, or
        // per two warps of 32 columns each; the last store has left its block
        uint8_t* block = smem + L::kO + (L::kFull ? s * L::kQBytes : 0) +
                         (kCols == 64 ? (half * 4 + quarter) : quarter) * 4096;
        if constexpr (!L::kFull) {
          if (lane == 0) tma_store_wait_read<0>();
          if (kCols == 64) __syncwarp();
          else bar_sync(7 + quarter, 64);
        }
#pragma unroll 1  // (as code that fits the instruction cache with the other warps')
        for (int c0 = 0; c0 < kCols; c0 += 16) {
          uint32_t x[16], y[16];
          tmem_ld16_issue(tmem + L::kIntra + lanes + col0 + c0, x);
          if (inter) {
            tmem_ld16_issue(tmem + L::kInter + lanes + col0 + c0, y);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) y[j] = 0;
          }
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
          // steps past the row's length are staged as zeros
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int q = (kCols == 64 ? 0 : half * 4) + c0 / 8 + e;
            *reinterpret_cast<uint4*>(block + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                make_uint4(p[4 * e], p[4 * e + 1], p[4 * e + 2], p[4 * e + 3]);
          }
        }
        tc_fence_before();
        fence_proxy_async_smem();
        warp_arrive(out_read, lane);
        if (kCols == 32) bar_sync(7 + quarter, 64);
        if (lane == 0 && (kCols == 64 || half == 0)) {
          const int c = kCols == 64 ? col0 : 0;
          const int64_t t = t0 + quarter * 32;
          if (t < u.hi && c < a.Dv) {
            tma_store_4d(&map_o, block, c, static_cast<int>(t), u.h * args.o_h, u.b * args.o_b);
          }
        }
        if (L::kFull && i + 1 < u.chunks) {
          owed = true;  // Q's stage is released under the next chunk's work
        } else if (lane == 0) {
          if (L::kFull) tma_store_wait_read<0>();
          mbar_arrive(&empty_q[s]);
        }
      }
      if (u.chunks < 0) continue;
      // whole chunks past the row's length: zeros
      for (int64_t t = u.lo + int64_t(u.chunks) * kC + r; t < u.hi; t += kC) {
        T* row = o + t * a.o.stride_t;
        for (int64_t c = col0; c < imin64(a.Dv, col0 + kCols); c += 8) {
          *reinterpret_cast<uint4*>(row + c) = make_uint4(0, 0, 0, 0);
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
  }
  tmem_free(tmem, warp);
}

// ---------------------------------------------------------------------------
// States: every unit's final memory (one segment: from `first` to `last`; more:
// each segment's own, from zero, to the workspace)
// ---------------------------------------------------------------------------
template <typename T, int DK, int DV, bool RANKED>
__global__ void __launch_bounds__(kTcThreads, 1)
    attn_states_kernel(const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ CUtensorMap map_m,
                       const __grid_constant__ TcArgs args) {
  constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 3;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  using L = StatesLayout<DK, DV, PARTS>;
  constexpr int kCols = DV / 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* key_top = reinterpret_cast<float*>(smem + L::kKeyTop);
  float* key_inv = reinterpret_cast<float*>(smem + L::kKeyInv);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* full_k = bars;      // [2]
  uint64_t* full_v = bars + 2;  // [2]
  uint64_t* empty = bars + 4;   // [2]
  uint64_t* kw_ready = bars + 6;   // [2] steps 0..63 and 64..127 of a chunk
  uint64_t* kw_used = bars + 8;    // [2] their products are complete
  uint64_t* delta_read = bars + 10;
  uint64_t* drained = bars + 11;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::kNumBars);

  const mb_decay_attention_args& a = args.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const bool reverse = a.reverse != 0;
  const bool whole = args.split.segments == 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&full_k[s], 1);
      mbar_init(&full_v[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&kw_ready[s], 4);
      // fp16: the second with the scale that the keys' weighers wrote
      mbar_init(&kw_used[s], kHalf && s == 1 ? 2 : 1);
    }
    mbar_init(delta_read, 8);
    mbar_init(drained, 1);
    fence_barrier_init();
  }
  uint16_t* order = RANKED ? reinterpret_cast<uint16_t*>(smem + L::kOrder) : nullptr;
  if constexpr (RANKED) rank_rows(args, order);
  const uint32_t tmem = tmem_alloc(tmem_slot, warp);
  const uint32_t visits = unit_visits(args, order);

  if (warp < 4) {
    reg_dec<56>();
    if (warp == 0 && elect_one()) {
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t unit = blockIdx.x; unit < visits && ok; unit += gridDim.x) {
        const Unit u = decode_unit(args, unit, order);
        const int kh = u.h * args.k_h, kb = u.b * args.k_b, vh = u.h * args.v_h,
                  vb = u.b * args.v_b;
        for (int i = 0; i < u.chunks; ++i, ++it) {
          const int s = it & 1;
          const int t = static_cast<int>(chunk_t0(u, i, reverse));
          if (it >= 2 && !mbar_wait_bounded(&empty[s], ((it >> 1) - 1) & 1)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full_k[s], L::kKBytes);
          mbar_arrive_expect_tx(&full_v[s], L::kVBytes);
#pragma unroll
          for (int x = 0; x < DK / 64; ++x) {
            tma_load_4d(smem + L::kK + s * L::kKBytes + x * kBlockBytes, &map_k, x * 64, t, kh, kb,
                        &full_k[s]);
          }
#pragma unroll
          for (int x = 0; x < DV / 64; ++x) {
            tma_load_4d(smem + L::kV + s * L::kVBytes + x * kBlockBytes, &map_v, x * 64, t, vh, vb,
                        &full_v[s]);
          }
        }
      }
      for (uint32_t j = it > 2 ? it - 2 : 0; j < it; ++j) {
        (void)mbar_wait_bounded(&full_k[j & 1], (j >> 1) & 1);
        (void)mbar_wait_bounded(&full_v[j & 1], (j >> 1) & 1);
      }
    } else if (warp == 1 && elect_one()) {
      const uint32_t i_delta = tc_idesc<T>(DV, true, true);
      const uint64_t dk = mn_desc(smem_addr(smem + L::kK), kBlockBytes);
      const uint64_t dlo = mn_desc(smem_addr(smem + L::kLo), kBlockBytes);
      const uint64_t dv = mn_desc(smem_addr(smem + L::kV), kBlockBytes);
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t unit = blockIdx.x; unit < visits && ok; unit += gridDim.x) {
        const Unit u = decode_unit(args, unit, order);
        for (int i = 0; i < u.chunks; ++i, ++it) {
          const int s = it & 1;
          ok = false;
          if (!mbar_wait_bounded(&full_v[s], (it >> 1) & 1)) break;
          if (it >= 1 && !mbar_wait_bounded(delta_read, (it - 1) & 1)) break;
          const uint64_t k0 = dk + ((s * L::kKBytes) >> 4), v0 = dv + ((s * L::kVBytes) >> 4);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (!mbar_wait_bounded(&kw_ready[x], it & 1)) break;
            tc_fence_after();
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) {  // the smallest parts first
              const uint64_t p0 = part == 0 ? k0 : dlo + (((part - 1) * L::kKBytes) >> 4);
#pragma unroll
              for (int k = 4 * x; k < 4 * x + 4; ++k) {
                mma_f16(tmem + L::kDelta, p0 + k * 128, v0 + k * 128, i_delta,
                        (x != 0 || part != PARTS - 1 || k != 0) ? 1u : 0u);
              }
            }
            mma_commit(&kw_used[x]);
            if (kHalf && x == 1) mbar_arrive(&kw_used[x]);
            ok = x == 1;
          }
          if (!ok) break;
          mma_commit(&empty[s]);
        }
      }
      mma_commit(drained);
      (void)mbar_wait_bounded(drained, 0);
    }
  } else if (warp < 12) {
    reg_dec<80>();
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;
    uint32_t it = 0;
    Waits wait;
    for (uint32_t unit = blockIdx.x; unit < visits; unit += gridDim.x) {
      const Unit u = decode_unit(args, unit, order);
      for (int i = 0; i < u.chunks; ++i, ++it) {
        const int s = it & 1;
        const int n = chunk_steps(u, chunk_t0(u, i, reverse));
        uint8_t* ks = smem + L::kK + s * L::kKBytes;
        wait(&full_k[s], (it >> 1) & 1);
        if (n < kC) {
          wait(&full_v[s], (it >> 1) & 1);
          if (r >= n) zero_v_row<DV>(smem + L::kV + s * L::kVBytes, r, half);
        }
        float w = r < n ? kv_weight(u, r, n, reverse) : 0.0f;
        float k_scale = 1.0f;
        if constexpr (kHalf) k_scale = key_scale<DK>(ks, key_top + s * 8, r, half, w, r < n);
        // the further parts' buffers are free once the last chunk's products are
        // complete; the two halves of a chunk's steps go through on their own
        if (it >= 1) wait(&kw_used[r >> 6], (it - 1) & 1);
        // (the last chunk but one's has been read: its sums left the accumulator before
        // the last chunk's second half was issued)
        if (kHalf && threadIdx.x == 6 * 32) key_inv[s] = 1.0f / k_scale;
        weigh_k_row<T, DK, PARTS>(ks, smem + L::kLo, r, half, w * k_scale, r < n);
        fence_proxy_async_smem();
        warp_arrive(&kw_ready[r >> 6], lane);
      }
    }
  } else {
    reg_inc<128>();
    const int quarter = warp & 3, half = (warp - 12) >> 2;
    const int r = quarter * 32 + lane;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    const int col0 = half * kCols;
    const bool holds = quarter * 32 < DK;
    const bool row_ok = r < a.Dk && col0 < a.Dv;
    uint32_t it = 0;
    Waits wait;
    for (uint32_t unit = blockIdx.x; unit < visits; unit += gridDim.x) {
      const Unit u = decode_unit(args, unit, order);
      if (u.chunks < 0) continue;
      float S[kCols];
      const float* from = nullptr;
      float* to = nullptr;
      int64_t from_sc = 1, to_sc = 1;
      if (row_ok) {
        if (whole) {
          if (a.first.data != nullptr) {
            from_sc = a.first.stride_col;
            from = a.first.data + u.b * a.first.stride_b + u.h * a.first.stride_h +
                   r * a.first.stride_row + col0 * from_sc;
          }
          to_sc = a.last.stride_col;
          to = a.last.data + u.b * a.last.stride_b + u.h * a.last.stride_h +
               r * a.last.stride_row + col0 * to_sc;
        } else {
          to = args.split.states + (((u.seg * a.B + u.b) * a.H + u.h) * a.Dk + r) * a.Dv + col0;
        }
      }
      load_memory_row<kCols>(from, from_sc, a.Dv - col0, S);
      for (int i = 0; i < u.chunks; ++i, ++it) {
        const int n = chunk_steps(u, chunk_t0(u, i, reverse));
        // (the second half's products come after the first's)
        wait(&kw_used[1], it & 1);
        const float d_scale = kHalf ? a.kv_scale * key_inv[it & 1] : a.kv_scale;
        tc_fence_after();
        if (holds) {
          const float gn = decay_pow(u.log2g, n);
#pragma unroll
          for (int c0 = 0; c0 < kCols; c0 += 16) {
            uint32_t x[16];
            tmem_ld16_issue(tmem + L::kDelta + lanes + col0 + c0, x);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              S[c0 + j] = fmaf(gn, S[c0 + j], d_scale * __uint_as_float(x[j]));
            }
          }
        }
        tc_fence_before();
        warp_arrive(delta_read, lane);
      }
      if (args.m_map) {
        // whole 128-byte rows by tensor stores, 32 x 32 values at a time (a lane's own
        // row-wise stores touch 32 lines per instruction)
        if (holds) {
          uint8_t* block = smem + L::kOut + (warp - 12) * 4096;
#pragma unroll
          for (int c0 = 0; c0 < kCols; c0 += 32) {
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
            float x[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = S[c0 + j];
            stage_row32<float>(block, lane, 0, x);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && quarter * 32 < a.Dk && col0 + c0 < a.Dv) {
              const int z = static_cast<int>(whole ? u.b : u.seg * a.B + u.b);
              tma_store_4d(&map_m, block, col0 + c0, quarter * 32, u.h, z);
            }
          }
        }
      } else {
        store_memory_row<kCols>(to, to_sc, a.Dv - col0, S);
      }
    }
    if (lane == 0) tma_store_wait_all();
  }
  tmem_free(tmem, warp);
}

// A [d, t, h, b] map of 64-column boxes of `rows` steps; a dimension of stride 0 or size 1 has
// extent 1 and its coordinate multiplied by 0.
bool make_attn_map(CUtensorMap* map, const mb_steps& x, int64_t T, int64_t H, int64_t B, int64_t D,
                   bool bf16, int rows, int32_t* h_on, int32_t* b_on) {
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
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1};
  cuuint32_t estride[4] = {1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            x.data, dims, strides, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A [col, row, h, b] map of 32 x 32 boxes over the memories that the states kernel
// writes: `last`, or with several segments the workspace (its segments and rows as
// one dimension). False where their rows are not whole 16-byte pieces.
bool make_memory_map(CUtensorMap* map, const mb_decay_attention_args& a, const AttnSplit& split) {
  auto fn = tma_encode_fn();
  mb_memory m = a.last;
  int64_t outer = a.B;
  if (split.segments > 1) {
    m.data = split.states;
    m.stride_col = 1;
    m.stride_row = a.Dv;
    m.stride_h = a.Dk * a.Dv;
    m.stride_b = a.H * m.stride_h;
    outer = split.segments * a.B;
  }
  if (fn == nullptr || m.stride_col != 1 || !aligned_to(m.data, 16)) return false;
  const int64_t strides64[3] = {m.stride_row, a.H > 1 ? m.stride_h : 4, outer > 1 ? m.stride_b : 4};
  for (int64_t x : strides64) {
    if (x <= 0 || x % 4 != 0 || x >= (int64_t(1) << 37)) return false;
  }
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.Dv), static_cast<cuuint64_t>(a.Dk),
                        static_cast<cuuint64_t>(a.H), static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(strides64[0] * 4),
                           static_cast<cuuint64_t>(strides64[1] * 4),
                           static_cast<cuuint64_t>(strides64[2] * 4)};
  cuuint32_t box[4] = {32, 32, 1, 1};
  cuuint32_t estride[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, m.data, dims, strides, box, estride,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int attn_sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n > 0 ? n : 148;
}

template <typename T, int DK, int DV>
int launch_tc(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
              const CUtensorMap& mo, TcArgs args, bool states, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(imin64(args.units, attn_sm_count()));
  // rows of different lengths, in more than one turn of the CTAs
  const bool ranked =
      args.a.lengths != nullptr && args.a.B > 1 && args.a.B <= kMaxOrder && args.units > grid;
  if (states) {
    constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 3;
    constexpr size_t smem = StatesLayout<DK, DV, PARTS>::kSmem;
    auto kern = ranked ? attn_states_kernel<T, DK, DV, true> : attn_states_kernel<T, DK, DV, false>;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    CUtensorMap mm;
    memset(&mm, 0, sizeof(mm));
    args.m_map = make_memory_map(&mm, args.a, args.split) ? 1 : 0;
    kern<<<grid, kTcThreads, smem, s>>>(mk, mv, mm, args);
    MB_CHECK_LAUNCH("mb_decay_attention (states)");
  } else {
    constexpr size_t smem = OutLayout<DK, DV>::kSmem;
    auto kern = args.a.reverse != 0
                    ? (ranked ? attn_out_kernel<T, DK, DV, true, true>
                              : attn_out_kernel<T, DK, DV, true, false>)
                    : (ranked ? attn_out_kernel<T, DK, DV, false, true>
                              : attn_out_kernel<T, DK, DV, false, false>);
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    kern<<<grid, kTcThreads, smem, s>>>(mq, mk, mv, mo, args);
    MB_CHECK_LAUNCH("mb_decay_attention (outputs)");
  }
  return 0;
}

template <typename T>
int launch_type(const mb_decay_attention_args& a, const AttnSplit& split, bool states,
                cudaStream_t s) {
  TcArgs args;
  args.a = a;
  args.split = split;
  args.units = split.segments * a.B * a.H;
  MB_CHECK_ARG(args.units < (int64_t(1) << 31) - 65536,
               "mb_decay_attention: too many (batch, head) rows");
  args.m_map = 0;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap mq, mk, mv, mo;
  MB_CHECK_ARG(make_attn_map(&mq, a.q, a.T, a.H, a.B, a.Dk, bf16, kC, &args.q_h, &args.q_b) &&
                   make_attn_map(&mk, a.k, a.T, a.H, a.B, a.Dk, bf16, kC, &args.k_h, &args.k_b) &&
                   make_attn_map(&mv, a.v, a.T, a.H, a.B, a.Dv, bf16, kC, &args.v_h, &args.v_b) &&
                   make_attn_map(&mo, a.o, a.T, a.H, a.B, a.Dv, bf16, 32, &args.o_h, &args.o_b),
               "mb_decay_attention: cuTensorMapEncodeTiled failed (shape or alignment)");
  const bool k64 = a.Dk <= 64, v64 = a.Dv <= 64;
  if (k64 && v64) return launch_tc<T, 64, 64>(mq, mk, mv, mo, args, states, s);
  if (k64) return launch_tc<T, 64, 128>(mq, mk, mv, mo, args, states, s);
  if (v64) return launch_tc<T, 128, 64>(mq, mk, mv, mo, args, states, s);
  return launch_tc<T, 128, 128>(mq, mk, mv, mo, args, states, s);
}

// Rows that the tensor-map copies and 16-byte stores take: 16-byte base and strides.
bool steps_ok(const mb_steps& x, int64_t T) {
  const int64_t limit = int64_t(1) << 38;  // strides below 2^40 bytes
  return aligned_to(x.data, 16) && x.stride_t % 8 == 0 && x.stride_h % 8 == 0 &&
         x.stride_b % 8 == 0 && x.stride_t >= 0 && x.stride_h >= 0 && x.stride_b >= 0 &&
         x.stride_t < limit && x.stride_h < limit && x.stride_b < limit &&
         (T <= 1 || x.stride_t > 0);
}

}  // namespace

bool attn_tc_supported(const mb_decay_attention_args& a) {
  if (a.dtype == MB_F32 || a.Dk > 128 || a.Dv > 128 || a.T < kTcMinSteps) return false;
  const bool o_dense = (a.H == 1 || a.o.stride_h > 0) && (a.B == 1 || a.o.stride_b > 0);
  return a.Dv % 8 == 0 && o_dense && steps_ok(a.q, a.T) && steps_ok(a.k, a.T) &&
         steps_ok(a.v, a.T) && steps_ok(a.o, a.T);
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

int attn_tc_launch(const mb_decay_attention_args& a, const AttnSplit& split, bool states,
                   cudaStream_t stream) {
  return a.dtype == MB_BF16 ? launch_type<__nv_bfloat16>(a, split, states, stream)
                            : launch_type<__half>(a, split, states, stream);
}

int attention_unit_status(bool clear) { return read_device_status(clear); }

cudaError_t attention_unit_wait_probe(uint32_t polls, cudaStream_t stream) {
  wait_timeout_probe_kernel<<<1, 32, 0, stream>>>(polls);
  return cudaGetLastError();
}

}  // namespace mb
