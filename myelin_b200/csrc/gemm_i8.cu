// Dense projection in 8-bit integers with a scale for each row and each output
// channel:
//
//   C[m, n] = a_scale[m] b_scale[n] sum_k A[m, k] B[n, k] (+ bias[n])
//
// A, B signed 8-bit, sums exact in int32, one fp32 scaling and one rounding to
// the output type. Also the quantisation of rows that feeds it:
//
//   scale = max|x| / 127,  q = round(x * (127 / max|x|)), ties to even.
//
// Three kernels by size:
// - up to kRowsMax input rows: every block streams a few weight rows through
//   dp4a, bound by the weights' bytes; floating rows are quantised inside it
//   (each block repeats that for its copy: no second launch);
// - otherwise tcgen05.mma kind::i8 (twice the 16-bit rate) on tiles of 128 x BN
//   per SM, or 256 x 256 per SM pair for large products.
#include <cuda.h>
#include <math.h>

#include <cstring>

#include "async_copy.cuh"
#include "common.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace mb {
namespace {

// ---------------------------------------------------------------------------
// Quantisation
// ---------------------------------------------------------------------------
constexpr float kTinyRow = 1e-30f;  // rows whose largest value is below this count as zero

struct RowScale {
  float inv;    // 127 / top, 0 for a zero row and for one that is not finite
  float scale;  // top / 127, 0 for a zero row, NaN for one that is not finite
};

__device__ __forceinline__ RowScale row_scale(float top) {
  if (!(top < INFINITY)) return RowScale{0.0f, __int_as_float(0x7fffffff)};
  if (top < kTinyRow) return RowScale{0.0f, 0.0f};
  return RowScale{__fdiv_rn(127.0f, top), __fdiv_rn(top, 127.0f)};
}

// Magnitudes as bit patterns: ordered like the numbers, with NaN above infinity, so
// that an integer maximum keeps a NaN (fmaxf would drop it).
__device__ __forceinline__ uint32_t top_of(uint32_t top, float x) {
  return max(top, __float_as_uint(x) & 0x7fffffffu);
}

// Eight (fewer) values times inv, rounded to integers, as bytes. Adding 1.5 * 2^23
// rounds to the nearest integer (ties to even) and leaves it in the low bits; the
// product is rounded on its own first, as the definition has it. |x| inv is at most
// 127 (1 + 2^-22). A row with inv = 0 is zero whatever it holds.
__device__ __forceinline__ uint32_t quantize_bits(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.0f));
}
__device__ __forceinline__ int8_t quantize(float x, float inv) {
  return inv == 0.0f ? int8_t(0) : static_cast<int8_t>(quantize_bits(x, inv) & 0xffu);
}
template <typename T>
__device__ __forceinline__ uint32_t quantize4(const T* v, float inv) {
  if (inv == 0.0f) return 0u;
  const uint32_t a = quantize_bits(Elem<T>::to_f(v[0]), inv);
  const uint32_t b = quantize_bits(Elem<T>::to_f(v[1]), inv);
  const uint32_t c = quantize_bits(Elem<T>::to_f(v[2]), inv);
  const uint32_t d = quantize_bits(Elem<T>::to_f(v[3]), inv);
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Largest magnitude of one 16-byte piece, joined with `top`: the bits of one fp32, or
// of two 16-bit values side by side (each half its own maximum).
template <typename T>
__device__ __forceinline__ uint32_t piece_top(uint32_t top, const uint4& x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    top = sizeof(T) == 2 ? __vmaxu2(top, w[i] & 0x7fff7fffu) : max(top, w[i] & 0x7fffffffu);
  }
  return top;
}

// The maximum that piece_top gathered, as an fp32 value's bits.
template <typename T>
__device__ __forceinline__ uint32_t whole_top(uint32_t top) {
  if constexpr (sizeof(T) == 2) {
    const uint16_t half = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
    return __float_as_uint(Elem<T>::to_f(*reinterpret_cast<const T*>(&half)));
  } else {
    return top;
  }
}

// A piece quantised: 8 bytes of a 16-bit type's values, 4 of fp32's.
template <typename T>
__device__ __forceinline__ void put_piece(int8_t* q, const uint4& x, float inv) {
  const T* v = reinterpret_cast<const T*>(&x);
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint2*>(q) = make_uint2(quantize4<T>(v, inv), quantize4<T>(v + 4, inv));
  } else {
    *reinterpret_cast<uint32_t*>(q) = quantize4<T>(v, inv);
  }
}

// TPR threads per row, HOLD 16-byte pieces of it in registers between the two passes
// (all on their way at once); what is longer, or not aligned, is read twice. Bound by
// DRAM: 3 bytes per 16-bit value (5 per fp32). A warp that holds a whole row needs no
// barrier; a block per row of 4096 columns reached 2.8 TB/s.
template <typename T, int TPR, int HOLD>
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t ldx,
                         int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale) {
  constexpr int RPB = 256 / TPR;
  constexpr int E = 16 / sizeof(T);
  __shared__ uint32_t tops[8];
  const int t = threadIdx.x % TPR;
  const int64_t row = int64_t(blockIdx.x) * RPB + threadIdx.x / TPR;
  const bool ok = row < rows;
  const T* xr = x + row * ldx;
  int8_t* qr = q + row * ldq;
  uint32_t top = 0;
  uint4 held[HOLD > 0 ? HOLD : 1];
  const int pieces = HOLD > 0 && ok ? cols / E : 0;
  const uint4* xp = reinterpret_cast<const uint4*>(xr);
  if constexpr (HOLD > 0) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      if (i * TPR + t < pieces) held[i] = xp[i * TPR + t];
    }
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      if (i * TPR + t < pieces) top = piece_top<T>(top, held[i]);
    }
    for (int p = HOLD * TPR + t; p < pieces; p += TPR) top = piece_top<T>(top, xp[p]);
    top = whole_top<T>(top);
  } else if (ok) {
    for (int c = t; c < cols; c += TPR) top = top_of(top, Elem<T>::to_f(xr[c]));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = tops[0];
#pragma unroll
    for (int w = 1; w < TPR / 32; ++w) top = max(top, tops[w]);
  }
  if (!ok) return;
  const RowScale rs = row_scale(__uint_as_float(top));
  if (t == 0) scale[row] = rs.scale;
  if constexpr (HOLD > 0) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      const int p = i * TPR + t;
      if (p < pieces) put_piece<T>(qr + p * E, held[i], rs.inv);
    }
    for (int p = HOLD * TPR + t; p < pieces; p += TPR) put_piece<T>(qr + p * E, xp[p], rs.inv);
  } else {
    for (int c = t; c < cols; c += TPR) qr[c] = quantize(Elem<T>::to_f(xr[c]), rs.inv);
  }
}

template <typename T, int TPR, int HOLD>
int launch_quantize_as(const T* x, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq,
                       float* scale, cudaStream_t s) {
  const int64_t blocks = ceil_div(rows, 256 / TPR);
  MB_CHECK_ARG(blocks <= 0x7fffffff, "mb_quantize_rows: too many rows");
  quantize_rows_kernel<T, TPR, HOLD><<<static_cast<unsigned>(blocks), 256, 0, s>>>(
      x, rows, static_cast<int>(cols), ldx, q, ldq, scale);
  MB_CHECK_LAUNCH("mb_quantize_rows");
  return 0;
}

// A warp per row while the row fits its registers, else the whole block.
template <typename T>
int launch_quantize(const void* x, int64_t rows, int64_t cols, int64_t ldx, int8_t* q,
                    int64_t ldq, float* scale, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const T* xs = static_cast<const T*>(x);
  const bool vector = cols % E == 0 && aligned_to(x, 16) && ldx % E == 0 && aligned_to(q, 8) &&
                      ldq % 8 == 0;
  const int64_t pieces = cols / E;
  if (!vector) {
    return cols <= 1024 ? launch_quantize_as<T, 32, 0>(xs, rows, cols, ldx, q, ldq, scale, s)
                        : launch_quantize_as<T, 256, 0>(xs, rows, cols, ldx, q, ldq, scale, s);
  }
  if (pieces <= 4 * 32) return launch_quantize_as<T, 32, 4>(xs, rows, cols, ldx, q, ldq, scale, s);
  if (pieces <= 16 * 32) return launch_quantize_as<T, 32, 16>(xs, rows, cols, ldx, q, ldq, scale, s);
  return launch_quantize_as<T, 256, 4>(xs, rows, cols, ldx, q, ldq, scale, s);
}

// ---------------------------------------------------------------------------
// Scaling of finished sums
// ---------------------------------------------------------------------------
struct I8Args {
  const float* a_scale;  // [M] or null (1)
  const float* b_scale;  // [N]
  const void* bias;      // [N] or null
  int bias_dtype;
  void* C;
  int64_t ldc;
  int64_t M, N, K;
  int tma_store;  // C rows are whole 16-byte pieces: bulk tensor stores
};

__device__ __forceinline__ float load_bias(const I8Args& a, int64_t n) {
  if (a.bias == nullptr) return 0.0f;
  if (a.bias_dtype == MB_F32) return static_cast<const float*>(a.bias)[n];
  if (a.bias_dtype == MB_BF16) {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n]);
  }
  return __half2float(static_cast<const __half*>(a.bias)[n]);
}

// One finished sum. The channel's scale first: the scales' own product may leave fp32's
// range where the result does not (rows of 1e-23 by weights of 1e-13), and a sum of 0 by
// an infinite product would be NaN.
__device__ __forceinline__ float scaled(int32_t acc, float sa, float sb, float bias) {
  return fmaf(static_cast<float>(acc) * sb, sa, bias);
}

// ---------------------------------------------------------------------------
// Few rows: C for M <= kRowsMax
// ---------------------------------------------------------------------------
constexpr int kRowsMax = 4;
constexpr int kRowsThreads = 256;
constexpr int kRowsVecs = 8;                   // 16-byte weight pieces in flight per lane
constexpr int64_t kRowsMaxBytes = 32 * 1024;   // staged input rows: M x K bytes

// X: the input element type (int8_t: already integers, a_scale applies).
// A warp owns one output channel: its lanes read the weight row 16 bytes at a
// time, the first pieces before the input is staged so that both latencies
// overlap, and the channel's partial sums are joined by shuffles.
template <typename X, typename TOut, int M>
__global__ void __launch_bounds__(kRowsThreads)
    linear_i8_rows_kernel(const X* __restrict__ x, int64_t ldx, const int8_t* __restrict__ w,
                          int64_t ldw, const __grid_constant__ I8Args args) {
  extern __shared__ __align__(16) int8_t sx[];  // [M][K rounded up to 16]
  __shared__ uint32_t tops[M][kRowsThreads / 32];
  __shared__ float sscale[M];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kWarps = kRowsThreads / 32;
  const int64_t K = args.K, Kp = (K + 15) / 16 * 16;
  const int64_t pieces = K / 16;
  int64_t n = int64_t(blockIdx.x) * kWarps + warp;  // this warp's channels: every gridDim * 8th

  int4 held[kRowsVecs];
  auto fetch = [&](int64_t channel) {  // the first pieces of a weight row
    const int8_t* wr = w + channel * ldw;
#pragma unroll
    for (int i = 0; i < kRowsVecs; ++i) {
      const int64_t p = int64_t(i) * 32 + lane;
      if (channel < args.N && p < pieces) held[i] = __ldg(reinterpret_cast<const int4*>(wr) + p);
    }
  };
  fetch(n);

  if constexpr (sizeof(X) == 1) {
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const X* xr = x + m * ldx;
      if ((reinterpret_cast<uintptr_t>(xr) & 15) == 0) {
        for (int64_t p = threadIdx.x; p < pieces; p += kRowsThreads) {
          *reinterpret_cast<int4*>(sx + m * Kp + p * 16) = *reinterpret_cast<const int4*>(xr + p * 16);
        }
        for (int64_t c = pieces * 16 + threadIdx.x; c < Kp; c += kRowsThreads) {
          sx[m * Kp + c] = c < K ? static_cast<int8_t>(xr[c]) : int8_t(0);
        }
      } else {
        for (int64_t c = threadIdx.x; c < Kp; c += kRowsThreads) {
          sx[m * Kp + c] = c < K ? static_cast<int8_t>(xr[c]) : int8_t(0);
        }
      }
    }
    if (threadIdx.x < M) {
      sscale[threadIdx.x] = args.a_scale != nullptr ? args.a_scale[threadIdx.x] : 1.0f;
    }
    __syncthreads();
  } else {
    constexpr int E = 16 / sizeof(X);
    using V = Vec<X, E>;
    const bool vector = K % E == 0 && ldx % E == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    uint32_t top[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      top[m] = 0;
      if (vector) {
        for (int64_t c = int64_t(threadIdx.x) * E; c < K; c += kRowsThreads * E) {
          const V v = load_vec<X, E>(x + m * ldx + c);
#pragma unroll
          for (int j = 0; j < E; ++j) top[m] = top_of(top[m], Elem<X>::to_f(v.v[j]));
        }
      } else {
        for (int64_t c = threadIdx.x; c < K; c += kRowsThreads) {
          top[m] = top_of(top[m], Elem<X>::to_f(x[m * ldx + c]));
        }
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        top[m] = max(top[m], __shfl_xor_sync(0xffffffffu, top[m], d));
      }
      if (lane == 0) tops[m][warp] = top[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      uint32_t t = tops[m][0];
#pragma unroll
      for (int i = 1; i < kWarps; ++i) t = max(t, tops[m][i]);
      const RowScale rs = row_scale(__uint_as_float(t));
      if (threadIdx.x == 0) sscale[m] = rs.scale;
      // the row again, from L1 or L2
      if (vector) {
        for (int64_t c = int64_t(threadIdx.x) * E; c < K; c += kRowsThreads * E) {
          const V v = load_vec<X, E>(x + m * ldx + c);
#pragma unroll
          for (int j = 0; j < E; j += 4) {
            *reinterpret_cast<uint32_t*>(sx + m * Kp + c + j) = quantize4<X>(v.v + j, rs.inv);
          }
        }
        for (int64_t c = K + threadIdx.x; c < Kp; c += kRowsThreads) sx[m * Kp + c] = 0;
      } else {
        for (int64_t c = threadIdx.x; c < Kp; c += kRowsThreads) {
          sx[m * Kp + c] = c < K ? quantize(Elem<X>::to_f(x[m * ldx + c]), rs.inv) : int8_t(0);
        }
      }
    }
    __syncthreads();
  }
  for (; n < args.N; n += int64_t(gridDim.x) * kWarps) {
    const int8_t* wr = w + n * ldw;
    int acc[M];
#pragma unroll
    for (int m = 0; m < M; ++m) acc[m] = 0;
    for (int64_t p0 = 0; p0 < pieces; p0 += kRowsVecs * 32) {
#pragma unroll
      for (int i = 0; i < kRowsVecs; ++i) {
        const int64_t p = p0 + i * 32 + lane;
        if (p >= pieces) continue;
        const int4 b = held[i];
        const int64_t ahead = p + kRowsVecs * 32;
        if (ahead < pieces) held[i] = __ldg(reinterpret_cast<const int4*>(wr) + ahead);
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const int4 a = *reinterpret_cast<const int4*>(sx + m * Kp + p * 16);
          acc[m] = __dp4a(a.x, b.x, acc[m]);
          acc[m] = __dp4a(a.y, b.y, acc[m]);
          acc[m] = __dp4a(a.z, b.z, acc[m]);
          acc[m] = __dp4a(a.w, b.w, acc[m]);
        }
      }
    }
    const int64_t c = pieces * 16 + lane;  // the row's last K % 16 bytes, one per lane
    if (c < K) {
#pragma unroll
      for (int m = 0; m < M; ++m) acc[m] += int(sx[m * Kp + c]) * int(wr[c]);
    }
    fetch(n + int64_t(gridDim.x) * kWarps);
#pragma unroll
    for (int m = 0; m < M; ++m) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], d);
    }
    if (lane == 0) {
      const float sb = args.b_scale[n], bias = load_bias(args, n);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        static_cast<TOut*>(args.C)[m * args.ldc + n] =
            Elem<TOut>::from_f(scaled(acc[m], sscale[m], sb, bias));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Tensor cores
// ---------------------------------------------------------------------------
constexpr int kI8BK = 128;  // K elements per stage: one 128-byte swizzle row
constexpr int kI8UmmaK = 32;

// kind::i8 instruction descriptor: signed A and B (both K-major), int32 sums.
__device__ __forceinline__ uint32_t i8_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// 2-D load whose bytes are counted on the barrier at cluster address `bar`
// (the pair leader's). Loads of this GPU's own memory only.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int c0, int c1,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

// Drains a warp's 32 accumulator rows (TMEM address `taddr`) x COLS columns from
// output column col0: scale, bias, one rounding, 128-byte-wide pieces through
// the staging block `slot` (32 rows x 128 bytes, swizzled), written by bulk
// tensor stores or, where C's rows are not whole 16-byte pieces, row by row with
// the lanes along the columns. `cols` (COLS pairs in shared memory, this warp's)
// holds each column's scale and bias: broadcast reads.
template <typename TOut, int COLS>
__device__ __forceinline__ void drain_i8(uint32_t taddr, int64_t row0, int64_t col0, int lane,
                                         const I8Args& args, const CUtensorMap* map, float sa,
                                         const float2* cols, uint8_t* slot) {
  // 32-column chunks per staged block (a 32-wide tile of 16-bit values fills half of one)
  constexpr int kPerStore = sizeof(TOut) == 4 || COLS == 32 ? 1 : 2;
  uint32_t r[32];
#pragma unroll
  for (int ci = 0; ci < COLS / 32; ++ci) {
    const int64_t block0 = col0 + (ci / kPerStore) * kPerStore * 32;
    if (block0 >= args.N || row0 >= args.M) break;  // warp-uniform
    tmem_ld32_issue(taddr + ci * 32, r);
    tmem_wait_ld();
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const float4 two = *reinterpret_cast<const float4*>(cols + ci * 32 + j);
      v[j] = scaled(static_cast<int32_t>(r[j]), sa, two.x, two.y);
      v[j + 1] = scaled(static_cast<int32_t>(r[j + 1]), sa, two.z, two.w);
    }
    const int part = ci % kPerStore;
    if (part == 0) {  // the slot's last block has been written out
      if (args.tma_store && lane == 0) tma_store_wait_read<0>();
      __syncwarp();
    }
    stage_row32<TOut>(slot, lane, part, v);
    if (part != kPerStore - 1) continue;
    if (args.tma_store) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tma_store_2d(map, slot, static_cast<int>(block0), static_cast<int>(row0));
    } else {
      __syncwarp();
      constexpr int W = 32 * kPerStore;
      const int rows = static_cast<int>(imin64(32, args.M - row0));
      TOut* c = static_cast<TOut*>(args.C) + row0 * args.ldc + block0;
#pragma unroll 1
      for (int i0 = 0; i0 < rows; i0 += 8) {  // eight rows' reads in flight
        TOut held[8][W / 32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int j = 0; j < W / 32; ++j) {
            const int byte = (j * 32 + lane) * int(sizeof(TOut));
            const int at = (i0 + i) * 128 + (((byte >> 4) ^ i) << 4) + (byte & 15);
            held[i][j] = *reinterpret_cast<const TOut*>(slot + at);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int j = 0; j < W / 32; ++j) {
            const int e = j * 32 + lane;
            if (i0 + i < rows && block0 + e < args.N) c[(i0 + i) * args.ldc + e] = held[i][j];
          }
        }
      }
    }
  }
}

template <int COLS>
__device__ __forceinline__ void load_cols(float2* cols, int64_t col0, int lane,
                                          const I8Args& args) {
#pragma unroll
  for (int i = 0; i < COLS / 32; ++i) {
    const int64_t n = col0 + i * 32 + lane;
    cols[i * 32 + lane] = n < args.N ? make_float2(args.b_scale[n], load_bias(args, n))
                                     : make_float2(0.0f, 0.0f);
  }
  __syncwarp();
}

__device__ __forceinline__ float row_a_scale(const I8Args& args, int64_t row) {
  return args.a_scale == nullptr ? 1.0f : row < args.M ? args.a_scale[row] : 0.0f;
}

// One SM: tiles of 128 x BN, 6 warps (copies, MMAs, 4 drain warps), two
// accumulators so that a tile drains under the next one's products.
template <int BN>
struct I8Layout {
  static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr int kABytes = 128 * kI8BK;
  static constexpr int kBBytes = BN * kI8BK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kSlotBytes = 32 * 128;
  static constexpr int kColBytes = BN * 8;
  static constexpr int kBarrierBytes = 256;
  static constexpr size_t kSmem =
      size_t(kStages) * kStageBytes + 4 * (kSlotBytes + kColBytes) + kBarrierBytes + 1024;
  static constexpr uint32_t kTmemCols = 2 * BN;
};
constexpr int kI8Threads = 192;

template <typename TOut, int BN>
__global__ void __launch_bounds__(kI8Threads, 1)
    gemm_i8_kernel(const __grid_constant__ CUtensorMap tma_a,
                   const __grid_constant__ CUtensorMap tma_b,
                   const __grid_constant__ CUtensorMap tma_c, const __grid_constant__ I8Args args) {
  using L = I8Layout<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* sa = smem;
  uint8_t* sb = sa + L::kStages * L::kABytes;
  uint8_t* sslot = sb + L::kStages * L::kBBytes;
  uint8_t* scol = sslot + 4 * L::kSlotBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(scol + 4 * L::kColBytes);
  uint64_t* empty = full + L::kStages;
  uint64_t* acc_full = empty + L::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drained = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n_tiles = (args.N + BN - 1) / BN;
  const int64_t tiles = (args.M + 127) / 128 * n_tiles;
  const int kblocks = static_cast<int>((args.K + kI8BK - 1) / kI8BK);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
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
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
        const int row = static_cast<int>(tile / n_tiles * 128);
        const int col = static_cast<int>(tile % n_tiles * BN);
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = static_cast<int>(it % L::kStages);
          const uint32_t use = it / L::kStages;
          if (use > 0 && !mbar_wait_bounded(&empty[s], (use - 1) & 1)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], L::kStageBytes);
          tma_load_box_2d(sa + s * L::kABytes, &tma_a, kb * kI8BK, row, &full[s]);
          tma_load_box_2d(sb + s * L::kBBytes, &tma_b, kb * kI8BK, col, &full[s]);
        }
      }
      // every issued copy has landed before the CTA can retire
      for (uint32_t j = it > L::kStages ? it - L::kStages : 0; j < it; ++j) {
        (void)mbar_wait_bounded(&full[j % L::kStages], (j / L::kStages) & 1);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = i8_idesc(128, BN);
      uint32_t it = 0, local = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++local) {
        const uint32_t b = local & 1, use_b = local >> 1;
        if (use_b > 0 && !mbar_wait_bounded(&acc_empty[b], (use_b - 1) & 1)) break;
        tc_fence_after();
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = static_cast<int>(it % L::kStages);
          if (!mbar_wait_bounded(&full[s], (it / L::kStages) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_addr(sa + s * L::kABytes);
          const uint32_t b0 = smem_addr(sb + s * L::kBBytes);
#pragma unroll
          for (int k = 0; k < kI8BK / kI8UmmaK; ++k) {
            mma_i8(tmem_base + b * BN, sw128_kmajor_desc(a0 + k * kI8UmmaK),
                   sw128_kmajor_desc(b0 + k * kI8UmmaK), idesc, (kb != 0 || k != 0) ? 1u : 0u);
          }
          mma_commit(&empty[s]);
        }
        if (ok) mma_commit(&acc_full[b]);
      }
      mma_commit(drained);
      (void)mbar_wait_bounded(drained, 0);
    }
  } else {
    const int quarter = warp & 3;
    uint8_t* slot = sslot + (warp - 2) * L::kSlotBytes;
    float2* cols = reinterpret_cast<float2*>(scol + (warp - 2) * L::kColBytes);
    Waits wait;
    uint32_t local = 0;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++local) {
      const uint32_t b = local & 1;
      const int64_t row0 = tile / n_tiles * 128 + quarter * 32;
      const int64_t col0 = tile % n_tiles * BN;
      __syncwarp();  // the previous tile's column scales have been read
      load_cols<BN>(cols, col0, lane, args);
      const float s_row = row_a_scale(args, row0 + lane);
      wait(&acc_full[b], (local >> 1) & 1);
      tc_fence_after();
      drain_i8<TOut, BN>(tmem_base + (uint32_t(quarter * 32) << 16) + b * BN, row0, col0, lane,
                         args, &tma_c, s_row, cols, slot);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[b]);
    }
    if (args.tma_store && lane == 0) tma_store_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(L::kTmemCols));
  }
}

// Two SMs: tiles of 256 x 256 with tcgen05.mma.cta_group::2, half of each operand
// loaded by each CTA, both CTAs' copies counted on the leader's barriers, 8 drain
// warps per CTA (128 columns each).
struct I8PairLayout {
  static constexpr int kStages = 5;
  static constexpr int kEpiWarps = 8;
  static constexpr int kABytes = 128 * kI8BK;
  static constexpr int kBBytes = 128 * kI8BK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kSlotBytes = 32 * 128;
  static constexpr int kColBytes = 128 * 8;
  static constexpr int kBarrierBytes = 256;
  static constexpr size_t kSmem = size_t(kStages) * kStageBytes +
                                  kEpiWarps * (kSlotBytes + kColBytes) + kBarrierBytes + 1024;
  static constexpr uint32_t kTmemCols = 512;
};
constexpr int kI8PairThreads = 64 + 32 * I8PairLayout::kEpiWarps;

template <typename TOut>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kI8PairThreads, 1)
    gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tma_a,
                        const __grid_constant__ CUtensorMap tma_b,
                        const __grid_constant__ CUtensorMap tma_c,
                        const __grid_constant__ I8Args args) {
  using L = I8PairLayout;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* sa = smem;
  uint8_t* sb = sa + L::kStages * L::kABytes;
  uint8_t* sslot = sb + L::kStages * L::kBBytes;
  uint8_t* scol = sslot + L::kEpiWarps * L::kSlotBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(scol + L::kEpiWarps * L::kColBytes);
  uint64_t* empty = full + L::kStages;
  uint64_t* acc_full = empty + L::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drained = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int64_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int64_t n_tiles = (args.N + 255) / 256;
  const int64_t tiles = (args.M + 255) / 256 * n_tiles;
  const int kblocks = static_cast<int>((args.K + kI8BK - 1) / kI8BK);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * L::kEpiWarps);
    }
    mbar_init(drained, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(tmem_slot)),
                 "r"(L::kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int64_t tile = pair; tile < tiles && ok; tile += pairs) {
        const int row = static_cast<int>(tile / n_tiles * 256 + int64_t(rank) * 128);
        const int col = static_cast<int>(tile % n_tiles * 256 + int64_t(rank) * 128);
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = static_cast<int>(it % L::kStages);
          const uint32_t use = it / L::kStages;
          if (use > 0 && !mbar_wait_bounded(&empty[s], (use - 1) & 1)) {
            ok = false;
            break;
          }
          const uint32_t bar = cluster_addr(smem_addr(&full[s]), 0);
          if (leader) mbar_arrive_expect_tx(&full[s], 2 * L::kStageBytes);
          tma_load_2d_pair(sa + s * L::kABytes, &tma_a, kb * kI8BK, row, bar);
          tma_load_2d_pair(sb + s * L::kBBytes, &tma_b, kb * kI8BK, col, bar);
        }
      }
      if (leader) {
        // both CTAs' copies complete on the leader's barriers: nothing is in
        // flight into either CTA after their last phases
        for (uint32_t j = it > L::kStages ? it - L::kStages : 0; j < it; ++j) {
          (void)mbar_wait_bounded(&full[j % L::kStages], (j / L::kStages) & 1);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      const uint32_t idesc = i8_idesc(256, 256);
      uint32_t it = 0, local = 0;
      bool ok = true;
      for (int64_t tile = pair; tile < tiles && ok; tile += pairs, ++local) {
        const uint32_t b = local & 1, use_b = local >> 1;
        if (use_b > 0 && !mbar_wait_bounded(&acc_empty[b], (use_b - 1) & 1)) break;
        tc_fence_after();
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = static_cast<int>(it % L::kStages);
          if (!mbar_wait_bounded(&full[s], (it / L::kStages) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_addr(sa + s * L::kABytes);
          const uint32_t b0 = smem_addr(sb + s * L::kBBytes);
#pragma unroll
          for (int k = 0; k < kI8BK / kI8UmmaK; ++k) {
            mma_i8_pair(tmem_base + b * 256, sw128_kmajor_desc(a0 + k * kI8UmmaK),
                        sw128_kmajor_desc(b0 + k * kI8UmmaK), idesc,
                        (kb != 0 || k != 0) ? 1u : 0u);
          }
          mma_commit_pair_both(&empty[s]);
        }
        if (ok) mma_commit_pair_both(&acc_full[b]);
      }
      mma_commit_pair(cluster_addr(smem_addr(drained), 0));
      (void)mbar_wait_bounded(drained, 0);
    }
  } else {
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    uint8_t* slot = sslot + (warp - 2) * L::kSlotBytes;
    float2* cols = reinterpret_cast<float2*>(scol + (warp - 2) * L::kColBytes);
    Waits wait;
    uint32_t local = 0;
    for (int64_t tile = pair; tile < tiles; tile += pairs, ++local) {
      const uint32_t b = local & 1;
      const int64_t row0 = tile / n_tiles * 256 + int64_t(rank) * 128 + quarter * 32;
      const int64_t col0 = tile % n_tiles * 256 + half * 128;
      __syncwarp();  // the previous tile's column scales have been read
      load_cols<128>(cols, col0, lane, args);
      const float s_row = row_a_scale(args, row0 + lane);
      wait(&acc_full[b], (local >> 1) & 1);
      tc_fence_after();
      drain_i8<TOut, 128>(tmem_base + (uint32_t(quarter * 32) << 16) + b * 256 + half * 128, row0,
                          col0, lane, args, &tma_c, s_row, cols, slot);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(cluster_addr(smem_addr(&acc_empty[b]), 0));
    }
    if (args.tma_store && lane == 0) tma_store_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(L::kTmemCols));
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
bool make_i8_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t k, int64_t ld,
                 int box_rows) {
  auto fn = tma_encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {kI8BK, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estride[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box,
            estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Boxes of 32 rows x 128 bytes of C, or false when its rows do not allow them.
bool make_i8_c_map(CUtensorMap* map, const I8Args& a, int out_dtype) {
  auto fn = tma_encode_fn();
  const int elt = out_dtype == MB_F32 ? 4 : 2;
  if (fn == nullptr || !aligned_to(a.C, 16) || (a.ldc * elt) % 16 != 0) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.N), static_cast<cuuint64_t>(a.M)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.ldc * elt)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / elt), 32};
  cuuint32_t estride[2] = {1, 1};
  const CUtensorMapDataType dt = out_dtype == MB_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : out_dtype == MB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return fn(map, dt, 2, a.C, dims, strides, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int i8_sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n > 0 ? n : 148;
}

template <typename TOut, int BN>
int launch_single(const CUtensorMap& ma, const CUtensorMap& mbm, const CUtensorMap& mc,
                  const I8Args& a, cudaStream_t s) {
  auto kern = gemm_i8_kernel<TOut, BN>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       static_cast<int>(I8Layout<BN>::kSmem));
  const int64_t tiles = ceil_div(a.M, 128) * ceil_div(a.N, BN);
  const int grid = static_cast<int>(imin64(tiles, i8_sm_count()));
  kern<<<grid, kI8Threads, I8Layout<BN>::kSmem, s>>>(ma, mbm, mc, a);
  return 0;
}

// Width of the one-SM tile: the one whose last wave costs least, counting a
// tile's time as its staged bytes per K step (128 + BN rows). Wide tiles re-read
// less, narrow ones spread few rows over every SM.
int choose_bn(int64_t M, int64_t N, int sms) {
  int best = 256;
  int64_t best_cost = INT64_MAX;
  for (int bn = 256; bn >= 32; bn /= 2) {
    const int64_t waves = ceil_div(ceil_div(M, 128) * ceil_div(N, bn), sms);
    const int64_t cost = waves * (128 + bn);
    if (cost < best_cost) {
      best = bn;
      best_cost = cost;
    }
  }
  return best;
}

template <typename TOut>
int launch_gemm_i8(const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb, I8Args a,
                   int out_dtype, cudaStream_t s) {
  CUtensorMap ma, mbm, mc;
  memset(&mc, 0, sizeof(mc));
  const int sms = i8_sm_count();
  const bool pair = a.M >= 256 && a.N >= 256 && ceil_div(a.M, 256) * ceil_div(a.N, 256) >= sms / 2;
  const int bn = pair ? 128 : choose_bn(a.M, a.N, sms);
  // a tile narrower than a staged block's 128 bytes goes row by row
  a.tma_store = bn * int(sizeof(TOut)) >= 128 && make_i8_c_map(&mc, a, out_dtype) ? 1 : 0;
  MB_CHECK_ARG(make_i8_map(&ma, A, a.M, a.K, lda, 128) && make_i8_map(&mbm, B, a.N, a.K, ldb, bn),
               "mb_gemm_i8: cuTensorMapEncodeTiled failed (shape or alignment)");
  if (pair) {
    auto kern = gemm_i8_pair_kernel<TOut>;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(I8PairLayout::kSmem));
    const int64_t tiles = ceil_div(a.M, 256) * ceil_div(a.N, 256);
    const int pairs = static_cast<int>(imin64(tiles, sms / 2));
    kern<<<2 * pairs, kI8PairThreads, I8PairLayout::kSmem, s>>>(ma, mbm, mc, a);
  } else if (bn == 256) {
    launch_single<TOut, 256>(ma, mbm, mc, a, s);
  } else if (bn == 128) {
    launch_single<TOut, 128>(ma, mbm, mc, a, s);
  } else if (bn == 64) {
    launch_single<TOut, 64>(ma, mbm, mc, a, s);
  } else {
    launch_single<TOut, 32>(ma, mbm, mc, a, s);
  }
  MB_CHECK_LAUNCH("mb_gemm_i8");
  return 0;
}

template <typename X, typename TOut>
int launch_rows(const void* x, int64_t ldx, const int8_t* w, int64_t ldw, const I8Args& a,
                cudaStream_t s) {
  // at most three blocks per SM: each stages the input rows once for all its channels
  const unsigned grid = static_cast<unsigned>(
      imin64(ceil_div(a.N, kRowsThreads / 32), int64_t(i8_sm_count()) * 3));
  const size_t smem = static_cast<size_t>(a.M * ((a.K + 15) / 16 * 16));
  const X* xs = static_cast<const X*>(x);
  switch (a.M) {
    case 1: linear_i8_rows_kernel<X, TOut, 1><<<grid, kRowsThreads, smem, s>>>(xs, ldx, w, ldw, a); break;
    case 2: linear_i8_rows_kernel<X, TOut, 2><<<grid, kRowsThreads, smem, s>>>(xs, ldx, w, ldw, a); break;
    case 3: linear_i8_rows_kernel<X, TOut, 3><<<grid, kRowsThreads, smem, s>>>(xs, ldx, w, ldw, a); break;
    default: linear_i8_rows_kernel<X, TOut, 4><<<grid, kRowsThreads, smem, s>>>(xs, ldx, w, ldw, a); break;
  }
  MB_CHECK_LAUNCH("mb_linear_i8_rows");
  return 0;
}

template <typename X>
int launch_rows_out(const void* x, int64_t ldx, const int8_t* w, int64_t ldw, const I8Args& a,
                    int out_dtype, cudaStream_t s) {
  switch (out_dtype) {
    case MB_F32: return launch_rows<X, float>(x, ldx, w, ldw, a, s);
    case MB_BF16: return launch_rows<X, __nv_bfloat16>(x, ldx, w, ldw, a, s);
    default: return launch_rows<X, __half>(x, ldx, w, ldw, a, s);
  }
}

bool float_dtype(int dtype) { return dtype == MB_F32 || dtype == MB_BF16 || dtype == MB_F16; }

// |sum| <= K 128^2 has to stay below 2^31
constexpr int64_t kI8MaxK = (int64_t(1) << 17) - 1;

int check_product(const char* what, int64_t M, int64_t N, int64_t K, const void* a, const void* b,
                  int64_t ldb, const float* b_scale, const void* bias, int bias_dtype,
                  int out_dtype, const void* C, int64_t ldc) {
  MB_CHECK_ARG(M >= 0 && N >= 0, "%s: negative size", what);
  MB_CHECK_ARG(K >= 1 && K <= kI8MaxK, "%s: K must be in [1, %lld] (got %lld)", what,
               static_cast<long long>(kI8MaxK), static_cast<long long>(K));
  MB_CHECK_ARG(M < (int64_t(1) << 31) && N < (int64_t(1) << 31), "%s: M and N must be below 2^31",
               what);
  MB_CHECK_ARG(float_dtype(out_dtype), "%s: unsupported output dtype %d", what, out_dtype);
  if (M == 0 || N == 0) return 0;
  MB_CHECK_ARG(a != nullptr && b != nullptr && b_scale != nullptr && C != nullptr,
               "%s: null tensor", what);
  MB_CHECK_ARG(bias == nullptr || float_dtype(bias_dtype), "%s: unsupported bias dtype %d", what,
               bias_dtype);
  MB_CHECK_ARG(ldb % 16 == 0 && ldb >= K && aligned_to(b, 16),
               "%s: weight rows must start on 16-byte boundaries (pitch %lld)", what,
               static_cast<long long>(ldb));
  MB_CHECK_ARG(ldc >= N, "%s: ldc below N", what);
  return 0;
}

}  // namespace

int gemm_i8_unit_status(bool clear) { return read_device_status(clear); }

cudaError_t gemm_i8_unit_wait_probe(uint32_t polls, cudaStream_t stream) {
  wait_timeout_probe_kernel<<<1, 32, 0, stream>>>(polls);
  return cudaGetLastError();
}

}  // namespace mb

extern "C" int mb_quantize_rows(int dtype, const void* x, int64_t rows, int64_t cols, int64_t ldx,
                                int8_t* q, int64_t ldq, float* scale, void* stream) {
  using namespace mb;
  clear_error();
  MB_CHECK_ARG(rows >= 0 && cols >= 1 && cols < (int64_t(1) << 30),
               "mb_quantize_rows: rows must be >= 0 and cols >= 1 and below 2^30");
  MB_CHECK_ARG(float_dtype(dtype), "mb_quantize_rows: unsupported dtype %d", dtype);
  if (rows == 0) return 0;
  MB_CHECK_ARG(x != nullptr && q != nullptr && scale != nullptr, "mb_quantize_rows: null tensor");
  MB_CHECK_ARG(ldx >= 0 && ldq >= cols, "mb_quantize_rows: bad row pitch");
  cudaStream_t s = as_stream(stream);
  switch (dtype) {
    case MB_F32: return launch_quantize<float>(x, rows, cols, ldx, q, ldq, scale, s);
    case MB_BF16: return launch_quantize<__nv_bfloat16>(x, rows, cols, ldx, q, ldq, scale, s);
    default: return launch_quantize<__half>(x, rows, cols, ldx, q, ldq, scale, s);
  }
}

extern "C" int mb_gemm_i8(const int8_t* a, int64_t lda, const float* a_scale, const int8_t* b,
                          int64_t ldb, const float* b_scale, const void* bias, int bias_dtype,
                          int out_dtype, void* c, int64_t ldc, int64_t M, int64_t N, int64_t K,
                          void* stream) {
  using namespace mb;
  clear_error();
  if (const int rc = check_product("mb_gemm_i8", M, N, K, a, b, ldb, b_scale, bias, bias_dtype,
                                   out_dtype, c, ldc)) {
    return rc;
  }
  if (M == 0 || N == 0) return 0;
  MB_CHECK_ARG(lda % 16 == 0 && lda >= K && aligned_to(a, 16),
               "mb_gemm_i8: input rows must start on 16-byte boundaries (pitch %lld)",
               static_cast<long long>(lda));
  const I8Args args{a_scale, b_scale, bias, bias_dtype, c, ldc, M, N, K, 0};
  cudaStream_t s = as_stream(stream);
  switch (out_dtype) {
    case MB_F32: return launch_gemm_i8<float>(a, lda, b, ldb, args, out_dtype, s);
    case MB_BF16: return launch_gemm_i8<__nv_bfloat16>(a, lda, b, ldb, args, out_dtype, s);
    default: return launch_gemm_i8<__half>(a, lda, b, ldb, args, out_dtype, s);
  }
}

extern "C" int mb_linear_i8_rows_supported(int64_t M, int64_t K) {
  using namespace mb;
  return M >= 1 && M <= kRowsMax && K >= 1 && M * ((K + 15) / 16 * 16) <= kRowsMaxBytes ? 1 : 0;
}

extern "C" int mb_linear_i8_rows(int dtype, const void* x, int64_t ldx, const float* x_scale,
                                 const int8_t* w, int64_t ldw, const float* w_scale,
                                 const void* bias, int bias_dtype, int out_dtype, void* c,
                                 int64_t ldc, int64_t M, int64_t N, int64_t K, void* stream) {
  using namespace mb;
  clear_error();
  if (const int rc = check_product("mb_linear_i8_rows", M, N, K, x, w, ldw, w_scale, bias,
                                   bias_dtype, out_dtype, c, ldc)) {
    return rc;
  }
  if (M == 0 || N == 0) return 0;
  MB_CHECK_ARG(mb_linear_i8_rows_supported(M, K) != 0,
               "mb_linear_i8_rows: at most %d rows and %lld bytes of them", kRowsMax,
               static_cast<long long>(kRowsMaxBytes));
  MB_CHECK_ARG(float_dtype(dtype) || dtype == MB_U8, "mb_linear_i8_rows: unsupported dtype %d",
               dtype);
  MB_CHECK_ARG(ldx >= 0, "mb_linear_i8_rows: negative row pitch");
  const I8Args args{x_scale, w_scale, bias, bias_dtype, c, ldc, M, N, K, 0};
  cudaStream_t s = as_stream(stream);
  switch (dtype) {
    case MB_F32: return launch_rows_out<float>(x, ldx, w, ldw, args, out_dtype, s);
    case MB_BF16: return launch_rows_out<__nv_bfloat16>(x, ldx, w, ldw, args, out_dtype, s);
    case MB_F16: return launch_rows_out<__half>(x, ldx, w, ldw, args, out_dtype, s);
    default: return launch_rows_out<int8_t>(x, ldx, w, ldw, args, out_dtype, s);
  }
}
