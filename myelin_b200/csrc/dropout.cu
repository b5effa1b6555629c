// Dropout whose mask comes from a counter-based generator and is never stored.
//
//   y[e] = x[e] * 65536 / (65536 - threshold)   if draw(e) >= threshold, else 0
//
// draw(e) is 16 bits of Philox 4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011) with key = seed and counter =
// (e / 8, offset): each call of the generator gives eight elements their bits
// (element e % 8 takes half e % 2 of word (e % 8) / 2). The backward is the same
// call on the gradient. With a mask shared over time, e counts within one step.
#include "common.cuh"

namespace mb {
namespace {

constexpr int kGroup = 8;  // elements per call of the generator
constexpr int kThreads = 256;

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t index, uint64_t offset, uint64_t seed) {
  uint32_t c0 = static_cast<uint32_t>(index), c1 = static_cast<uint32_t>(index >> 32);
  uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = uint64_t(c0) * 0xD2511F53u, b = uint64_t(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

// Bit j set: element j of the group is kept.
__device__ __forceinline__ uint32_t keep_bits(const Words& r, uint32_t threshold) {
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < kGroup; ++j) {
    const uint32_t draw = (j & 1) ? r.w[j / 2] >> 16 : r.w[j / 2] & 0xffffu;
    bits |= (draw >= threshold ? 1u : 0u) << j;
  }
  return bits;
}

// A select, not a product: a dropped infinity or NaN becomes 0.
template <typename T>
__device__ __forceinline__ T drop(T x, bool keep, float scale) {
  return keep ? Elem<T>::from_f(Elem<T>::to_f(x) * scale) : Elem<T>::zero();
}

// One thread owns group `g` of a step's n elements and walks the rows [row0, row1)
// that share its mask (one row, of all elements, without sharing). VECTOR: rows
// are whole groups at aligned addresses. Four rows of loads are in flight.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T* __restrict__ x, T* __restrict__ y, int64_t rows, int64_t n,
                   int64_t rows_per_block, uint32_t threshold, float scale,
                   const int64_t* __restrict__ seed) {
  using V = Vec<T, kGroup>;
  const int64_t groups = (n + kGroup - 1) / kGroup;
  const int64_t g = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (g >= groups) return;
  const int64_t row0 = int64_t(blockIdx.y) * rows_per_block;
  const int64_t row1 = imin64(rows, row0 + rows_per_block);
  const uint32_t bits =
      keep_bits(philox(static_cast<uint64_t>(g), static_cast<uint64_t>(seed[1]),
                       static_cast<uint64_t>(seed[0])),
                threshold);
  const int64_t e0 = g * kGroup;
  if constexpr (VECTOR) {
    constexpr int FLIGHT = 4;
    for (int64_t r = row0; r < row1; r += FLIGHT) {
      V v[FLIGHT];
#pragma unroll
      for (int i = 0; i < FLIGHT; ++i) {
        if (r + i < row1) v[i] = load_vec<T, kGroup>(x + (r + i) * n + e0);
      }
#pragma unroll
      for (int i = 0; i < FLIGHT; ++i) {
        if (r + i >= row1) break;
#pragma unroll
        for (int j = 0; j < kGroup; ++j) v[i].v[j] = drop(v[i].v[j], (bits >> j) & 1u, scale);
        store_vec<T, kGroup>(y + (r + i) * n + e0, v[i]);
      }
    }
  } else {
    const int valid = static_cast<int>(imin64(kGroup, n - e0));
    for (int64_t r = row0; r < row1; ++r) {
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        const int64_t e = r * n + e0 + j;
        if (j < valid) y[e] = drop(x[e], (bits >> j) & 1u, scale);
      }
    }
  }
}

template <typename T>
int launch(const void* x, void* y, int64_t rows, int64_t n, uint32_t threshold, float scale,
           const int64_t* seed, cudaStream_t stream) {
  const int64_t groups = ceil_div(n, kGroup);
  const int64_t bx = ceil_div(groups, kThreads);
  MB_CHECK_ARG(bx <= 0x7fffffff, "mb_dropout: too many elements");
  // rows that share a mask: as many per thread as still leave four blocks per SM
  // slot of eight (the generator then runs once for all of them)
  int64_t by = rows;
  const int64_t want = ceil_div(int64_t(148) * 32, bx);
  if (by > want) by = want;
  if (by > 65535) by = 65535;
  const int64_t per = ceil_div(rows, by);
  by = ceil_div(rows, per);
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by));
  const bool vector = n % kGroup == 0 && aligned_to(x, 16) && aligned_to(y, 16);
  const T* xs = static_cast<const T*>(x);
  T* ys = static_cast<T*>(y);
  if (vector) {
    dropout_kernel<T, true><<<grid, kThreads, 0, stream>>>(xs, ys, rows, n, per, threshold, scale,
                                                           seed);
  } else {
    dropout_kernel<T, false><<<grid, kThreads, 0, stream>>>(xs, ys, rows, n, per, threshold,
                                                            scale, seed);
  }
  MB_CHECK_LAUNCH("mb_dropout");
  return 0;
}

}  // namespace
}  // namespace mb

extern "C" int mb_dropout(int dtype, const void* x, void* y, int64_t rows, int64_t n,
                          int threshold, const int64_t* seed, void* stream) {
  using namespace mb;
  clear_error();
  MB_CHECK_ARG(rows >= 0 && n >= 0, "mb_dropout: negative size");
  MB_CHECK_ARG(threshold >= 0 && threshold <= 65536, "mb_dropout: threshold %d outside [0, 65536]",
               threshold);
  MB_CHECK_ARG(dtype == MB_F32 || dtype == MB_BF16 || dtype == MB_F16,
               "mb_dropout: unsupported dtype %d", dtype);
  if (rows == 0 || n == 0) return 0;
  MB_CHECK_ARG(x != nullptr && y != nullptr && seed != nullptr, "mb_dropout: null tensor");
  // everything is dropped at 65536: the scale is then not used
  const float scale = threshold < 65536 ? 65536.0f / static_cast<float>(65536 - threshold) : 0.0f;
  const uint32_t t = static_cast<uint32_t>(threshold);
  cudaStream_t s = as_stream(stream);
  switch (dtype) {
    case MB_F32: return launch<float>(x, y, rows, n, t, scale, seed, s);
    case MB_BF16: return launch<__nv_bfloat16>(x, y, rows, n, t, scale, seed, s);
    default: return launch<__half>(x, y, rows, n, t, scale, seed, s);
  }
}
