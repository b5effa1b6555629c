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

// Whether element j of the group is kept; `cut` = threshold << 16. The upper half of
// a word is compared where it is (what lies below cannot change the result).
__device__ __forceinline__ bool kept(const Words& r, int j, uint32_t cut) {
  return ((j & 1) ? r.w[j / 2] : r.w[j / 2] << 16) >= cut;
}

// A select, not a product: a dropped infinity or NaN becomes 0.
template <typename T>
__device__ __forceinline__ T drop(T x, bool keep, float scale) {
  return Elem<T>::from_f(keep ? Elem<T>::to_f(x) * scale : 0.0f);
}

// A group's elements as pieces of BYTES bytes, each of which has to start on a multiple
// of that: 16 (two pieces of fp32), or 32 for fp32 groups in one access.
template <typename T, int BYTES>
struct Group {
  static constexpr int kPiece = BYTES / sizeof(T);
  Vec<T, kPiece> piece[kGroup / kPiece];
  __device__ __forceinline__ T& operator[](int j) { return piece[j / kPiece].v[j % kPiece]; }
};

template <typename T, int BYTES>
__device__ __forceinline__ Group<T, BYTES> load_group(const T* p) {
  constexpr int E = Group<T, BYTES>::kPiece;
  Group<T, BYTES> g;
#pragma unroll
  for (int i = 0; i < kGroup / E; ++i) g.piece[i] = load_vec<T, E>(p + i * E);
  return g;
}

template <typename T, int BYTES>
__device__ __forceinline__ void store_group(T* p, const Group<T, BYTES>& g) {
  constexpr int E = Group<T, BYTES>::kPiece;
#pragma unroll
  for (int i = 0; i < kGroup / E; ++i) store_vec<T, E>(p + i * E, g.piece[i]);
}

// Every element its own draw: kFlight groups per thread, a block's width apart, all
// loads on their way before the generator runs. Bound by DRAM (4 bytes per 16-bit
// element); the generator and the selects are about 110 issue slots per group, half
// of what the copy bandwidth leaves. One group per thread, with the draws first made
// into a bit mask, took 0.262 ms for 134 M bf16 elements. fp32 in 32-byte accesses where
// both bases allow them (4 M elements in L2: 6.2 us, 8.3 in 16-byte ones; 67 M: 82 and 84).
constexpr int kFlight = 4;

template <typename T, int BYTES>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T* __restrict__ x, T* __restrict__ y, int64_t n, uint32_t cut, float scale,
                   const int64_t* __restrict__ seed) {
  const int64_t groups = n / kGroup;
  const int64_t g0 = int64_t(blockIdx.x) * (kThreads * kFlight) + threadIdx.x;
  Group<T, BYTES> v[kFlight];
#pragma unroll
  for (int i = 0; i < kFlight; ++i) {
    const int64_t g = g0 + i * kThreads;
    if (g < groups) v[i] = load_group<T, BYTES>(x + g * kGroup);
  }
  const uint64_t key = static_cast<uint64_t>(seed[0]), offset = static_cast<uint64_t>(seed[1]);
#pragma unroll
  for (int i = 0; i < kFlight; ++i) {
    const int64_t g = g0 + i * kThreads;
    if (g >= groups) return;
    const Words r = philox(static_cast<uint64_t>(g), offset, key);
#pragma unroll
    for (int j = 0; j < kGroup; ++j) v[i][j] = drop(v[i][j], kept(r, j, cut), scale);
    store_group<T, BYTES>(y + g * kGroup, v[i]);
  }
}

// One mask for `rows` rows, and any alignment: a thread owns one group of the n
// elements and walks the rows [row0, row1), four in flight. fp32 in 16-byte accesses
// whatever the alignment (256 rows of 262144: 86 us, 103 in 32-byte ones).
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kThreads)
    dropout_rows_kernel(const T* __restrict__ x, T* __restrict__ y, int64_t rows, int64_t n,
                        int64_t rows_per_block, uint32_t cut, float scale,
                        const int64_t* __restrict__ seed) {
  const int64_t groups = (n + kGroup - 1) / kGroup;
  const int64_t g = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (g >= groups) return;
  const int64_t row0 = int64_t(blockIdx.y) * rows_per_block;
  const int64_t row1 = imin64(rows, row0 + rows_per_block);
  const int64_t e0 = g * kGroup;
  const uint64_t key = static_cast<uint64_t>(seed[0]), offset = static_cast<uint64_t>(seed[1]);
  if constexpr (VECTOR) {
    Group<T, 16> v[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      if (row0 + i < row1) v[i] = load_group<T, 16>(x + (row0 + i) * n + e0);
    }
    const Words r = philox(static_cast<uint64_t>(g), offset, key);
    bool keep[kGroup];
#pragma unroll
    for (int j = 0; j < kGroup; ++j) keep[j] = kept(r, j, cut);
    for (int64_t row = row0; row < row1; row += kFlight) {
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        if (row + i >= row1) break;
        Group<T, 16> out;
#pragma unroll
        for (int j = 0; j < kGroup; ++j) out[j] = drop(v[i][j], keep[j], scale);
        if (row + i + kFlight < row1) v[i] = load_group<T, 16>(x + (row + i + kFlight) * n + e0);
        store_group<T, 16>(y + (row + i) * n + e0, out);
      }
    }
  } else {
    const Words r = philox(static_cast<uint64_t>(g), offset, key);
    const int valid = static_cast<int>(imin64(kGroup, n - e0));
    for (int64_t row = row0; row < row1; ++row) {
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        const int64_t e = row * n + e0 + j;
        if (j < valid) y[e] = drop(x[e], kept(r, j, cut), scale);
      }
    }
  }
}

template <typename T>
int launch(const void* x, void* y, int64_t rows, int64_t n, int threshold, const int64_t* seed,
           cudaStream_t stream) {
  const T* xs = static_cast<const T*>(x);
  T* ys = static_cast<T*>(y);
  const float scale = 65536.0f / static_cast<float>(65536 - threshold);
  const uint32_t cut = static_cast<uint32_t>(threshold) << 16;
  static_assert(alignof(Group<T, 16>) == 16 && alignof(Group<float, 32>) == 32, "accesses");
  const bool vector = n % kGroup == 0 && aligned_to(x, 16) && aligned_to(y, 16);
  const bool wide = sizeof(T) == 4 && aligned_to(x, 32) && aligned_to(y, 32);
  const int64_t groups = ceil_div(n, kGroup);
  if (rows == 1 && vector) {
    const int64_t blocks = ceil_div(groups, kThreads * kFlight);
    MB_CHECK_ARG(blocks <= 0x7fffffff, "mb_dropout: too many elements");
    auto kern = wide ? dropout_kernel<T, 8 * sizeof(T)> : dropout_kernel<T, 16>;
    kern<<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(xs, ys, n, cut, scale, seed);
  } else {
    const int64_t bx = ceil_div(groups, kThreads);
    MB_CHECK_ARG(bx <= 0x7fffffff, "mb_dropout: too many elements");
    // rows that share a mask: as many per thread as still leave eight blocks per SM
    // (the generator runs once for all of a thread's rows)
    int64_t by = imin64(rows, ceil_div(int64_t(148) * 8, bx));
    if (by > 65535) by = 65535;
    const int64_t per = ceil_div(rows, by);
    by = ceil_div(rows, per);
    const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by));
    if (vector) {
      dropout_rows_kernel<T, true><<<grid, kThreads, 0, stream>>>(xs, ys, rows, n, per, cut, scale,
                                                                  seed);
    } else {
      dropout_rows_kernel<T, false><<<grid, kThreads, 0, stream>>>(xs, ys, rows, n, per, cut,
                                                                   scale, seed);
    }
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
  cudaStream_t s = as_stream(stream);
  if (threshold == 65536) {  // everything is dropped
    const int64_t bytes = rows * n * (dtype == MB_F32 ? 4 : 2);
    const cudaError_t err = cudaMemsetAsync(y, 0, static_cast<size_t>(bytes), s);
    if (err != cudaSuccess) {
      set_error("mb_dropout: cudaMemsetAsync failed: %s", cudaGetErrorString(err));
      return 2;
    }
    return 0;
  }
  switch (dtype) {
    case MB_F32: return launch<float>(x, y, rows, n, threshold, seed, s);
    case MB_BF16: return launch<__nv_bfloat16>(x, y, rows, n, threshold, seed, s);
    default: return launch<__half>(x, y, rows, n, threshold, seed, s);
  }
}
