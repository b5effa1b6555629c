// Attention with a decay for each head over [T, B, H, D]: entry points, the
// recurrent kernels and the single-step form (formulas: decay_attention.cuh).
#include <math.h>

#include "decay_attention.cuh"

namespace mb {
namespace {

constexpr int kRecThreads = 256;
constexpr int kRecWarps = kRecThreads / 32;

__host__ __device__ constexpr int rec_steps(int rows, int cols) {
  return rows >= 32 || cols > 1 ? 8 : 16;
}

// ---------------------------------------------------------------------------
// Recurrent kernel: any head size up to 256, any element type and stride, sums in
// fp32. A block holds 32 C columns of one memory in registers (C per lane, each warp
// R of the Dk rows), stages TC steps of q, k and v in shared memory as fp32
// (the next ones on their way meanwhile), walks them without a barrier and then adds
// the eight warps' partial outputs.
//
// The leak is taken out of the inner loop: over a burst of steps p = 0 .. P-1 the
// block keeps g^(P-1-p) S_p, so that a step is two FMAs per memory element (in pairs,
// f32x2) instead of a product and two FMAs:
//   S~ += (g^(P-1-p) k_p) v_p^T,   o_p = g^-(P-1-p) q_p^T S~,
// from S~ = g^P S_-1; in reverse from g^(P-1) H, and H = g S~ after it. The
// powers are formed in double, so that g^-i g^i is 1 to two roundings. What is kept is
// never above the memory itself, and bursts are as long as keep g^(P-1) at 2^-15 or
// more (burst_steps): it may round where fp32 ends, which costs the memory 2^-135. About 2 Dk Dv FMAs per step and head bound it, once a lane has
// several columns: a broadcast 16-byte read of k or q fills a warp's registers in four
// cycles whatever it is used for, so that with one column per lane those reads took
// 0.906 ms at T=1024, 256 rows of 128 x 128 heads (19 TFLOP/s).
// ---------------------------------------------------------------------------
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
        "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}

// Steps of a burst: 16 down to g = 2^-1, 8 to 2^(-15/7), 4 to 2^-5, 2 to 2^-15, then 1,
// as also for memories that grow (whose powers would overflow).
template <int TC>
__device__ __forceinline__ int burst_steps(float g) {
  if (!(g <= 1.0f)) return 1;
  const int most = g >= 0.5f ? 16 : g >= 0.2265f ? 8 : g >= 0.03125f ? 4 : g >= 0x1p-15f ? 2 : 1;
  return most < TC ? most : TC;
}

template <typename T, int R, int C, bool STATES_ONLY>
__global__ void __launch_bounds__(kRecThreads)
    attn_recurrent_kernel(const __grid_constant__ mb_decay_attention_args a,
                          const __grid_constant__ AttnSplit split) {
  constexpr int TC = rec_steps(R, C);
  constexpr int kCols = 32 * C;
  constexpr int ROWS = R * kRecWarps;
  constexpr int NK = TC * ROWS / kRecThreads;               // staged k (q) elements per thread
  constexpr int NV = (TC * kCols + kRecThreads - 1) / kRecThreads;
  __shared__ __align__(16) float sk[TC][ROWS];
  __shared__ __align__(16) float sq[STATES_ONLY ? 1 : TC][ROWS];
  __shared__ float sv[TC][kCols];
  __shared__ float part[STATES_ONLY ? 1 : TC][kRecWarps][kCols];
  __shared__ float s_pow[TC + 1], s_inv[TC];  // g^i, g^-i (i < burst)
  __shared__ float s_in[TC], s_out[TC];       // weights of a staged step's key and output

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tiles = (a.Dv + kCols - 1) / kCols;
  int64_t u = blockIdx.x;
  const int64_t tile = u % tiles;
  u /= tiles;
  const int64_t h = u % a.H;
  u /= a.H;
  const int64_t b = u % a.B;
  const int64_t seg = u / a.B;
  const int64_t col0 = tile * kCols;
  const int row0 = warp * R;

  const int64_t L = attn_row_length(a.lengths, b, a.T);
  const int64_t lo = seg * split.len;
  const int64_t hi = imin64(a.T, lo + split.len);
  const int64_t end = imin64(hi, L);  // valid steps of this segment: [lo, end)
  const int64_t n = end > lo ? end - lo : 0;

  const T* q = static_cast<const T*>(a.q.data) + b * a.q.stride_b + h * a.q.stride_h;
  const T* k = static_cast<const T*>(a.k.data) + b * a.k.stride_b + h * a.k.stride_h;
  const T* v = static_cast<const T*>(a.v.data) + b * a.v.stride_b + h * a.v.stride_h;
  T* o = static_cast<T*>(a.o.data) + b * a.o.stride_b + h * a.o.stride_h;
  const float g = a.decay[h];
  const bool reverse = a.reverse != 0;
  const int burst = burst_steps<TC>(g);
  // the weights of a group of `steps` staged steps, by their place from their burst's end
  // (keys past the last step are zeros)
  auto weights = [&](int steps) {
    const int s = threadIdx.x;
    if (s >= steps) return;
    const int p = s & (burst - 1);
    const int left = min(burst, steps - s + p) - 1 - p;
    s_in[s] = s_pow[left];
    s_out[s] = a.out_scale * s_inv[left];
  };
  if (threadIdx.x <= TC) {
    double p = 1.0;
    for (int i = 0; i < int(threadIdx.x); ++i) p *= static_cast<double>(g);
    s_pow[threadIdx.x] = static_cast<float>(p);
    if (threadIdx.x < burst) s_inv[threadIdx.x] = threadIdx.x == 0 ? 1.0f : static_cast<float>(1.0 / p);
  }

  float2 S[C][R / 2];  // columns col0 + lane + 32 c
  const int64_t seg_at = ((seg * a.B + b) * a.H + h) * a.Dk;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int64_t col = col0 + lane + 32 * c;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = row0 + i;
      float x = 0.0f;
      if (col < a.Dv && r < a.Dk && !STATES_ONLY) {
        if (split.segments > 1) {
          x = split.states[(seg_at + r) * a.Dv + col];
        } else if (a.first.data != nullptr) {
          x = a.first.data[b * a.first.stride_b + h * a.first.stride_h + r * a.first.stride_row +
                           col * a.first.stride_col];
        }
      }
      (i & 1 ? S[c][i / 2].y : S[c][i / 2].x) = x;
    }
  }

  // this thread's elements of the next steps' k, q and v
  float rk[NK], rq[STATES_ONLY ? 1 : NK], rv[NV];
  auto step_at = [&](int64_t p) { return reverse ? end - 1 - p : lo + p; };
  auto fetch = [&](int64_t p0) {
    const int steps = static_cast<int>(imin64(TC, n - p0));
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int e = threadIdx.x + i * kRecThreads, s = e / ROWS, d = e % ROWS;
      const bool ok = s < steps && d < a.Dk;
      const int64_t t = step_at(p0 + s);
      rk[i] = ok ? Elem<T>::to_f(k[t * a.k.stride_t + d]) : 0.0f;
      if constexpr (!STATES_ONLY) rq[i] = ok ? Elem<T>::to_f(q[t * a.q.stride_t + d]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = threadIdx.x + i * kRecThreads, s = e / kCols, c = e % kCols;
      rv[i] = s < steps && col0 + c < a.Dv
                  ? Elem<T>::to_f(v[step_at(p0 + s) * a.v.stride_t + col0 + c])
                  : 0.0f;
    }
  };
  auto scale_memory = [&](float w) {
    const float2 w2 = make_float2(w, w), zero = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < R / 2; ++i) S[c][i] = fma_pair(S[c][i], w2, zero);
    }
  };
  if (n > 0) fetch(0);
  __syncthreads();  // the powers are written
  weights(static_cast<int>(imin64(TC, n)));
  const float full = s_pow[burst];
  int untouched = reverse ? 1 : 0;
  for (int64_t p0 = 0; p0 < n; p0 += TC) {
    const int steps = static_cast<int>(imin64(TC, n - p0));
    __syncthreads();  // the previous steps' staging and weights have been read
    if (steps < TC && p0 > 0) {
      weights(steps);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int e = threadIdx.x + i * kRecThreads, s = e / ROWS;
      // (rows past the last step are zeros: any weight)
      sk[s][e % ROWS] = rk[i] * a.kv_scale * s_in[s];
      if constexpr (!STATES_ONLY) sq[s][e % ROWS] = rq[i];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = threadIdx.x + i * kRecThreads;
      if (e < TC * kCols) sv[e / kCols][e % kCols] = rv[i];
    }
    __syncthreads();
    if (p0 + TC < n) fetch(p0 + TC);
    for (int s0 = 0; s0 < steps; s0 += burst) {
      const int s1 = min(steps, s0 + burst);
      // (in reverse the leak of the last burst's last step is still to come, except the first time)
      scale_memory(s1 - s0 == burst && !untouched ? full : s_pow[s1 - s0 - untouched]);
      untouched = 0;
      auto step = [&](int s) {
        float2 vc[C], acc[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const float x = sv[s][lane + 32 * c];
          vc[c] = make_float2(x, x);
          acc[c] = make_float2(0.0f, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < R; i += 4) {
          const float4 kk = *reinterpret_cast<const float4*>(&sk[s][row0 + i]);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            S[c][i / 2] = fma_pair(make_float2(kk.x, kk.y), vc[c], S[c][i / 2]);
            S[c][i / 2 + 1] = fma_pair(make_float2(kk.z, kk.w), vc[c], S[c][i / 2 + 1]);
          }
          if constexpr (!STATES_ONLY) {
            const float4 qq = *reinterpret_cast<const float4*>(&sq[s][row0 + i]);
#pragma unroll
            for (int c = 0; c < C; ++c) {
              acc[c] = fma_pair(make_float2(qq.x, qq.y), S[c][i / 2], acc[c]);
              acc[c] = fma_pair(make_float2(qq.z, qq.w), S[c][i / 2 + 1], acc[c]);
            }
          }
        }
        if constexpr (!STATES_ONLY) {
#pragma unroll
          for (int c = 0; c < C; ++c) part[s][warp][lane + 32 * c] = acc[c].x + acc[c].y;
        }
      };
      if (s1 - s0 == TC) {  // whole bursts unrolled: the steps' loads run ahead of their sums
#pragma unroll
        for (int s = 0; s < TC; ++s) step(s);
      } else {
        for (int s = s0; s < s1; ++s) step(s);
      }
    }
    if constexpr (!STATES_ONLY) {
      __syncthreads();
      for (int e = threadIdx.x; e < steps * kCols; e += kRecThreads) {
        const int s = e / kCols, c = e % kCols;
        if (col0 + c >= a.Dv) continue;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kRecWarps; ++w) sum += part[s][w][c];
        o[step_at(p0 + s) * a.o.stride_t + col0 + c] = Elem<T>::from_f(sum * s_out[s]);
      }
    }
  }

  if (reverse && n > 0) scale_memory(g);

  if constexpr (!STATES_ONLY) {  // steps past the row's length: zeros
    const int64_t z0 = end > lo ? end : lo;
    for (int64_t e = threadIdx.x; e < (hi - z0) * kCols; e += kRecThreads) {
      const int64_t t = z0 + e / kCols, c = col0 + e % kCols;
      if (c < a.Dv) o[t * a.o.stride_t + c] = Elem<T>::zero();
    }
  }
  const bool whole = !STATES_ONLY && split.segments == 1 && a.last.data != nullptr;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int64_t col = col0 + lane + 32 * c;
    if (col >= a.Dv) continue;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = row0 + i;
      const float x = i & 1 ? S[c][i / 2].y : S[c][i / 2].x;
      if (r >= a.Dk) continue;
      if constexpr (STATES_ONLY) {
        split.states[(seg_at + r) * a.Dv + col] = x;
      } else if (whole) {
        a.last.data[b * a.last.stride_b + h * a.last.stride_h + r * a.last.stride_row +
                    col * a.last.stride_col] = x;
      }
    }
  }
}

// Between the two launches of a split time axis: every segment's own memory
// becomes the carry it starts from, in processing order; the last carry is the
// final memory. One thread per memory element; `segments` reads and writes (a
// length past the row's end decays nothing).
__global__ void __launch_bounds__(256)
    attn_segment_scan_kernel(const __grid_constant__ mb_decay_attention_args a,
                             const __grid_constant__ AttnSplit split) {
  const int64_t per_head = a.Dk * a.Dv;
  const int64_t total = a.B * a.H * per_head;
  const int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (e >= total) return;
  const int64_t bh = e / per_head, b = bh / a.H, h = bh % a.H;
  const int64_t r = (e % per_head) / a.Dv, c = e % a.Dv;
  const int64_t L = attn_row_length(a.lengths, b, a.T);
  const float log2g = log2f(a.decay[h]);
  float carry = 0.0f;
  if (a.first.data != nullptr) {
    carry = a.first.data[b * a.first.stride_b + h * a.first.stride_h + r * a.first.stride_row +
                         c * a.first.stride_col];
  }
  constexpr int FLIGHT = 8;  // segments' memories on their way at once
  for (int i0 = 0; i0 < split.segments; i0 += FLIGHT) {
    float own[FLIGHT];
#pragma unroll
    for (int x = 0; x < FLIGHT; ++x) {
      const int s = a.reverse ? split.segments - 1 - i0 - x : i0 + x;
      if (i0 + x < split.segments) own[x] = split.states[s * total + e];
    }
#pragma unroll
    for (int x = 0; x < FLIGHT; ++x) {
      if (i0 + x >= split.segments) break;
      const int s = a.reverse ? split.segments - 1 - i0 - x : i0 + x;
      const int64_t left = L - s * split.len;
      const int64_t n = left < 0 ? 0 : imin64(left, split.len);
      split.states[s * total + e] = carry;
      carry = fmaf(decay_pow(log2g, n), carry, own[x]);
    }
  }
  if (a.last.data != nullptr) {
    a.last.data[b * a.last.stride_b + h * a.last.stride_h + r * a.last.stride_row +
                c * a.last.stride_col] = carry;
  }
}

// ---------------------------------------------------------------------------
// Single step over a batch of memories [B, H, Dk, Dv] (contiguous fp32):
//   S' = g S + k v^T,  o = scale q^T S'
// Bound by the memory's own bytes (read once, written once). A block holds LPR
// lanes x VEC columns of one memory; its rows are dealt to the 256 / LPR row
// groups, 8 rows in flight per thread, and the groups' partial outputs are added
// in a fixed order through shared memory. Rows of `active` that are zero keep
// their memory and give zero outputs.
// ---------------------------------------------------------------------------
template <typename T, int LPR, int VEC>
__global__ void __launch_bounds__(256)
    attn_step_kernel(const __grid_constant__ mb_decay_attention_step_args a) {
  constexpr int GROUPS = 256 / LPR;
  constexpr int TILE = LPR * VEC;
  constexpr int FLIGHT = 8;
  using V = Vec<float, VEC>;
  __shared__ float sk[kAttnMaxHead], sq[kAttnMaxHead];
  __shared__ float part[GROUPS][TILE];
  const int64_t tiles = (a.Dv + TILE - 1) / TILE;
  int64_t u = blockIdx.x;
  const int64_t col0 = (u % tiles) * TILE;
  u /= tiles;
  const int64_t h = u % a.H, b = u / a.H;
  const bool active = a.active == nullptr || a.active[b] != 0;
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride_b + h * a.q_stride_h;
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride_b + h * a.k_stride_h;
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride_b + h * a.v_stride_h;
  T* o = static_cast<T*>(a.o) + (b * a.H + h) * a.Dv;
  const int group = threadIdx.x / LPR, lane = threadIdx.x % LPR;
  const int64_t col = col0 + lane * VEC;
  const bool col_ok = col < a.Dv;
  const float* in = a.memory_in + (b * a.H + h) * a.Dk * a.Dv + col;
  float* out = a.memory_out + (b * a.H + h) * a.Dk * a.Dv + col;

  if (!active) {
    if (col_ok && a.memory_in != a.memory_out) {
      for (int64_t r = group; r < a.Dk; r += GROUPS) {
        store_vec<float, VEC>(out + r * a.Dv, load_vec<float, VEC>(in + r * a.Dv));
      }
    }
    if (group == 0 && col_ok) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[col + e] = Elem<T>::zero();
    }
    return;
  }

  // the first rows of the memory are on their way while k, q and v are read
  V s[FLIGHT];
#pragma unroll
  for (int i = 0; i < FLIGHT; ++i) {
    const int64_t r = group + i * GROUPS;
    if (col_ok && r < a.Dk) s[i] = load_vec<float, VEC>(in + r * a.Dv);
  }
  for (int d = threadIdx.x; d < a.Dk; d += 256) {
    sk[d] = Elem<T>::to_f(k[d]);
    sq[d] = Elem<T>::to_f(q[d]);
  }
  const float g = a.decay[h];
  float vc[VEC], acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    vc[e] = col_ok ? Elem<T>::to_f(v[col + e]) : 0.0f;
    acc[e] = 0.0f;
  }
  __syncthreads();
  for (int64_t r0 = group; r0 < a.Dk; r0 += FLIGHT * GROUPS) {
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
      const int64_t r = r0 + i * GROUPS;
      if (!col_ok || r >= a.Dk) continue;
      const float kr = sk[r], qr = sq[r];
      V next;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        next.v[e] = fmaf(g, s[i].v[e], kr * vc[e]);
        acc[e] = fmaf(qr, next.v[e], acc[e]);
      }
      store_vec<float, VEC>(out + r * a.Dv, next);
      const int64_t ahead = r + FLIGHT * GROUPS;
      if (ahead < a.Dk) s[i] = load_vec<float, VEC>(in + ahead * a.Dv);
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) part[group][lane * VEC + e] = acc[e];
  __syncthreads();
  for (int c = threadIdx.x; c < TILE; c += 256) {
    if (col0 + c >= a.Dv) continue;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < GROUPS; ++w) sum += part[w][c];
    o[col0 + c] = Elem<T>::from_f(sum * a.scale);
  }
}

bool valid_dtype(int dtype) { return dtype == MB_F32 || dtype == MB_BF16 || dtype == MB_F16; }

int check_args(const mb_decay_attention_args* a, const char* what) {
  MB_CHECK_ARG(a != nullptr, "%s: args is null", what);
  MB_CHECK_ARG(valid_dtype(a->dtype), "%s: unsupported dtype %d", what, a->dtype);
  MB_CHECK_ARG(a->T >= 0 && a->B >= 0 && a->H >= 0, "%s: negative size", what);
  MB_CHECK_ARG(a->Dk >= 1 && a->Dk <= kAttnMaxHead && a->Dv >= 1 && a->Dv <= kAttnMaxHead,
               "%s: head sizes must be in [1, %d] (got Dk=%lld, Dv=%lld)", what, kAttnMaxHead,
               static_cast<long long>(a->Dk), static_cast<long long>(a->Dv));
  MB_CHECK_ARG(a->B < (int64_t(1) << 31) && a->H < (int64_t(1) << 31) &&
                   a->T < (int64_t(1) << 31),
               "%s: T, B and H must be below 2^31", what);
  return 0;
}

// Columns per lane: as many as the head has (four only while a warp's rows fit its
// registers), fewer where that leaves less than two blocks per SM.
int recurrent_cols(const mb_decay_attention_args& a) {
  int c = a.Dv > 64 && a.Dk <= 128 ? 4 : a.Dv > 32 ? 2 : 1;
  const int64_t most = a.T >= 1024 ? a.T / 128 : 1;  // segments
  while (c > 1 && a.B * a.H * ceil_div(a.Dv, 32 * c) * most < 2 * 148) c /= 2;
  return c;
}

// Segments of the recurrent kernel: enough blocks for every SM (two resident each)
// when batch x heads x column tiles are few, at least 128 steps apiece. A split costs
// a second pass over k and v and two more launches: below four segments, or 1024
// steps, one pass is as fast.
AttnSplit recurrent_split(const mb_decay_attention_args& a) {
  const int64_t blocks = a.B * a.H * ceil_div(a.Dv, 32 * recurrent_cols(a));
  int64_t segments = blocks > 0 ? (148 * 2) / blocks : 1;
  segments = imin64(segments, a.T / 128);
  if (segments < 4 || a.T < 1024) segments = 1;
  const int64_t len = segments > 1 ? ceil_div(a.T, segments) : a.T;
  segments = segments > 1 ? ceil_div(a.T, len) : 1;
  return AttnSplit{static_cast<int>(segments), len, nullptr};
}

template <typename T, int R, int C>
int launch_recurrent_rc(const mb_decay_attention_args& a, const AttnSplit& split, bool states_only,
                        cudaStream_t stream) {
  const int64_t blocks = split.segments * a.B * a.H * ceil_div(a.Dv, 32 * C);
  MB_CHECK_ARG(blocks <= 0x7fffffff, "mb_decay_attention: too many (batch, head) rows");
  if (states_only) {
    attn_recurrent_kernel<T, R, C, true>
        <<<static_cast<unsigned>(blocks), kRecThreads, 0, stream>>>(a, split);
  } else {
    attn_recurrent_kernel<T, R, C, false>
        <<<static_cast<unsigned>(blocks), kRecThreads, 0, stream>>>(a, split);
  }
  MB_CHECK_LAUNCH("mb_decay_attention");
  return 0;
}

template <typename T, int R>
int launch_recurrent_r(const mb_decay_attention_args& a, const AttnSplit& split, bool states_only,
                       cudaStream_t stream) {
  const int c = recurrent_cols(a);
  if constexpr (R <= 16) {
    if (c == 4) return launch_recurrent_rc<T, R, 4>(a, split, states_only, stream);
  }
  if (c >= 2) return launch_recurrent_rc<T, R, 2>(a, split, states_only, stream);
  return launch_recurrent_rc<T, R, 1>(a, split, states_only, stream);
}

template <typename T>
int launch_recurrent_t(const mb_decay_attention_args& a, const AttnSplit& split, bool states_only,
                       cudaStream_t stream) {
  if (a.Dk <= 32) return launch_recurrent_r<T, 4>(a, split, states_only, stream);
  if (a.Dk <= 64) return launch_recurrent_r<T, 8>(a, split, states_only, stream);
  if (a.Dk <= 128) return launch_recurrent_r<T, 16>(a, split, states_only, stream);
  return launch_recurrent_r<T, 32>(a, split, states_only, stream);
}

int launch_recurrent(const mb_decay_attention_args& a, const AttnSplit& split, bool states_only,
                     cudaStream_t stream) {
  switch (a.dtype) {
    case MB_F32: return launch_recurrent_t<float>(a, split, states_only, stream);
    case MB_BF16: return launch_recurrent_t<__nv_bfloat16>(a, split, states_only, stream);
    default: return launch_recurrent_t<__half>(a, split, states_only, stream);
  }
}

// The tensor-core kernel where its rules allow it, else the recurrent one.
AttnSplit choose_split(const mb_decay_attention_args& a, bool tc) {
  return tc ? attn_tc_split(a) : recurrent_split(a);
}

int launch_pass(const mb_decay_attention_args& a, const AttnSplit& split, bool tc,
                bool states, cudaStream_t stream) {
  return tc ? attn_tc_launch(a, split, states, stream)
            : launch_recurrent(a, split, states, stream);
}

int64_t split_bytes(const mb_decay_attention_args& a, const AttnSplit& split) {
  return split.segments > 1 ? split.segments * a.B * a.H * a.Dk * a.Dv * int64_t(sizeof(float))
                            : 0;
}

template <typename T, int LPR, int VEC>
int launch_step(const mb_decay_attention_step_args& a, cudaStream_t stream) {
  const int64_t blocks = a.B * a.H * ceil_div(a.Dv, LPR * VEC);
  MB_CHECK_ARG(blocks <= 0x7fffffff, "mb_decay_attention_step: too many (batch, head) rows");
  attn_step_kernel<T, LPR, VEC><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
  MB_CHECK_LAUNCH("mb_decay_attention_step");
  return 0;
}

// Columns per block: the widest tile (128 columns, whole 512-byte rows) when
// the blocks fill the SMs twice, else 32 columns so that few memories still
// spread over many SMs. Rows that are not whole 16-byte pieces go one column
// per lane.
template <typename T>
int launch_step_t(const mb_decay_attention_step_args& a, cudaStream_t stream) {
  const bool vec = a.Dv % 4 == 0 && aligned_to(a.memory_in, 16) && aligned_to(a.memory_out, 16);
  if (!vec) return launch_step<T, 32, 1>(a, stream);
  if (a.Dv > 32 && a.B * a.H * ceil_div(a.Dv, 128) >= 2 * 148) {
    return launch_step<T, 32, 4>(a, stream);
  }
  return launch_step<T, 8, 4>(a, stream);
}

}  // namespace
}  // namespace mb

extern "C" int64_t mb_decay_attention_workspace_bytes(const mb_decay_attention_args* args) {
  using namespace mb;
  if (check_args(args, "mb_decay_attention_workspace_bytes") != 0) return -1;
  if (args->B == 0 || args->H == 0) return 0;
  return split_bytes(*args, choose_split(*args, attn_tc_supported(*args)));
}

extern "C" int mb_decay_attention(const mb_decay_attention_args* args, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  using namespace mb;
  clear_error();
  if (const int rc = check_args(args, "mb_decay_attention")) return rc;
  const mb_decay_attention_args& a = *args;
  if (a.B == 0 || a.H == 0) return 0;
  MB_CHECK_ARG(a.decay != nullptr, "mb_decay_attention: decay is null");
  MB_CHECK_ARG(a.T == 0 || (a.q.data != nullptr && a.k.data != nullptr && a.v.data != nullptr &&
                            a.o.data != nullptr),
               "mb_decay_attention: q, k, v and o must not be null");
  MB_CHECK_ARG(a.last.data == nullptr || a.last.data != a.first.data,
               "mb_decay_attention: last must not be the buffer of first");
  if (a.T == 0 && a.last.data == nullptr) return 0;
  const bool tc = attn_tc_supported(a);
  AttnSplit split = choose_split(a, tc);
  const int64_t need = split_bytes(a, split);
  MB_CHECK_ARG(need <= workspace_bytes && (need == 0 || workspace != nullptr),
               "mb_decay_attention: workspace of %lld bytes, %lld needed",
               static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  split.states = static_cast<float*>(workspace);
  cudaStream_t s = as_stream(stream);
  // the tensor-core kernel for outputs keeps no exact memory: the final one comes
  // from the states kernel, which also starts a split time axis
  const bool states = split.segments > 1 || (tc && a.last.data != nullptr);
  if (states) {
    if (const int rc = launch_pass(a, split, tc, true, s)) return rc;
  }
  if (split.segments > 1) {
    const int64_t total = a.B * a.H * a.Dk * a.Dv;
    const int64_t blocks = ceil_div(total, 256);
    MB_CHECK_ARG(blocks <= 0x7fffffff, "mb_decay_attention: too many memory elements");
    attn_segment_scan_kernel<<<static_cast<unsigned>(blocks), 256, 0, s>>>(a, split);
    MB_CHECK_LAUNCH("mb_decay_attention (segment scan)");
  }
  return launch_pass(a, split, tc, false, s);
}

extern "C" int mb_decay_attention_step(const mb_decay_attention_step_args* args, void* stream) {
  using namespace mb;
  clear_error();
  MB_CHECK_ARG(args != nullptr, "mb_decay_attention_step: args is null");
  const mb_decay_attention_step_args& a = *args;
  MB_CHECK_ARG(valid_dtype(a.dtype), "mb_decay_attention_step: unsupported dtype %d", a.dtype);
  MB_CHECK_ARG(a.B >= 0 && a.H >= 0, "mb_decay_attention_step: negative size");
  MB_CHECK_ARG(a.Dk >= 1 && a.Dk <= kAttnMaxHead && a.Dv >= 1 && a.Dv <= kAttnMaxHead,
               "mb_decay_attention_step: head sizes must be in [1, %d] (got Dk=%lld, Dv=%lld)",
               kAttnMaxHead, static_cast<long long>(a.Dk), static_cast<long long>(a.Dv));
  if (a.B == 0 || a.H == 0) return 0;
  MB_CHECK_ARG(a.q != nullptr && a.k != nullptr && a.v != nullptr && a.o != nullptr &&
                   a.decay != nullptr && a.memory_in != nullptr && a.memory_out != nullptr,
               "mb_decay_attention_step: null tensor");
  cudaStream_t s = as_stream(stream);
  switch (a.dtype) {
    case MB_F32: return launch_step_t<float>(a, s);
    case MB_BF16: return launch_step_t<__nv_bfloat16>(a, s);
    default: return launch_step_t<__half>(a, s);
  }
}
