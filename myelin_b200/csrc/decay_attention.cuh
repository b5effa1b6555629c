// Shared by the kernels of attention with a decay for each head
// (decay_attention.cu: entry points, recurrent kernels; decay_attention_tc.cu:
// chunked tensor-core kernel).
//
//   forward   S_t = g S_{t-1} + c k_t v_t^T            o_t = a q_t^T S_t
//   reverse   G_t = H_{t+1} + c k_t v_t^T, H_t = g G_t  o_t = a q_t^T G_t
//
// per batch row b and head h, with g = decay[h], a = out_scale, c = kv_scale
// and S_{-1} = H_L = first. Within n steps processed at positions r = 0..n-1
// of the time axis both directions are one formula:
//
//   o_r = a c sum_j g^|r-j| (q_r . k_j) v_j + a W_out[r] q_r^T carry
//   carry' = g^n carry + c sum_r W_kv[r] k_r v_r^T
//
// summed over j <= r with W_out = g^(r+1), W_kv = g^(n-1-r) forward, and over
// j >= r with the two weights exchanged in reverse.
#pragma once

#include "common.cuh"

namespace mb {

constexpr int kAttnMaxHead = 256;

// The split of the time axis: segment s covers [s * len, min(T, (s + 1) * len)).
// With one segment the kernel reads `first` and writes `last` itself. With more,
// a first launch forms every segment's own memory (from zero) in the workspace
// [segments, B, H, Dk, Dv], a scan turns those into each segment's carry-in and
// writes `last`, and a second launch forms the outputs.
struct AttnSplit {
  int segments;
  int64_t len;
  float* states;
};

// Valid steps of batch row b.
__device__ __forceinline__ int64_t attn_row_length(const int32_t* lengths, int64_t b, int64_t T) {
  if (lengths == nullptr) return T;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > T ? T : n);
}

// g^n for n >= 0; exact 1 at n = 0 (also for g = 0, whose log2 is -inf).
__device__ __forceinline__ float decay_pow(float log2g, int64_t n) {
  return n == 0 ? 1.0f : exp2f(static_cast<float>(n) * log2g);
}

// Whether the tensor-core kernels take these arguments, and their launches: `states`
// (memories only; with one segment from `first` to `last`) or the outputs.
bool attn_tc_supported(const mb_decay_attention_args& a);
AttnSplit attn_tc_split(const mb_decay_attention_args& a);
int attn_tc_launch(const mb_decay_attention_args& a, const AttnSplit& split, bool states,
                   cudaStream_t stream);

}  // namespace mb
