// Linear attention with decay: what its kernels share.
//
// One operator does all the work.  For sequences of q, k (width I, "inner") and v (width O, "outer")
//   out_t = sum_{s <= t} pair_scale * g^(t-s) (q_t.k_s) v_s  +  row_scale * g^(t+1) S^T q_t        S: the state before token 0
//   S_end = g^n S + sum_s key_scale * g^(n-1-s) k_s v_s^T
// is the forward with (q, k, v), and, with the roles of the tensors exchanged, each part of the backward.  With dO the gradient
// of the outputs, E_t the gradient of S_t and "reverse" the same sums from the last token to the first (below: what changes):
//   dQ = forward (dO, V, K), state S transposed;   dK = reverse (V, dO, Q), state E transposed;   dV = reverse (K, Q, dO), state E
// In reverse the state entering from behind is dS_last, and what leaves in front is dS_0 = g E_0, so a row's factor is
// g^(n-1-t) and a key's g^(s+1): E_t = scale q_t dO_t^T + g E_{t+1}.  Hence three "jobs" of one kernel make a backward, in one
// launch if the widths agree, and nothing has to be kept from the forward.
//
// A long sequence of few heads is cut into segments.  Their own sums (states from zero) are formed first, a scan over segments
// turns them into the state each one starts from, and then all run at once.
#pragma once

#include "ringrnn_common.cuh"

namespace ringrnn {

struct LaOperand {
  const void* p;
  long long sb, st, sh;  // strides between sequences, tokens and heads, in elements
};

struct LaJob {
  LaOperand q, k, v;
  void* out;          // [B, T, H, outer] contiguous
  int inner, outer;   // widths I and O
  int reverse;
  float pair_scale, row_scale, key_scale;
  // states: matrices of inner x outer elements; element (i, o) at i * s_in + o * s_out of matrix (b * H + h) * segments + segment
  const float* init;  // nullptr: zero
  float* fin;         // nullptr: not wanted
  int s_in, s_out;
  int precise;  // the state keeps 24 bits of what is added, for somebody sees it (tensor cores; sums always do)
};

constexpr int LA_MAX_JOBS = 3;
struct LaLaunch {
  int B, T, H;
  int segments, segment_tokens;  // segment_tokens * segments >= T; a multiple of the kernel's chunk unless segments == 1
  int jobs;
  const float* log_decay;
  const int* lengths;
  LaJob job[LA_MAX_JOBS];
};

// g^n for whole n >= 0 in fp32, to a few units in the last place also where n log2 g is in the tens: the product is formed in
// two parts.  A decay of zero (log -infinity) gives 0^0 = 1 and zero beyond.
struct LaDecay {
  float hi, lo;
  __device__ __forceinline__ explicit LaDecay(float log_decay) {
    hi = log_decay * 1.44269502f;
    lo = fmaf(log_decay, 1.44269502f, -hi) + log_decay * 1.92596299e-8f;
    if (hi < -1e30f) hi = -1e30f, lo = 0.f;
  }
  __device__ __forceinline__ float power(int n) const {
    const float x = (float)n, a = hi * x;
    return exp2f(a) * fmaf(fmaf(hi, x, -a) + lo * x, 0.693147182f, 1.f);
  }
};

// g^n as the sum of two floats, for the factor a state is multiplied by chunk after chunk: one float's rounding, the same every
// time, would add up over the chunks a long memory spans (1e-6 after 64 chunks of a memory of 4096 steps).
struct LaFactor {
  float hi, lo;
  __device__ __forceinline__ LaFactor(float log_decay, int n) {
    const double x = n == 0 ? 1.0 : exp((double)log_decay * n);
    hi = (float)x;
    lo = (float)(x - (double)hi);
  }
  __device__ __forceinline__ float times(float state, float add) const { return fmaf(hi, state, fmaf(lo, state, add)); }
};

__device__ __forceinline__ int la_length(const LaLaunch& L, int b) {
  if (L.lengths == nullptr) return L.T;
  const int n = L.lengths[b];
  return n < 0 ? 0 : n > L.T ? L.T : n;
}

// Tensor-core path (tc_linear.cu): bf16 and fp16, widths up to 128.  Operands need 16-byte aligned bases and strides.
bool la_tc_operand_ok(const LaOperand& o, int B, int T, int H);
int la_tc_launch(const LaLaunch& L, int dtype, bool states_only, cudaStream_t s);
constexpr int LA_TC_CHUNK = 128, LA_TC_WIDTH = 128, LA_TC_BLOCKS = 148;  // blocks: what runs at once

}  // namespace ringrnn
