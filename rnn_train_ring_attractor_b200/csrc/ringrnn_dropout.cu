// Dropout whose mask is a function of (seed, stream, row, element) and is never stored.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011): ten rounds of two 32 x 32 ->
// 64-bit products on a counter of four words, each giving four random words, one per element.  Bound by the memory: x (and the
// residual) read, y written.  A counter costs 20 wide products and about as many three-input logic operations for 4 elements,
// which at bf16 is the next bound, not far behind.  Measured, 67 M elements: bf16 71 us (3.8 TB/s, bound by those instructions),
// with a residual 78 (5.2 TB/s), fp32 with a residual 141 (5.7 TB/s).  Rows that are not a multiple of 16 bytes
// shift the mask from lane to lane: bf16 94 us, with a residual 102 (178 and more element by element).
#include <math.h>

#include "element.cuh"
#include "ringrnn_common.cuh"

namespace ringrnn {
namespace {

// the ten rounds' keys: from the host they are constants of the launch, which an instruction takes as they are
struct Keys {
  uint32_t k[10][2];
  __host__ __device__ explicit Keys(unsigned long long seed) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      k[i][0] = (uint32_t)seed + (uint32_t)i * 0x9E3779B9u;
      k[i][1] = (uint32_t)(seed >> 32) + (uint32_t)i * 0xBB67AE85u;
    }
  }
};
__device__ __forceinline__ uint4 philox10(uint4 c, const Keys& key) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ key.k[i][0], (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ key.k[i][1], (uint32_t)a);
  }
  return c;
}

struct DropoutArgs {
  long long n, packs;        // elements of a row; packs of V elements in it (the last may be short where V does not divide n)
  unsigned long long total;  // rows * packs
  long long step_rows, step_packs;  // what the grid's threads add up to, in whole rows and packs of one
  uint32_t threshold;        // kept iff word >= threshold
  bool none;                 // p = 1: nothing is kept
  float scale;
  Keys keys;
  uint32_t stream_id;
  const long long* seed_and_stream;  // DEVICE_SEED: in the place of both
  unsigned long long first_row;
};

// V elements of one row at a time: a whole number of counters.  WHOLE: n is a multiple of V and addresses are aligned, so a pack
// is one vector of each tensor.
template <class E, int V, bool WHOLE, bool RESIDUAL, bool DEVICE_SEED>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutArgs a, const E* x, const E* residual, E* y) {
  typedef Pack<E, V> P;
  const Keys own(DEVICE_SEED ? (unsigned long long)a.seed_and_stream[0] : 0ull);
  const Keys& keys = DEVICE_SEED ? own : a.keys;
  const uint32_t stream_id = DEVICE_SEED ? (uint32_t)a.seed_and_stream[1] : a.stream_id;
  unsigned long long id = blockIdx.x * 256ULL + threadIdx.x;
  const unsigned long long step = gridDim.x * 256ULL;
  long long row = (long long)(id / (unsigned long long)a.packs), pack = (long long)id - row * a.packs;
  for (; id < a.total; id += step) {
    const long long i = row * a.n + pack * V;
    const int here = WHOLE || pack * V + V <= a.n ? V : (int)(a.n - pack * V);
    P v, r;
    if constexpr (WHOLE) {
      v = *reinterpret_cast<const P*>(x + i);
      if (RESIDUAL) r = *reinterpret_cast<const P*>(residual + i);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v.v[e] = e < here ? x[i + e] : down<E>(0.f);
        if (RESIDUAL) r.v[e] = e < here ? residual[i + e] : down<E>(0.f);
      }
    }
    const unsigned long long in_all = a.first_row + (unsigned long long)row;
    uint4 w[V / 4];
#pragma unroll
    for (int g = 0; g < V / 4; ++g)
      w[g] = philox10(make_uint4((uint32_t)(pack * (V / 4) + g), stream_id, (uint32_t)in_all, (uint32_t)(in_all >> 32)), keys);
#pragma unroll
    for (int g = 0; g < V / 4; ++g) {
      const uint32_t word[4] = {w[g].x, w[g].y, w[g].z, w[g].w};
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // selected, not multiplied by zero: an infinity that is dropped is gone
        f[e] = word[e] >= a.threshold && !a.none ? up(v.v[4 * g + e]) * a.scale : 0.f;
        if (RESIDUAL) f[e] += up(r.v[4 * g + e]);
      }
      down2(f[0], f[1], v.v + 4 * g);
      down2(f[2], f[3], v.v + 4 * g + 2);
    }
    if constexpr (WHOLE) {
      *reinterpret_cast<P*>(y + i) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < here) y[i + e] = v.v[e];
    }
    row += a.step_rows;
    pack += a.step_packs;
    if (pack >= a.packs) {
      pack -= a.packs;
      ++row;
    }
  }
}

// Rows that start anywhere: vectors go by the addresses, and counters by the row, d elements further on.  A thread forms the mask
// of its own counters as bits and takes the last d of the lane before it; a warp's first lane only lends, so a warp has 31
// vectors.  a.packs: vectors of a row that starts V - 1 elements behind a boundary, so the last may be empty.  x, residual and y
// are `off` elements behind a boundary, all three.
template <class E, int V, bool RESIDUAL, bool DEVICE_SEED>
__global__ void __launch_bounds__(256) dropout_shifted_kernel(const __grid_constant__ DropoutArgs a, uint32_t off, const E* x, const E* residual, E* y) {
  typedef Pack<E, V> P;
  const Keys own(DEVICE_SEED ? (unsigned long long)a.seed_and_stream[0] : 0ull);
  const Keys& keys = DEVICE_SEED ? own : a.keys;
  const uint32_t stream_id = DEVICE_SEED ? (uint32_t)a.seed_and_stream[1] : a.stream_id;
  const int lane = threadIdx.x & 31;
  unsigned long long at = (blockIdx.x * 8ULL + (threadIdx.x >> 5)) * 31;  // of the warp
  const unsigned long long step = gridDim.x * 8ULL * 31;
  // (counted a row ahead: the very first lane stands before the first row)
  const unsigned long long id = at + a.packs + lane - 1;
  long long row = (long long)(id / (unsigned long long)a.packs) - 1, pack = (long long)(id % (unsigned long long)a.packs);
  for (; at < a.total; at += step) {
    const int d = (int)(((uint32_t)row * (uint32_t)a.n + off) & (V - 1));
    const unsigned long long in_all = a.first_row + (unsigned long long)row;
    uint32_t mask = 0;
#pragma unroll
    for (int g = 0; g < V / 4; ++g) {
      const uint4 w = philox10(make_uint4((uint32_t)(pack * (V / 4) + g), stream_id, (uint32_t)in_all, (uint32_t)(in_all >> 32)), keys);
      mask |= ((w.x >= a.threshold ? 1u : 0u) | (w.y >= a.threshold ? 2u : 0u) | (w.z >= a.threshold ? 4u : 0u) | (w.w >= a.threshold ? 8u : 0u)) << (4 * g);
    }
    if (a.none) mask = 0;
    const uint32_t before = __shfl_up_sync(0xffffffffu, mask, 1);
    const uint32_t keep = mask << d | before >> (V - d);
    const long long col = pack * V - d, i = row * a.n + col;
    if (lane > 0 && row >= 0 && at + lane - 1 < a.total && col < a.n) {
      const int first = col < 0 ? d : 0, end = col + V <= a.n ? V : (int)(a.n - col);
      const bool whole = first == 0 && end == V;
      P v, r;
      if (whole) {
        v = *reinterpret_cast<const P*>(x + i);
        if (RESIDUAL) r = *reinterpret_cast<const P*>(residual + i);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const bool in = e >= first && e < end;
          v.v[e] = in ? x[i + e] : down<E>(0.f);
          if (RESIDUAL) r.v[e] = in ? residual[i + e] : down<E>(0.f);
        }
      }
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        float f[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f[k] = keep >> (e + k) & 1 ? up(v.v[e + k]) * a.scale : 0.f;
          if (RESIDUAL) f[k] += up(r.v[e + k]);
        }
        down2(f[0], f[1], v.v + e);
      }
      if (whole) {
        *reinterpret_cast<P*>(y + i) = v;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e >= first && e < end) y[i + e] = v.v[e];
      }
    }
    row += a.step_rows;
    pack += a.step_packs;
    if (pack >= a.packs) {
      pack -= a.packs;
      ++row;
    }
  }
}

template <class E, bool RESIDUAL, bool DEVICE_SEED>
int launch(DropoutArgs a, long long rows, const void* x, const void* residual, void* y, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y);
  const bool whole = a.n % V == 0 && at % 16 == 0;
  const uintptr_t off = reinterpret_cast<uintptr_t>(x) % 16;
  if (!whole && off % sizeof(E) == 0 && reinterpret_cast<uintptr_t>(y) % 16 == off && (!RESIDUAL || reinterpret_cast<uintptr_t>(residual) % 16 == off)) {
    a.packs = (a.n + 2 * V - 2) / V;
    a.total = (unsigned long long)rows * (unsigned long long)a.packs;
    const unsigned long long need = (a.total + 31 * 8 - 1) / (31 * 8);
    const unsigned blocks = (unsigned)(need < 148 * 16 ? need : 148 * 16);
    a.step_rows = (long long)blocks * 8 * 31 / a.packs;
    a.step_packs = (long long)blocks * 8 * 31 % a.packs;
    LaunchScope ls(K_LAYER, s);
    dropout_shifted_kernel<E, V, RESIDUAL, DEVICE_SEED><<<blocks, 256, 0, s>>>(a, (uint32_t)(off / sizeof(E)), static_cast<const E*>(x),
                                                                               static_cast<const E*>(residual), static_cast<E*>(y));
    RINGRNN_CUDA_TRY(cudaGetLastError());
    return RINGRNN_OK;
  }
  a.packs = (a.n + V - 1) / V;
  a.total = (unsigned long long)rows * (unsigned long long)a.packs;
  const unsigned long long need = (a.total + 255) / 256;
  const unsigned blocks = (unsigned)(need < 148 * 16 ? need : 148 * 16);
  a.step_rows = (long long)blocks * 256 / a.packs;
  a.step_packs = (long long)blocks * 256 % a.packs;
  LaunchScope ls(K_LAYER, s);
  const E *px = static_cast<const E*>(x), *pr = static_cast<const E*>(residual);
  if (whole) dropout_kernel<E, V, true, RESIDUAL, DEVICE_SEED><<<blocks, 256, 0, s>>>(a, px, pr, static_cast<E*>(y));
  else dropout_kernel<E, V, false, RESIDUAL, DEVICE_SEED><<<blocks, 256, 0, s>>>(a, px, pr, static_cast<E*>(y));
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}
template <class E>
int launch(const DropoutArgs& a, long long rows, const void* x, const void* residual, void* y, cudaStream_t s) {
  const bool device_seed = a.seed_and_stream != nullptr;
  return residual != nullptr ? (device_seed ? launch<E, true, true>(a, rows, x, residual, y, s) : launch<E, true, false>(a, rows, x, residual, y, s))
                             : (device_seed ? launch<E, false, true>(a, rows, x, residual, y, s) : launch<E, false, false>(a, rows, x, residual, y, s));
}

}  // namespace
}  // namespace ringrnn

extern "C" int ringrnn_dropout(int dtype, long long rows, long long n, const void* x, const void* residual, void* y, double p,
                               unsigned long long seed, unsigned long long stream_id, const long long* seed_and_stream,
                               unsigned long long first_row, void* stream) {
  using namespace ringrnn;
  if (rows <= 0 || n <= 0 || n > (1LL << 34) || rows > (1LL << 46) / n) return RINGRNN_ERR_SHAPE;
  if (!x || !y || !(p >= 0.0 && p <= 1.0) || (seed_and_stream == nullptr && stream_id > 0xFFFFFFFFull)) return RINGRNN_ERR_ARG;
  const unsigned long long threshold = (unsigned long long)rint(p * 4294967296.0);  // halves to even
  const bool none = threshold > 0xFFFFFFFFull;
  DropoutArgs a{n, 0, 0, 0, 0, (uint32_t)(none ? 0 : threshold), none, p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f, Keys(seed),
                (uint32_t)stream_id, seed_and_stream, first_row};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case RINGRNN_F32: return launch<float>(a, rows, x, residual, y, s);
    case RINGRNN_BF16: return launch<__nv_bfloat16>(a, rows, x, residual, y, s);
    case RINGRNN_F16: return launch<__half>(a, rows, x, residual, y, s);
    default: return RINGRNN_ERR_ARG;
  }
}
