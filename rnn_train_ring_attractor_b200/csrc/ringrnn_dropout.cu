// Dropout whose mask is a function of (seed, stream, row, element) and is never stored.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011): ten rounds of two 32 x 32 ->
// 64-bit products on a counter of four words, each giving four random words, one per element.  Bound by the memory: x (and the
// residual) read, y written.  A counter costs 20 wide products and about as many three-input logic operations for 4 elements,
// which at bf16 is the next bound, not far behind: see the launch.
#include <math.h>

#include "element.cuh"
#include "ringrnn_common.cuh"

namespace ringrnn {
namespace {

__device__ __forceinline__ uint4 philox10(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k1, (uint32_t)a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

struct DropoutArgs {
  long long n, packs;        // elements of a row; packs of V elements in it (the last may be short where V does not divide n)
  unsigned long long total;  // rows * packs
  unsigned long long threshold;  // kept iff word >= threshold; 2^32 keeps nothing
  float scale;
  unsigned long long seed, stream_id;
  const long long* seed_and_stream;
  unsigned long long first_row;
};

// V elements of one row at a time: a whole number of counters.  WHOLE: n is a multiple of V and addresses are aligned, so a pack
// is one vector of each tensor.
template <class E, int V, bool WHOLE>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs a, const E* x, const E* residual, E* y) {
  typedef Pack<E, V> P;
  unsigned long long seed = a.seed, stream_id = a.stream_id;
  if (a.seed_and_stream != nullptr) {
    seed = (unsigned long long)a.seed_and_stream[0];
    stream_id = (unsigned long long)a.seed_and_stream[1];
  }
  const unsigned long long step = gridDim.x * 256ULL;
  for (unsigned long long id = blockIdx.x * 256ULL + threadIdx.x; id < a.total; id += step) {
    // (32-bit division where it can be: half the instructions of a counter otherwise)
    const unsigned long long row = (a.total >> 32) == 0 ? (unsigned)id / (unsigned)a.packs : id / (unsigned long long)a.packs;
    const unsigned long long pack = id - row * a.packs;
    const long long i = (long long)(row * a.n + pack * V);
    const int here = WHOLE || (long long)pack * V + V <= a.n ? V : (int)(a.n - (long long)pack * V);
    P v, r;
    if constexpr (WHOLE) {
      v = *reinterpret_cast<const P*>(x + i);
      if (residual != nullptr) r = *reinterpret_cast<const P*>(residual + i);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v.v[e] = e < here ? x[i + e] : down<E>(0.f);
        r.v[e] = residual != nullptr && e < here ? residual[i + e] : down<E>(0.f);
      }
    }
    const unsigned long long in_all = a.first_row + row;
#pragma unroll
    for (int g = 0; g < V / 4; ++g) {
      const uint4 w = philox10(make_uint4((uint32_t)(pack * (V / 4) + g), (uint32_t)stream_id, (uint32_t)in_all, (uint32_t)(in_all >> 32)),
                               (uint32_t)seed, (uint32_t)(seed >> 32));
      const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // selected, not multiplied by zero: an infinity that is dropped is gone
        float f = word[e] >= a.threshold ? up(v.v[4 * g + e]) * a.scale : 0.f;
        if (residual != nullptr) f += up(r.v[4 * g + e]);
        v.v[4 * g + e] = down<E>(f);
      }
    }
    if constexpr (WHOLE) {
      *reinterpret_cast<P*>(y + i) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < here) y[i + e] = v.v[e];
    }
  }
}

template <class E>
int launch(DropoutArgs a, long long rows, const void* x, const void* residual, void* y, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y);
  const bool whole = a.n % V == 0 && at % 16 == 0;
  a.packs = (a.n + V - 1) / V;
  a.total = (unsigned long long)rows * (unsigned long long)a.packs;
  const unsigned long long need = (a.total + 255) / 256;
  const unsigned blocks = (unsigned)(need < 148 * 32 ? need : 148 * 32);
  LaunchScope ls(K_LAYER, s);
  if (whole) dropout_kernel<E, V, true><<<blocks, 256, 0, s>>>(a, static_cast<const E*>(x), static_cast<const E*>(residual), static_cast<E*>(y));
  else dropout_kernel<E, V, false><<<blocks, 256, 0, s>>>(a, static_cast<const E*>(x), static_cast<const E*>(residual), static_cast<E*>(y));
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}

}  // namespace
}  // namespace ringrnn

extern "C" int ringrnn_dropout(int dtype, long long rows, long long n, const void* x, const void* residual, void* y, double p,
                               unsigned long long seed, unsigned long long stream_id, const long long* seed_and_stream,
                               unsigned long long first_row, void* stream) {
  using namespace ringrnn;
  if (rows <= 0 || n <= 0 || n > (1LL << 34) || rows > (1LL << 46) / n) return RINGRNN_ERR_SHAPE;
  if (!x || !y || !(p >= 0.0 && p <= 1.0) || (seed_and_stream == nullptr && stream_id > 0xFFFFFFFFull)) return RINGRNN_ERR_ARG;
  DropoutArgs a;
  a.n = n;
  a.packs = 0;
  a.total = 0;
  a.threshold = (unsigned long long)rint(p * 4294967296.0);  // halves to even
  a.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
  a.seed = seed;
  a.stream_id = stream_id;
  a.seed_and_stream = seed_and_stream;
  a.first_row = first_row;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case RINGRNN_F32: return launch<float>(a, rows, x, residual, y, s);
    case RINGRNN_BF16: return launch<__nv_bfloat16>(a, rows, x, residual, y, s);
    case RINGRNN_F16: return launch<__half>(a, rows, x, residual, y, s);
    default: return RINGRNN_ERR_ARG;
  }
}
