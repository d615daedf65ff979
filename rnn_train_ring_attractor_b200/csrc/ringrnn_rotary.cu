// Rotary positions: pairs of a head's elements turned by position * frequency.
//
// Bound by the memory: each element is read and written once, next to 2-3 operations.  What could cost more is the angles, so a
// thread forms the cosines and sines of its pairs once and applies them to several heads of its token.  Angles: the position
// times the frequency in turns, reduced to half a turn, in 64 bits (a product in 32 bits is off by 0.06 rad at position
// 10^6); the rest in 32 bits.
#include "element.cuh"
#include "ringrnn_common.cuh"

namespace ringrnn {
namespace {

struct RotaryArgs {
  int T, Hq, Hk, D, half;  // half = rotated / 2
  int inverse;
  float amplitude;
  const char *q, *k;
  long long qb, qt, qh, kb, kt, kh;
  const double* frequency;
  const void* positions;
  int position_bytes;
  long long pb, pt, first;
  char *q_out, *k_out;
  long long tokens;       // B * T
  int slots, turn_slots;  // per head: turn_slots of V pairs each, then slots of 2 V copied elements (the last may be short)
  int groups;             // threads share a token's heads: group g takes heads g, g + groups, ...
};

// One thread: one slot of one token for the heads of its group, two heads in flight.
template <class E, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  typedef Pack<E, V> P;
  const long long id = blockIdx.x * 256LL + threadIdx.x;
  const int per_token = a.slots * a.groups;
  const long long token = id / per_token;
  if (token >= a.tokens) return;
  const int rest = (int)(id - token * per_token), group = rest / a.slots, slot = rest - group * a.slots;
  const long long b = token / a.T, t = token - b * a.T;
  const int heads = a.Hq + a.Hk;
  const E* q = reinterpret_cast<const E*>(a.q) + b * a.qb + t * a.qt;
  const E* k = reinterpret_cast<const E*>(a.k) + b * a.kb + t * a.kt;
  E* qo = reinterpret_cast<E*>(a.q_out) + token * a.Hq * a.D;
  E* ko = reinterpret_cast<E*>(a.k_out) + token * a.Hk * a.D;
  auto from = [&](int h) { return h < a.Hq ? q + h * a.qh : k + (h - a.Hq) * a.kh; };
  auto to = [&](int h) { return h < a.Hq ? qo + (long long)h * a.D : ko + (long long)(h - a.Hq) * a.D; };
  if (slot < a.turn_slots) {
    const int p0 = slot * V, i0 = INTERLEAVED ? 2 * p0 : p0, i1 = INTERLEAVED ? 2 * p0 + V : a.half + p0;
    // pos * frequency in turns, less the nearest whole number of them
    long long pos = a.first;
    if (a.position_bytes == 8) pos += static_cast<const long long*>(a.positions)[b * a.pb + t * a.pt];
    else if (a.position_bytes == 4) pos += static_cast<const int*>(a.positions)[b * a.pb + t * a.pt];
    else pos += t;
    float c[V], s[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const double turns = (double)pos * (a.frequency[p0 + e] * 0.15915494309189535);
      sincospif((float)(2.0 * (turns - rint(turns))), &s[e], &c[e]);
      c[e] *= a.amplitude;
      s[e] *= a.inverse ? -a.amplitude : a.amplitude;
    }
    auto turn = [&](const P& x0, const P& x1, E* o) {
      P y0, y1;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (INTERLEAVED) {
          // element pairs run through both vectors in order
          const int i = 2 * e, j = 2 * e + 1;
          const float u = up(i < V ? x0.v[i % V] : x1.v[i % V]), w = up(j < V ? x0.v[j % V] : x1.v[j % V]);
          const E yu = down<E>(u * c[e] - w * s[e]), yw = down<E>(w * c[e] + u * s[e]);
          if (i < V) y0.v[i % V] = yu; else y1.v[i % V] = yu;
          if (j < V) y0.v[j % V] = yw; else y1.v[j % V] = yw;
        } else {
          const float u = up(x0.v[e]), w = up(x1.v[e]);
          y0.v[e] = down<E>(u * c[e] - w * s[e]);
          y1.v[e] = down<E>(w * c[e] + u * s[e]);
        }
      }
      *reinterpret_cast<P*>(o + i0) = y0;
      *reinterpret_cast<P*>(o + i1) = y1;
    };
    int h = group;
    for (; h + 3 * a.groups < heads; h += 4 * a.groups) {
      P x[4][2];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const E* f = from(h + m * a.groups);
        x[m][0] = *reinterpret_cast<const P*>(f + i0);
        x[m][1] = *reinterpret_cast<const P*>(f + i1);
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) turn(x[m][0], x[m][1], to(h + m * a.groups));
    }
    for (; h < heads; h += a.groups) {
      const E* f = from(h);
      turn(*reinterpret_cast<const P*>(f + i0), *reinterpret_cast<const P*>(f + i1), to(h));
    }
  } else {
    const int i0 = 2 * a.half + (slot - a.turn_slots) * 2 * V;
    const bool both = i0 + V < a.D;
    int h = group;
    for (; h < heads; h += a.groups) {
      const E* f = from(h);
      E* o = to(h);
      const P x0 = *reinterpret_cast<const P*>(f + i0);
      if (both) *reinterpret_cast<P*>(o + i0 + V) = *reinterpret_cast<const P*>(f + i0 + V);
      *reinterpret_cast<P*>(o + i0) = x0;
    }
  }
}

template <class E, int V>
int launch(RotaryArgs a, int interleaved, cudaStream_t s) {
  a.turn_slots = a.half / V;
  a.slots = a.turn_slots + (a.D - 2 * a.half + 2 * V - 1) / (2 * V);
  // Heads per thread: all of a token's, if the tokens alone give the GPU its threads (148 SMs, 1024 each), else as few as it
  // takes for that.
  const int heads = a.Hq + a.Hk;
  const long long one = a.tokens * a.slots, want = 148LL * 1024;
  long long groups = (want + one - 1) / one;
  groups = groups > heads ? heads : groups;
  a.groups = (int)groups;
  const long long blocks = (one * groups + 255) / 256;
  if (blocks > 2147483647LL) return RINGRNN_ERR_SHAPE;
  LaunchScope ls(K_LAYER, s);
  if (interleaved) rotary_kernel<E, V, true><<<(unsigned)blocks, 256, 0, s>>>(a);
  else rotary_kernel<E, V, false><<<(unsigned)blocks, 256, 0, s>>>(a);
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}

// The widest vectors (16 bytes) that divide both halves and the rest and that every address is a multiple of.
template <class E>
int dispatch(const RotaryArgs& a, int interleaved, cudaStream_t s) {
  constexpr int MOST = 16 / sizeof(E);
  auto fits = [&](int v) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) |
                         (a.Hk ? reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.k_out) : 0);
    const long long strides = a.qb | a.qt | a.qh | (a.Hk ? a.kb | a.kt | a.kh : 0) | a.half | a.D;
    return strides % v == 0 && at % (v * sizeof(E)) == 0;
  };
  if (fits(MOST)) return launch<E, MOST>(a, interleaved, s);
  if (fits(MOST / 2)) return launch<E, MOST / 2>(a, interleaved, s);
  if constexpr (MOST == 8)
    if (fits(2)) return launch<E, 2>(a, interleaved, s);
  return launch<E, 1>(a, interleaved, s);
}

}  // namespace
}  // namespace ringrnn

extern "C" int ringrnn_rotary(const RingRnnRotary* p, void* stream) {
  using namespace ringrnn;
  if (p == nullptr) return RINGRNN_ERR_ARG;
  const bool with_k = p->k.data != nullptr;
  if (p->B <= 0 || p->T <= 0 || p->Hq <= 0 || (with_k && p->Hk <= 0) || p->D <= 0 || p->rotated <= 0 || p->rotated % 2 != 0 || p->rotated > p->D)
    return RINGRNN_ERR_SHAPE;
  if (p->D > 65536 || p->Hq > 65536 || (with_k && p->Hk > 65536)) return RINGRNN_ERR_SHAPE;
  if (!p->q.data || !p->q_out || (with_k && !p->k_out) || !p->frequency) return RINGRNN_ERR_ARG;
  if (p->position_bytes != 0 && p->position_bytes != 4 && p->position_bytes != 8) return RINGRNN_ERR_ARG;
  if (p->position_bytes != 0 && !p->positions) return RINGRNN_ERR_ARG;
  RotaryArgs a;
  a.T = p->T; a.Hq = p->Hq; a.Hk = with_k ? p->Hk : 0; a.D = p->D; a.half = p->rotated / 2;
  a.inverse = p->inverse; a.amplitude = p->amplitude;
  a.q = static_cast<const char*>(p->q.data); a.k = static_cast<const char*>(p->k.data);
  a.qb = p->q.batch; a.qt = p->q.token; a.qh = p->q.head;
  a.kb = p->k.batch; a.kt = p->k.token; a.kh = p->k.head;
  a.frequency = p->frequency;
  a.positions = p->positions; a.position_bytes = p->position_bytes;
  a.pb = p->position_batch; a.pt = p->position_token; a.first = p->first;
  a.q_out = static_cast<char*>(p->q_out); a.k_out = static_cast<char*>(p->k_out);
  a.tokens = (long long)p->B * p->T;
  a.slots = a.turn_slots = a.groups = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p->dtype) {
    case RINGRNN_F32: return dispatch<float>(a, p->interleaved, s);
    case RINGRNN_BF16: return dispatch<__nv_bfloat16>(a, p->interleaved, s);
    case RINGRNN_F16: return dispatch<__half>(a, p->interleaved, s);
    default: return RINGRNN_ERR_ARG;
  }
}
