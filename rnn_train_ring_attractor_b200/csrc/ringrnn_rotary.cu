// Rotary positions: pairs of a head's elements turned by position * frequency.
//
// Bound by the memory: each element is read and written once, next to 2-3 operations.  What costs more is instructions for
// anything else, so a thread stays with a place in the head and a token, forms the cosines and sines of its pairs once and goes
// from head to head by one addition to each address.  Angles: the position times the frequency in turns, reduced to half a turn,
// in 64 bits (a product in 32 bits is off by 0.06 rad at position 10^6); the rest in 32 bits.
// 8 x 2048 tokens, 32 query and 8 key heads of 128 in bf16: 61 us, 5.5 TB/s (with eight vectors on their way per thread 75, for
// the registers they take; with the angles in a table in shared memory and rows shared out evenly 115, for the address arithmetic).
#include "element.cuh"
#include "ringrnn_common.cuh"

namespace ringrnn {
namespace {

constexpr int THREADS = 128;
// threads per SM that heads are shared out for; measured at the sizes below, adjacent pairs and halves (us): 1536: 62.5, 2560: 61.4
// and 67.6, 2944: 61.5 and 63.5, 4096: 71.7 and 69.7
constexpr long long WANTED = 2944;

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
  int slots, turn_slots;  // per head: first the slots whose elements turn, then those that are copied
  int groups;             // threads share a token's heads: group g takes heads g, g + groups, ...
};

// One thread: one slot of one token for the heads of its group, some of them on their way at once.  A slot is V consecutive
// elements if pairs are adjacent, else V of each half; copied elements go through the same loads and stores, since a warp has
// slots of both kinds.
template <class E, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS, 8) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  typedef Pack<E, V> P;
  constexpr int NV = INTERLEAVED && V > 1 ? 1 : 2, PAIRS = NV * V / 2;  // vectors and pairs of a slot
  constexpr int AHEAD = 4 / NV;
  const long long id = blockIdx.x * (long long)THREADS + threadIdx.x;
  const int per_token = a.slots * a.groups;
  const long long token = id / per_token;
  if (token >= a.tokens) return;
  const int rest = (int)(id - token * per_token), group = rest / a.slots, slot = rest - group * a.slots;
  const long long b = token / a.T, t = token - b * a.T;
  const bool turns = slot < a.turn_slots;
  const int p0 = slot * PAIRS;  // first pair
  int i0, apart = 0;            // where the slot's vectors stand
  if (NV == 1) {
    i0 = slot * V;
  } else if (turns) {
    i0 = INTERLEAVED ? 2 * p0 : p0;
    apart = INTERLEAVED ? V : a.half;
  } else {
    i0 = 2 * a.half + (slot - a.turn_slots) * 2 * V;
    apart = i0 + V < a.D ? V : 0;  // (a lone vector at the end is copied twice)
  }
  float c[PAIRS], s[PAIRS];
  if (turns) {
    long long pos = a.first;
    if (a.position_bytes == 8) pos += static_cast<const long long*>(a.positions)[b * a.pb + t * a.pt];
    else if (a.position_bytes == 4) pos += static_cast<const int*>(a.positions)[b * a.pb + t * a.pt];
    else pos += t;
#pragma unroll
    for (int e = 0; e < PAIRS; ++e) {
      // pos * frequency in turns, less the nearest whole number of them
      const double turn = (double)pos * (a.frequency[p0 + e] * 0.15915494309189535);
      sincospif((float)(2.0 * (turn - rint(turn))), &s[e], &c[e]);
      c[e] *= a.amplitude;
      s[e] *= a.inverse ? -a.amplitude : a.amplitude;
    }
  }
  auto turn = [&](P* x) {
#pragma unroll
    for (int e = 0; e < PAIRS; e += PAIRS > 1 ? 2 : 1) {
      // pairs of pairs, so that two results that stand side by side are rounded at once
      constexpr int W = PAIRS > 1 ? 2 : 1;
      float y[2], z[2];
#pragma unroll
      for (int d = 0; d < W; ++d) {
        const int j = e + d;
        const float u = up(NV == 1 ? x[0].v[2 * j] : INTERLEAVED ? x[2 * j / V].v[2 * j % V] : x[0].v[j]);
        const float w = up(NV == 1 ? x[0].v[2 * j + 1] : INTERLEAVED ? x[(2 * j + 1) / V].v[(2 * j + 1) % V] : x[NV - 1].v[j]);
        y[d] = u * c[j] - w * s[j];
        z[d] = w * c[j] + u * s[j];
      }
      if constexpr (NV == 1) {
#pragma unroll
        for (int d = 0; d < W; ++d) down2(y[d], z[d], x[0].v + 2 * (e + d));
      } else if constexpr (V == 1) {
        x[0].v[0] = down<E>(y[0]);
        x[NV - 1].v[0] = down<E>(z[0]);
      } else {
        down2(y[0], y[1], x[0].v + e);
        down2(z[0], z[1], x[NV - 1].v + e);
      }
    }
  };
  // heads group, group + groups, ... of one tensor
  auto heads = [&](const char* data, long long at, long long head, char* out, int H) {
    const E* from = reinterpret_cast<const E*>(data) + at + group * head + i0;
    E* to = reinterpret_cast<E*>(out) + (token * H + group) * a.D + i0;
    const long long from_step = a.groups * head;
    const int to_step = a.groups * a.D;
    int left = (H - group + a.groups - 1) / a.groups;
#pragma unroll 1
    for (; left >= AHEAD; left -= AHEAD) {
      P x[AHEAD][NV];
#pragma unroll
      for (int m = 0; m < AHEAD; ++m, from += from_step)
#pragma unroll
        for (int n = 0; n < NV; ++n) x[m][n] = *reinterpret_cast<const P*>(from + n * apart);
      if (turns)
#pragma unroll
        for (int m = 0; m < AHEAD; ++m) turn(x[m]);
#pragma unroll
      for (int m = 0; m < AHEAD; ++m, to += to_step)
#pragma unroll
        for (int n = 0; n < NV; ++n) *reinterpret_cast<P*>(to + n * apart) = x[m][n];
    }
#pragma unroll 1
    for (; left > 0; --left, from += from_step, to += to_step) {
      P x[NV];
#pragma unroll
      for (int n = 0; n < NV; ++n) x[n] = *reinterpret_cast<const P*>(from + n * apart);
      if (turns) turn(x);
#pragma unroll
      for (int n = 0; n < NV; ++n) *reinterpret_cast<P*>(to + n * apart) = x[n];
    }
  };
  heads(a.q, b * a.qb + t * a.qt, a.qh, a.q_out, a.Hq);
  if (a.Hk > 0) heads(a.k, b * a.kb + t * a.kt, a.kh, a.k_out, a.Hk);
}

template <class E, int V>
int launch(RotaryArgs a, int interleaved, cudaStream_t s) {
  const int pairs = interleaved && V > 1 ? V / 2 : V;
  a.turn_slots = a.half / pairs;
  a.slots = a.turn_slots + (a.D - 2 * a.half + 2 * pairs - 1) / (2 * pairs);
  // Heads per thread: all of a token's, if the tokens alone give the GPU threads for two or three rounds, else as few as it takes.
  const int most = a.Hq > a.Hk ? a.Hq : a.Hk;
  const long long one = a.tokens * a.slots, want = 148 * WANTED;
  const long long groups = (want + one - 1) / one;
  a.groups = (int)(groups > most ? most : groups);
  const long long blocks = (one * a.groups + THREADS - 1) / THREADS;
  if (blocks > 2147483647LL) return RINGRNN_ERR_SHAPE;
  LaunchScope ls(K_LAYER, s);
  if (interleaved) rotary_kernel<E, V, true><<<(unsigned)blocks, THREADS, 0, s>>>(a);
  else rotary_kernel<E, V, false><<<(unsigned)blocks, THREADS, 0, s>>>(a);
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}

// The widest vectors (16 bytes) that divide what turns (each half of it, unless pairs are adjacent) and the rest, and that every
// address is a multiple of.
template <class E>
int dispatch(const RotaryArgs& a, int interleaved, cudaStream_t s) {
  constexpr int MOST = 16 / sizeof(E);
  auto fits = [&](int v) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) |
                         (a.Hk ? reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.k_out) : 0);
    const long long strides = a.qb | a.qt | a.qh | (a.Hk ? a.kb | a.kt | a.kh : 0) | (interleaved ? 2 * a.half : a.half) | a.D;
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
