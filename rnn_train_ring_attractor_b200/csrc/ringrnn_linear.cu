// Linear attention with decay: entry points, the fp32-arithmetic kernel, the scan over segments, and the single-token step.
#include <string.h>

#include "element.cuh"
#include "linear_attention.cuh"

namespace ringrnn {
namespace {

// ---- fp32 arithmetic: any type, any width up to 256 -----------------------------------------------------------------
// One CTA per (job, sequence, head, segment) and slice of 64 outer columns, chunks of 32 tokens (of 16, 32 and 64, 32 has the
// fewest products per token next to the state's own 2 * inner * 64 that still leave several CTAs per SM their shared memory).
//
// Products on the tensor cores' tf32 type: x = hi + lo with hi rounded to tf32's eleven bits; what is left, of up to twelve bits, goes
// in as it is, and the tensor cores take eleven of them, so a factor is off by a unit of fp32's last place at most (2^-23).
// x y = hi hi + hi lo + lo hi but for lo lo, at most 2^-22 of it: together 2^-21 of a product, where fp32 rounds to 2^-24 (a state of one
// product, with its sums: 8.8 * 2^-24 measured); over a long sum, with either sign, 3e-7 of it where plain fp32 leaves 2e-7.
// (Infinities may become NaN on the way.)  The same products on the CUDA cores were bound by the operands' way through shared
// memory, four cycles for each 16 bytes a thread reads; a fragment's element is read once per product of 16 x 8 x 8.  Measured in
// fp32, 16 x 512 x 16 heads of 64, on CUDA cores and so: forward 183 and 119 us, backward 532 and 340 (the memory alone 21 and
// 36 us: what bounds it is three products for one, on mma.sync, and their fragments' way from shared memory).
// The state stays in registers as an accumulator and is copied to shared memory once a chunk, where the outputs read it.  A chunk's
// numbers are loaded into registers while the one before is at work (widths up to 128).
constexpr int PC = 32, PO = 64, P_THREADS = 256, P_WARPS = P_THREADS / 32;
constexpr int P_LD = PC + 4, V_LD = PO + 8;  // rows 4 (8) banks apart: the lanes of a fragment then read 32 different ones

__host__ __device__ constexpr int plain_width(int inner) { return (inner + 15) / 16 * 16; }
size_t plain_smem(int inner) {
  return sizeof(float) * (2 * PC * (plain_width(inner) + 4) + PC * V_LD + PC * P_LD + 3 * PC + 4 + (size_t)plain_width(inner) * V_LD);
}

struct Split {
  uint32_t hi, lo;
  __device__ __forceinline__ explicit Split(float x) {
    // (to the largest number of eleven bits at most: plain rounding makes infinities of what lies above it, and NaN of those)
    asm("cvt.rn.satfinite.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    lo = __float_as_uint(x - __uint_as_float(hi));
  }
};
// c += a b for a 16 x 8 by 8 x 8 product; lane 4 g + t holds of a: (g, t), (g + 8, t), (g, t + 4), (g + 8, t + 4); of b: (t, g),
// (t + 4, g); of c: (g, 2 t), (g, 2 t + 1), (g + 8, 2 t), (g + 8, 2 t + 1)
__device__ __forceinline__ void mma_tf32(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The tensor cores cut a sum off instead of rounding it, 2^-24 of it and always the same way, which over the thousands of sums
// behind a state would show (2.6e-6 of an output, where the CUDA cores leave 2e-7).  So they add up 32 products at a time, the
// small ones apart, and the CUDA cores the rest.
struct Sums {
  float big[4] = {0.f, 0.f, 0.f, 0.f}, small[4] = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(const Split* a, const Split* b) {
    mma_tf32(small, a[0].lo, a[1].lo, a[2].lo, a[3].lo, b[0].hi, b[1].hi);
    mma_tf32(big, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[0].hi, b[1].hi);
    mma_tf32(small, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[0].lo, b[1].lo);
  }
  __device__ __forceinline__ float value(int e) const { return big[e] + small[e]; }
};

// NC: inner columns a lane loads of each row, 32 apart
template <class E, bool STATES, int NC>
__global__ void __launch_bounds__(P_THREADS, NC <= 4 ? 2 : 1) la_plain_kernel(const __grid_constant__ LaLaunch L) {
  extern __shared__ float sm[];
  constexpr bool AHEAD = NC <= 4;
  constexpr int ROWS = PC / P_WARPS;  // a warp loads rows warp, warp + 8, ...
  constexpr int MT = NC / 2;          // a warp's tiles of the state: rows 16 ((warp & 3) + 4 i), columns 32 (warp >> 2) and on
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int ji = (int)(blockIdx.x % L.jobs);
  const LaJob& J = L.job[ji];
  const int at = (int)(blockIdx.x / L.jobs), seg = at % L.segments, bh = at / L.segments, h = bh % L.H, b = bh / L.H;
  const int o0 = blockIdx.y * PO;
  if (o0 >= J.outer) return;
  const int I = J.inner, IP = plain_width(I), ld = IP + 4, on = min(PO, J.outer - o0);
  float* Q = sm;               // [PC][ld]
  float* K = Q + PC * ld;      // [PC][ld]
  float* V = K + PC * ld;      // [PC][V_LD]
  float* P = V + PC * V_LD;    // [PC][P_LD]
  float* pw = P + PC * P_LD;   // [PC + 4] powers of the decay
  float* wk = pw + PC + 4;     // [PC] factor of a key in the state
  float* wr = wk + PC;         // [PC] factor of the state in a row
  float* S = wr + PC;          // [IP][V_LD]
  const int len = la_length(L, b);
  const int begin = seg * L.segment_tokens, stop = min(L.T, begin + L.segment_tokens), end = min(len, stop);
  const size_t mat = (size_t)at * J.inner * J.outer;
  if (tid <= PC) pw[tid] = LaDecay(L.log_decay[h]).power(tid);
  const int col0 = (warp >> 2) * 32;
  float state[MT][4][4];  // tile, 8 columns, element of the fragment
  auto state_row = [&](int i, int e) { return 16 * ((warp & 3) + 4 * i) + g + (e >> 1) * 8; };
  auto state_col = [&](int n, int e) { return col0 + 8 * n + 2 * t + (e & 1); };
  {
    const bool given = !STATES && J.init != nullptr;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = state_row(i, e), o = state_col(n, e);
          state[i][n][e] = given && r < I && o < on ? J.init[mat + (size_t)r * J.s_in + (size_t)(o0 + o) * J.s_out] : 0.f;
        }
  }
  const E* q = static_cast<const E*>(J.q.p) + b * J.q.sb + h * J.q.sh;
  const E* k = static_cast<const E*>(J.k.p) + b * J.k.sb + h * J.k.sh;
  const E* v = static_cast<const E*>(J.v.p) + b * J.v.sb + h * J.v.sh + o0;
  E* out = static_cast<E*>(J.out);

  const int chunks = end > begin ? (end - begin + PC - 1) / PC : 0;
  auto chunk_at = [&](int c) { return begin + (J.reverse ? chunks - 1 - c : c) * PC; };
  const LaFactor whole(L.log_decay[h], PC);
  float qr[AHEAD ? ROWS : 1][NC], kr[AHEAD ? ROWS : 1][NC], vr[AHEAD ? ROWS : 1][2];
  // row j of this warp's: what is not there counts as zero
  auto load_row = [&](int t0, int n, int j, float* x, float* y, float* z) {
    const int r = warp + j * P_WARPS;
    const bool row = r < n;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const bool in = row && lane + 32 * i < I;
      if (!STATES) x[i] = in ? up(q[(t0 + r) * J.q.st + lane + 32 * i]) : 0.f;
      y[i] = in ? up(k[(t0 + r) * J.k.st + lane + 32 * i]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) z[i] = row && lane + 32 * i < on ? up(v[(t0 + r) * J.v.st + lane + 32 * i]) : 0.f;
  };
  auto store_row = [&](int j, const float* x, const float* y, const float* z) {
    const int r = warp + j * P_WARPS;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (lane + 32 * i < IP) {
        if (!STATES) Q[r * ld + lane + 32 * i] = x[i];
        K[r * ld + lane + 32 * i] = y[i];
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) V[r * V_LD + lane + 32 * i] = z[i];
  };
  auto load_chunk = [&](int c) {
    const int t0 = chunk_at(c), n = min(PC, end - t0);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) load_row(t0, n, j, qr[j], kr[j], vr[j]);
  };
  // fragments: a's rows are rows of memory; b's k index is a column (by_column) or a row of memory
  auto frag_a = [&](const float* m, int stride, int k0, Split* x) {
    x[0] = Split(m[g * stride + k0 + t]);
    x[1] = Split(m[(g + 8) * stride + k0 + t]);
    x[2] = Split(m[g * stride + k0 + t + 4]);
    x[3] = Split(m[(g + 8) * stride + k0 + t + 4]);
  };
  if (AHEAD && chunks > 0) load_chunk(0);
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    const int t0 = chunk_at(c), n = min(PC, end - t0);
    __syncthreads();
    if (AHEAD) {
#pragma unroll
      for (int j = 0; j < ROWS; ++j) store_row(j, qr[j], kr[j], vr[j]);
    } else {
      for (int j = 0; j < ROWS; ++j) {
        load_row(t0, n, j, qr[0], kr[0], vr[0]);
        store_row(j, qr[0], kr[0], vr[0]);
      }
    }
    if (!STATES) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
        if (state_row(i, 0) - g < IP)
#pragma unroll
          for (int n8 = 0; n8 < 4; ++n8)
#pragma unroll
            for (int e = 0; e < 4; e += 2)
              *reinterpret_cast<float2*>(S + state_row(i, e) * V_LD + state_col(n8, 0)) = make_float2(state[i][n8][e], state[i][n8][e + 1]);
    }
    if (tid < PC) wk[tid] = tid < n ? J.key_scale * pw[J.reverse ? tid + 1 : n - 1 - tid] : 0.f;
    else if (tid < 2 * PC) {
      const int r = tid - PC;
      wr[r] = r < n ? J.row_scale * pw[J.reverse ? n - 1 - r : r + 1] : 0.f;
    }
    __syncthreads();
    if (AHEAD && c + 1 < chunks) load_chunk(c + 1);
    if (!STATES) {
      const int row0 = (warp & 1) * 16;
      {  // scores: 16 tokens by 8 keys
        const int key0 = (warp >> 1) * 8;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int k32 = 0; k32 < IP; k32 += 32) {
          Sums sums;
#pragma unroll
          for (int k0 = k32; k0 < k32 + 32; k0 += 8) {
            if (k0 >= IP) break;
            Split x[4] = {Split(0.f), Split(0.f), Split(0.f), Split(0.f)};
            frag_a(Q + row0 * ld, ld, k0, x);
            const Split y[2] = {Split(K[(key0 + g) * ld + k0 + t]), Split(K[(key0 + g) * ld + k0 + t + 4])};
            sums.add(x, y);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += sums.value(e);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = row0 + g + (e >> 1) * 8, j = key0 + 2 * t + (e & 1), far = J.reverse ? j - i : i - j;
          acc[e] = far >= 0 && i < n && j < n ? acc[e] * (J.pair_scale * pw[far]) : 0.f;
        }
        *reinterpret_cast<float2*>(P + (row0 + g) * P_LD + key0 + 2 * t) = make_float2(acc[0], acc[1]);
        *reinterpret_cast<float2*>(P + (row0 + g + 8) * P_LD + key0 + 2 * t) = make_float2(acc[2], acc[3]);
      }
      __syncthreads();
      {  // outputs: 16 tokens by 16 columns; the state's part, then the pairs'
        const int o = (warp >> 1) * 16;
        float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        auto step = [&](const float* a, int a_ld, const float* m, int k32, int end_k) {
          Sums sums[2];
#pragma unroll
          for (int k0 = k32; k0 < k32 + 32; k0 += 8) {
            if (k0 >= end_k) break;
            Split x[4] = {Split(0.f), Split(0.f), Split(0.f), Split(0.f)};
            frag_a(a + row0 * a_ld, a_ld, k0, x);
#pragma unroll
            for (int n8 = 0; n8 < 2; ++n8) {
              const Split y[2] = {Split(m[(k0 + t) * V_LD + o + 8 * n8 + g]), Split(m[(k0 + t + 4) * V_LD + o + 8 * n8 + g])};
              sums[n8].add(x, y);
            }
          }
#pragma unroll
          for (int n8 = 0; n8 < 2; ++n8)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n8][e] += sums[n8].value(e);
        };
#pragma unroll 1
        for (int k32 = 0; k32 < IP; k32 += 32) step(Q, ld, S, k32, IP);
        const float w0 = wr[row0 + g], w1 = wr[row0 + g + 8];
#pragma unroll
        for (int n8 = 0; n8 < 2; ++n8)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n8][e] *= e < 2 ? w0 : w1;
        step(P, P_LD, V, 0, PC);
#pragma unroll
        for (int n8 = 0; n8 < 2; ++n8)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = row0 + g + (e >> 1) * 8, x = o + 8 * n8 + 2 * t + (e & 1);
            if (r < n && x < on) out[(((size_t)b * L.T + t0 + r) * L.H + h) * J.outer + o0 + x] = down<E>(acc[n8][e]);
          }
      }
    }
    {  // the state: its rows are the keys' columns
      const LaFactor gn = n == PC ? whole : LaFactor(L.log_decay[h], n);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int r = 16 * ((warp & 3) + 4 * i);
        if (r >= IP) break;
        Sums sums[4];
#pragma unroll 1
        for (int k0 = 0; k0 < PC; k0 += 8) {
          const float w0 = wk[k0 + t], w1 = wk[k0 + t + 4];
          const Split x[4] = {Split(K[(k0 + t) * ld + r + g]), Split(K[(k0 + t) * ld + r + g + 8]), Split(K[(k0 + t + 4) * ld + r + g]),
                              Split(K[(k0 + t + 4) * ld + r + g + 8])};
#pragma unroll
          for (int n8 = 0; n8 < 4; ++n8) {
            const Split y[2] = {Split(w0 * V[(k0 + t) * V_LD + col0 + 8 * n8 + g]), Split(w1 * V[(k0 + t + 4) * V_LD + col0 + 8 * n8 + g])};
            sums[n8].add(x, y);
          }
        }
#pragma unroll
        for (int n8 = 0; n8 < 4; ++n8)
#pragma unroll
          for (int e = 0; e < 4; ++e) state[i][n8][e] = gn.times(state[i][n8][e], sums[n8].value(e));
      }
    }
  }
  if (!STATES) {  // rows behind the sequence
    // (by rows: rows times columns may not fit 31 bits)
    for (int r = max(begin, end) + tid / PO; r < stop; r += P_THREADS / PO)
      if (tid % PO < on) out[(((size_t)b * L.T + r) * L.H + h) * J.outer + o0 + tid % PO] = down<E>(0.f);
  }
  if (J.fin != nullptr)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n8 = 0; n8 < 4; ++n8)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = state_row(i, e), o = state_col(n8, e);
          if (r < I && o < on) J.fin[mat + (size_t)r * J.s_in + (size_t)(o0 + o) * J.s_out] = state[i][n8][e];
        }
}

template <class E, bool STATES, int NC>
int plain_launch(const LaLaunch& L, int inner, int outer, cudaStream_t s) {
  RINGRNN_CUDA_TRY(cudaFuncSetAttribute(la_plain_kernel<E, STATES, NC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plain_smem(32 * NC)));
  const dim3 grid((unsigned)(L.B * L.H * L.segments * L.jobs), (unsigned)((outer + PO - 1) / PO));
  LaunchScope ls(K_LAYER, s);
  la_plain_kernel<E, STATES, NC><<<grid, P_THREADS, plain_smem(inner), s>>>(L);
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}
template <class E, bool STATES>
int plain_launch(const LaLaunch& L, cudaStream_t s) {
  int inner = 0, outer = 0;
  for (int j = 0; j < L.jobs; ++j) {
    inner = L.job[j].inner > inner ? L.job[j].inner : inner;
    outer = L.job[j].outer > outer ? L.job[j].outer : outer;
  }
  return inner <= 64    ? plain_launch<E, STATES, 2>(L, inner, outer, s)
         : inner <= 128 ? plain_launch<E, STATES, 4>(L, inner, outer, s)
                        : plain_launch<E, STATES, 8>(L, inner, outer, s);
}
template <bool STATES>
int plain_launch(int dtype, const LaLaunch& L, cudaStream_t s) {
  return dtype == RINGRNN_F32    ? plain_launch<float, STATES>(L, s)
         : dtype == RINGRNN_BF16 ? plain_launch<__nv_bfloat16, STATES>(L, s)
                                 : plain_launch<__half, STATES>(L, s);
}

// ---- scan over segments -----------------------------------------------------------------------------------------------
// sums[bh][segment][elems] (each segment's own sum) becomes the state it starts from, in place; `last`: the state behind all
// of them.  A thread owns one element.  Bound by latency (18 segments of 8 heads of 128 x 128: 9 us, 19 MB): sixteen segments
// are on their way while two threads of the block form the decays, over a whole segment and over the one that may be shorter.
__global__ void __launch_bounds__(256) la_scan_kernel(int B, int T, int H, int segments, int segment_tokens, int elems,
                                                      int reverse, const float* log_decay, const int* lengths,
                                                      const float* init, float* sums, float* last) {
  const int bh = blockIdx.x, b = bh / H, e = blockIdx.y * 256 + threadIdx.x;
  const bool mine = e < elems;
  __shared__ float2 factor[2];
  int len = lengths == nullptr ? T : lengths[b];
  len = len < 0 ? 0 : len > T ? T : len;
  float x = init != nullptr && mine ? init[(size_t)bh * elems + e] : 0.f;
  float* u = sums + (size_t)bh * segments * elems + e;
  constexpr int AHEAD = 16;
  for (int j0 = 0; j0 < segments; j0 += AHEAD) {
    float y[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int j = reverse ? segments - 1 - (j0 + a) : j0 + a;
      y[a] = j0 + a < segments && mine ? u[(size_t)j * elems] : 0.f;
    }
    if (j0 == 0) {
      if ((threadIdx.x & 31) == 0 && threadIdx.x < 64) {
        const LaFactor f(log_decay[bh % H], threadIdx.x == 0 ? segment_tokens : len % segment_tokens);
        factor[threadIdx.x >> 5] = make_float2(f.hi, f.lo);
      }
      __syncthreads();
    }
    const float2 whole = factor[0], rest = factor[1];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (j0 + a >= segments) break;
      const int j = reverse ? segments - 1 - (j0 + a) : j0 + a, n = len - j * segment_tokens;
      if (mine) u[(size_t)j * elems] = x;
      const float2 f = n >= segment_tokens ? whole : n > 0 ? rest : make_float2(1.f, 0.f);
      x = fmaf(f.x, x, fmaf(f.y, x, y[a]));
    }
  }
  if (last != nullptr && mine) last[(size_t)bh * elems + e] = x;
}
int scan_launch(const LaLaunch& L, int elems, int reverse, const float* init, float* sums, float* last, cudaStream_t s) {
  LaunchScope ls(K_LAYER, s);
  la_scan_kernel<<<dim3(L.B * L.H, (elems + 255) / 256), 256, 0, s>>>(L.B, L.T, L.H, L.segments, L.segment_tokens, elems, reverse,
                                                                     L.log_decay, L.lengths, init, sums, last);
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}

// ---- one token ----------------------------------------------------------------------------------------------------------
// Bound by the state, read and written once: 8 * dk * dv bytes per sequence and head.  A CTA takes 32 columns of one state:
// they are independent of one another, a single head then spreads over dv / 32 SMs, and a row's part is a whole 128-byte line.
// VEC = 4: a thread owns 4 columns of every THREADS / 8th row; VEC = 1 (odd widths or addresses): 1 column of every THREADS / 32nd.
// Threads: as many as leave each four rows, all of them under way at once; a block for each 32 x 64 of a small state would be
// half idle with 256 (256 sequences of 32 heads of 64: 62 us, and 47 with 128, 5.7 TB/s; heads of 128: 174 us, 6.2 TB/s).
// WHOLE: a CTA takes all columns, its threads a few rows of them, which lie one behind the other; for widths that are no multiple of
// 32, whose slices would share sectors and leave the last one half empty, where there are states enough for the GPU (256 sequences
// of 32 heads of 100: 109 us, in slices 223; of 101: 158 and 249; with the decay as two floats 109 and 175, for one more operation
// for each element, which at one element a load is what bounds the kernel).
constexpr int STEP_COLS = 32, STEP_MAX_DK = 1024;
template <class E, int VEC, int STEP_THREADS, bool WHOLE>
__global__ void __launch_bounds__(STEP_THREADS) la_step_kernel(int H, int dk, int dv, float scale, LaOperand q, LaOperand k,
                                                               LaOperand v, const float* __restrict__ log_decay,
                                                               const unsigned char* __restrict__ active,
                                                               float* __restrict__ state, E* __restrict__ out) {
  const int COLS = WHOLE ? dv : STEP_COLS, CG = COLS / VEC, ROWS = STEP_THREADS / CG;
  __shared__ float sq[STEP_MAX_DK], sk[STEP_MAX_DK];
  __shared__ float part[STEP_THREADS * VEC];  // [ROWS][COLS]
  const int tid = threadIdx.x, bh = blockIdx.x, h = bh % H, b = bh / H;
  const int cg = tid % CG, row = tid / CG, col = blockIdx.y * COLS + cg * VEC;
  if (active != nullptr && active[b] == 0) {
    if (row == 0)
      for (int e = 0; e < VEC; ++e)
        if (col + e < dv) out[(size_t)bh * dv + col + e] = down<E>(0.f);
    return;
  }
  const bool in = col < dv && row < ROWS;  // VEC == 4: dv is a multiple of 4
  float* S = state + (size_t)bh * dk * dv + col;
  // the state's first rows are under way while q and k come in
  constexpr int AHEAD = VEC == 4 ? 4 : 8;
  float s0[AHEAD][VEC];
  auto fetch = [&](float* x, int i) {
    if constexpr (VEC == 4) {
      const float4 y = *reinterpret_cast<const float4*>(S + (size_t)i * dv);
      x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
    } else {
      x[0] = S[(size_t)i * dv];
    }
  };
#pragma unroll
  for (int a = 0; a < AHEAD; ++a)
    if (in && row + a * ROWS < dk) fetch(s0[a], row + a * ROWS);
  const E* qp = static_cast<const E*>(q.p) + b * q.sb + h * q.sh;
  const E* kp = static_cast<const E*>(k.p) + b * k.sb + h * k.sh;
  const E* vp = static_cast<const E*>(v.p) + b * v.sb + h * v.sh;
  for (int i = tid; i < dk; i += STEP_THREADS) {
    sq[i] = up(qp[i]);
    sk[i] = up(kp[i]);
  }
  // The decay as two floats: one float's rounding, the same at every token, would add up over a memory (LaFactor).  expm1 is as exact
  // next to zero as exp is next to one, and hi - 1 has no rounding; below a half no memory is long enough.
  const float l = log_decay[h], hi = expf(l), lo = hi >= 0.5f && hi <= 2.f ? expm1f(l) - (hi - 1.f) : 0.f;
  float vv[VEC], acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    vv[e] = in ? up(vp[col + e]) : 0.f;
    acc[e] = 0.f;
  }
  __syncthreads();
  if (in) {
    for (int i0 = row; i0 < dk; i0 += AHEAD * ROWS) {
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int i = i0 + a * ROWS;
        if (i >= dk) break;
        const float kk = sk[i], qq = sq[i];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          s0[a][e] = fmaf(hi, s0[a][e], fmaf(lo, s0[a][e], kk * vv[e]));
          acc[e] = fmaf(qq, s0[a][e], acc[e]);
        }
        if constexpr (VEC == 4) *reinterpret_cast<float4*>(S + (size_t)i * dv) = make_float4(s0[a][0], s0[a][1], s0[a][2], s0[a][3]);
        else S[(size_t)i * dv] = s0[a][0];
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a)
        if (i0 + (AHEAD + a) * ROWS < dk) fetch(s0[a], i0 + (AHEAD + a) * ROWS);
    }
  }
  if (row < ROWS) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[row * COLS + cg * VEC + e] = acc[e];
  }
  __syncthreads();
  for (int o = tid; o < COLS && blockIdx.y * COLS + o < dv; o += STEP_THREADS) {
    float x = 0.f;
#pragma unroll 8
    for (int r = 0; r < ROWS; ++r) x += part[r * COLS + o];
    out[(size_t)bh * dv + blockIdx.y * COLS + o] = down<E>(scale * x);
  }
}
template <class E, int VEC, int THREADS, bool WHOLE = false>
int step_launch(const RingRnnLinearAttention& p, const LaOperand& q, const LaOperand& k, const LaOperand& v, float* state,
                const unsigned char* active, void* out, cudaStream_t s) {
  const dim3 grid(p.B * p.H, WHOLE ? 1 : (p.dv + STEP_COLS - 1) / STEP_COLS);
  LaunchScope ls(K_LAYER, s);
  la_step_kernel<E, VEC, THREADS, WHOLE><<<grid, THREADS, 0, s>>>(p.H, p.dk, p.dv, p.scale, q, k, v, p.log_decay, active, state, static_cast<E*>(out));
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}
template <class E>
int step_launch(const RingRnnLinearAttention& p, const LaOperand& q, const LaOperand& k, const LaOperand& v, float* state,
                const unsigned char* active, void* out, cudaStream_t s) {
  const int vec = p.dv % 4 != 0 || (reinterpret_cast<uintptr_t>(state) & 15) != 0 ? 1 : 4;
  if (p.dv % STEP_COLS != 0 && p.dv / vec <= 256 && (long long)p.B * p.H >= 2 * 148)
    return vec == 1 ? step_launch<E, 1, 256, true>(p, q, k, v, state, active, out, s) : step_launch<E, 4, 256, true>(p, q, k, v, state, active, out, s);
  if (vec == 1) return step_launch<E, 1, 256>(p, q, k, v, state, active, out, s);
  return p.dk <= 64 ? step_launch<E, 4, 128>(p, q, k, v, state, active, out, s) : step_launch<E, 4, 256>(p, q, k, v, state, active, out, s);
}

// ---- host -----------------------------------------------------------------------------------------------------------------
int check_linear(const RingRnnLinearAttention& p, bool step) {
  if (p.B <= 0 || p.H <= 0 || p.dk <= 0 || p.dv <= 0 || (!step && p.T <= 0)) return RINGRNN_ERR_SHAPE;
  if (step ? p.dk > STEP_MAX_DK : p.dk > 256 || p.dv > 256) return RINGRNN_ERR_SHAPE;
  // grid sizes (segments times jobs is at most 3 where there are that many heads)
  if ((long long)p.B * p.H > (1 << 29) || (step && (p.dv + STEP_COLS - 1) / STEP_COLS > 65535)) return RINGRNN_ERR_SHAPE;
  if (!step && p.T > (1 << 30)) return RINGRNN_ERR_SHAPE;
  if (p.dtype != RINGRNN_F32 && p.dtype != RINGRNN_BF16 && p.dtype != RINGRNN_F16) return RINGRNN_ERR_ARG;
  return RINGRNN_OK;
}
LaOperand operand(const RingRnnStrided& t) { return LaOperand{t.data, t.batch, t.token, t.head}; }

// ---- operands for the tensor cores ------------------------------------------------------------------------------------
// A tensor that TMA cannot read as it is (a stride or an address that is not a multiple of 16 bytes, tokens that share a row)
// is copied to rows of a multiple of 8 elements first, as many elements at a time as addresses and strides allow.  A thread writes
// eight and goes on by a fixed distance, kept as a number of packs, heads, tokens and sequences, where dividing for each pack cost
// as much as the copy.  8 x 2048 x 16 heads in bf16, this copy: of 60 31 us, of 121, where elements go one by one, 76.
struct PackJobs {
  LaOperand from[4];
  void* to[4];
  int width[4], per[4], vec[4];  // packs of a row; elements that are read at a time
  int step[4][4];                // the distance: packs, heads, tokens, sequences
};
template <int VEC>
__device__ __forceinline__ uint4 pack_of_8(const unsigned short* x, int left) {
  typedef Pack<unsigned short, VEC> P;
  Pack<unsigned short, 8> y;
#pragma unroll
  for (int e = 0; e < 8; e += VEC) {
    P z;
    if (e < left) {  // left is a multiple of VEC
      z = *reinterpret_cast<const P*>(x + e);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) z.v[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) y.v[e + i] = z.v[i];
  }
  return *reinterpret_cast<const uint4*>(&y);
}
__global__ void __launch_bounds__(256) la_pack_kernel(const __grid_constant__ PackJobs p, int B, int T, int H) {
  const int j = blockIdx.y, per = p.per[j], vec = p.vec[j];
  const LaOperand o = p.from[j];
  const size_t total = (size_t)B * T * H * per, step = (size_t)gridDim.x * 256;
  size_t id = blockIdx.x * (size_t)256 + threadIdx.x;
  const size_t row = id / per, bt = row / H;
  int i = (int)(id - row * per), h = (int)(row % H), t = (int)(bt % T), b = (int)(bt / T);
  for (; id < total; id += step) {
    const unsigned short* x = static_cast<const unsigned short*>(o.p) + b * o.sb + t * o.st + h * o.sh + i * 8;
    const int left = p.width[j] - i * 8;
    static_cast<uint4*>(p.to[j])[id] = vec == 4 ? pack_of_8<4>(x, left) : vec == 2 ? pack_of_8<2>(x, left) : pack_of_8<1>(x, left);
    i += p.step[j][0];
    const int ci = i >= per;
    i -= ci ? per : 0;
    h += p.step[j][1] + ci;
    const int ch = h >= H;
    h -= ch ? H : 0;
    t += p.step[j][2] + ch;
    const int ct = t >= T;
    t -= ct ? T : 0;
    b += p.step[j][3] + ct;
  }
}

// How a call runs.
struct Plan {
  bool tensor_cores;
  int segments, segment_tokens;
  size_t sums;         // bytes of a set of segment sums
  LaOperand op[4];     // q, k, v, d_out
  int width[4];
  size_t packed[4];    // bytes of a packed copy, 0: read as it is
  size_t bytes;        // whole workspace: one set of sums (backward: two), then the copies
};

// Segments of a sequence.  Forming their sums reads keys and values once more and is a launch of its own, with the scan behind it,
// so a sequence is only cut where that brings more CTAs to work: the number of segments with the least time by the model
//   rounds of CTAs x (start + chunks of a segment x chunk), for n > 1 the same again with part of a chunk's time, and the scan.
// Measured (us): tensor cores start 6, chunk 3, sums 0.55 of it; fp32 arithmetic start 6, chunk 4, sums 0.4 of it; a scan with the
// gaps between launches 10, the two scans of gradients 12.  (64 heads of 64, 16384 tokens, forward: cut in two 258 us, whole 311;
// 48 heads of 128, 2048 tokens: in three 66, whole 62.)  Gradients are three CTAs a segment, or two where those of keys and values
// go together (1.55 of a CTA's time): those first, then the others on what is free.
int cut(const RingRnnLinearAttention& p, bool tensor_cores, bool backward) {
  const int chunk = tensor_cores ? LA_TC_CHUNK : PC, at_once = tensor_cores ? LA_TC_BLOCKS : 296;
  const long long slices = tensor_cores ? 1 : ((p.dk > p.dv && backward ? p.dk : p.dv) + PO - 1) / PO;
  const long long each_job = (long long)p.B * p.H * slices, chunks = ((long long)p.T + chunk - 1) / chunk;
  const double start = 6, each = tensor_cores ? 3 : 4, sums = tensor_cores ? 0.55 : 0.4, scan = backward ? 12 : 10;
  auto rounds = [&](long long ctas) { return (double)((ctas + at_once - 1) / at_once); };
  auto rounds_of_all = [&](long long n) {
    const long long ctas = each_job * n;
    if (!backward || !tensor_cores || 3 * ctas <= at_once) return rounds((backward ? 3 : 1) * ctas);
    const long long full = ctas / at_once, more = ctas % at_once;  // after the pairs, `more` are free a pair's time after the others
    const double pair = 1.55, free[2] = {pair * full, pair * (full + 1)};
    auto whole = [](double x) { return x < 0 ? 0 : (long long)(x + 1e-9); };
    double least = more > 0 ? free[1] : free[0], end = 1e30;
    for (double from : free)
      for (long long k = full > 2 ? full - 2 : 0;; ++k) {
        const double t = from + k;
        if (more * whole(t - free[1]) + (at_once - more) * whole(t - free[0]) < ctas) continue;
        end = t < end ? t : end;
        break;
      }
    return end > least ? end : least;
  };
  int best = 1;
  double least = 0.9 * rounds_of_all(1) * (start + chunks * each);  // (a model: it has to promise a tenth)
  for (long long n = 2; n <= chunks / 2 && each_job * (backward ? 3 : 1) * (n - 1) < 2 * at_once; ++n) {
    const long long per = (chunks + n - 1) / n;
    const double t = rounds_of_all(n) * (start + per * each) + rounds((backward ? 2 : 1) * each_job * n) * (start + per * each * sums) + scan;
    if (t < least) least = t, best = (int)n;
  }
  return best;
}

Plan make_plan(const RingRnnLinearAttention& p, const RingRnnStrided* d_out) {
  Plan l;
  memset(&l, 0, sizeof(l));
  const bool backward = d_out != nullptr;
  // A few sequences of one chunk of the fp32 kernel are faster there (5 x 15 x 20 heads of 95 and 64, forward: 17 us and 28; many are
  // not: 64 x 32 x 24 heads of 128: 214 and 116) and more exact, for P and the state are not rounded.  The rule goes by time alone, so
  // a short sequence has other last bits, of the types' own size, in a large batch than in a small one.
  const int widest = p.dk > p.dv && backward ? p.dk : p.dv;
  const bool one_round = p.T <= PC && (long long)p.B * p.H * (backward ? 3 : 1) * ((widest + PO - 1) / PO) <= 2 * LA_TC_BLOCKS;
  l.tensor_cores = p.dtype != RINGRNN_F32 && p.dk <= LA_TC_WIDTH && p.dv <= LA_TC_WIDTH && !one_round;
  const int chunk = l.tensor_cores ? LA_TC_CHUNK : PC, n = cut(p, l.tensor_cores, backward);
  l.segment_tokens = (int)((((long long)p.T + n - 1) / n + chunk - 1) / chunk * chunk);
  l.segments = (int)(((long long)p.T + l.segment_tokens - 1) / l.segment_tokens);
  l.sums = l.segments > 1 ? align_up((size_t)p.B * p.H * l.segments * p.dk * p.dv * sizeof(float), 256) : 0;
  l.bytes = l.sums * (backward ? 2 : 1);
  l.op[0] = operand(p.q); l.op[1] = operand(p.k); l.op[2] = operand(p.v);
  l.width[0] = l.width[1] = p.dk; l.width[2] = l.width[3] = p.dv;
  if (backward) l.op[3] = operand(*d_out);
  if (l.tensor_cores)
    for (int x = 0; x < (backward ? 4 : 3); ++x)
      if (!la_tc_operand_ok(l.op[x], p.B, p.T, p.H)) {
        l.packed[x] = align_up((size_t)p.B * p.T * p.H * align_up(l.width[x], 8) * 2, 256);
        l.bytes += l.packed[x];
      }
  return l;
}

// Copies what has to be copied into the workspace behind the sums; l.op then names the copies.
int pack(const RingRnnLinearAttention& p, Plan* l, char* at, cudaStream_t s) {
  PackJobs jobs;
  memset(&jobs, 0, sizeof(jobs));
  int n = 0, most = 0;
  for (int x = 0; x < 4; ++x) {
    if (l->packed[x] == 0) continue;
    const int padded = (int)align_up(l->width[x], 8);
    jobs.from[n] = l->op[x];
    jobs.to[n] = at;
    jobs.width[n] = l->width[x];
    jobs.per[n++] = padded / 8;
    most = padded > most ? padded : most;
    l->op[x] = LaOperand{at, (long long)p.T * p.H * padded, (long long)p.H * padded, padded};
    at += l->packed[x];
  }
  if (n == 0) return RINGRNN_OK;
  const size_t need = ((size_t)p.B * p.T * p.H * (most / 8) + 255) / 256, blocks = need < 148 * 16 ? need : 148 * 16;
  for (int x = 0; x < n; ++x) {
    const LaOperand& o = jobs.from[x];
    const long long all = (long long)(reinterpret_cast<uintptr_t>(o.p) / 2) | jobs.width[x] | (p.B > 1 ? o.sb : 0) | (p.T > 1 ? o.st : 0) | (p.H > 1 ? o.sh : 0);
    jobs.vec[x] = reinterpret_cast<uintptr_t>(o.p) % 2 != 0 ? 1 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
    size_t step = blocks * 256;
    const int sizes[3] = {jobs.per[x], p.H, p.T};
    for (int y = 0; y < 3; ++y) jobs.step[x][y] = (int)(step % sizes[y]), step /= sizes[y];
    jobs.step[x][3] = (int)step;
  }
  LaunchScope ls(K_LAYER, s);
  la_pack_kernel<<<dim3((unsigned)blocks, n), 256, 0, s>>>(jobs, p.B, p.T, p.H);
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}

LaLaunch base_launch(const RingRnnLinearAttention& p, const Plan& l) {
  LaLaunch L;
  memset(&L, 0, sizeof(L));
  L.B = p.B; L.T = p.T; L.H = p.H;
  L.segments = l.segments; L.segment_tokens = l.segment_tokens;
  L.log_decay = p.log_decay; L.lengths = p.lengths;
  return L;
}
int check_workspace(const Plan& l, const void* workspace, size_t bytes) {
  if (l.bytes == 0) return RINGRNN_OK;
  return workspace == nullptr || bytes < l.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0 ? RINGRNN_ERR_WORKSPACE : RINGRNN_OK;
}
template <bool STATES>
int launch(const RingRnnLinearAttention& p, const Plan& l, const LaLaunch& L, cudaStream_t s) {
  return l.tensor_cores ? la_tc_launch(L, p.dtype, STATES, s) : plain_launch<STATES>(p.dtype, L, s);
}

}  // namespace
}  // namespace ringrnn

using namespace ringrnn;

extern "C" size_t ringrnn_linear_attention_bytes(const RingRnnLinearAttention* p, const RingRnnStrided* d_out) {
  if (p == nullptr || check_linear(*p, false) != RINGRNN_OK) return (size_t)-1;
  return make_plan(*p, d_out).bytes;
}

extern "C" int ringrnn_linear_attention_fwd(const RingRnnLinearAttention* p, void* out, float* final_state, void* workspace,
                                            size_t workspace_bytes, void* stream) {
  if (p == nullptr) return RINGRNN_ERR_ARG;
  int rc = check_linear(*p, false);
  if (rc != RINGRNN_OK) return rc;
  if (!p->q.data || !p->k.data || !p->v.data || !p->log_decay || !out) return RINGRNN_ERR_ARG;
  Plan l = make_plan(*p, nullptr);
  rc = check_workspace(l, workspace, workspace_bytes);
  if (rc == RINGRNN_OK && l.tensor_cores) rc = earlier_failure();
  if (rc != RINGRNN_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = pack(*p, &l, static_cast<char*>(workspace) + l.sums, s);
  if (rc != RINGRNN_OK) return rc;
  LaLaunch L = base_launch(*p, l);
  float* sums = static_cast<float*>(workspace);
  L.jobs = 1;
  LaJob& j = L.job[0];
  j.q = l.op[0]; j.k = l.op[1]; j.v = l.op[2];
  j.out = out;
  j.inner = p->dk; j.outer = p->dv;
  j.pair_scale = j.row_scale = p->scale;
  j.key_scale = 1.f;
  j.s_in = p->dv; j.s_out = 1;
  if (l.segments > 1) {
    j.fin = sums;
    rc = launch<true>(*p, l, L, s);
    if (rc == RINGRNN_OK) rc = scan_launch(L, p->dk * p->dv, 0, p->initial_state, sums, final_state, s);
    if (rc != RINGRNN_OK) return rc;
    j.init = sums;
    j.fin = nullptr;
  } else {
    j.init = p->initial_state;
    j.fin = final_state;
    j.precise = 1;
  }
  return launch<false>(*p, l, L, s);
}

extern "C" int ringrnn_linear_attention_bwd(const RingRnnLinearAttention* p, const RingRnnStrided* d_out, const float* d_final,
                                            void* dq, void* dk, void* dv, float* d_initial, void* workspace,
                                            size_t workspace_bytes, void* stream) {
  if (p == nullptr || d_out == nullptr) return RINGRNN_ERR_ARG;
  int rc = check_linear(*p, false);
  if (rc != RINGRNN_OK) return rc;
  if (!p->q.data || !p->k.data || !p->v.data || !p->log_decay || !d_out->data || !dq || !dk || !dv) return RINGRNN_ERR_ARG;
  Plan l = make_plan(*p, d_out);
  rc = check_workspace(l, workspace, workspace_bytes);
  if (rc == RINGRNN_OK && l.tensor_cores) rc = earlier_failure();
  if (rc != RINGRNN_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = pack(*p, &l, static_cast<char*>(workspace) + 2 * l.sums, s);
  if (rc != RINGRNN_OK) return rc;
  const LaOperand q = l.op[0], k = l.op[1], v = l.op[2], g = l.op[3];
  LaLaunch L = base_launch(*p, l);
  L.jobs = 3;
  LaJob &jq = L.job[0], &jk = L.job[1], &jv = L.job[2];
  jq.q = g; jq.k = v; jq.v = k; jq.out = dq;
  jk.q = v; jk.k = g; jk.v = q; jk.out = dk;
  jv.q = k; jv.k = q; jv.v = g; jv.out = dv;
  jq.inner = jk.inner = p->dv; jq.outer = jk.outer = p->dk;
  jv.inner = p->dk; jv.outer = p->dv;
  jk.reverse = jv.reverse = 1;
  jq.pair_scale = jk.pair_scale = jv.pair_scale = p->scale;
  jq.row_scale = p->scale; jq.key_scale = 1.f;
  jk.row_scale = jv.row_scale = 1.f; jk.key_scale = jv.key_scale = p->scale;
  jq.s_in = jk.s_in = 1; jq.s_out = jk.s_out = p->dv;  // states are kept as [dk][dv]
  jv.s_in = p->dv; jv.s_out = 1;
  if (l.segments > 1) {
    float* S = static_cast<float*>(workspace);
    float* E = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.sums);
    LaLaunch M = L;
    M.jobs = 2;
    M.job[0] = jq; M.job[0].fin = S;
    M.job[1] = jv; M.job[1].fin = E;
    rc = launch<true>(*p, l, M, s);
    if (rc == RINGRNN_OK) rc = scan_launch(L, p->dk * p->dv, 0, p->initial_state, S, nullptr, s);
    if (rc == RINGRNN_OK) rc = scan_launch(L, p->dk * p->dv, 1, d_final, E, d_initial, s);
    if (rc != RINGRNN_OK) return rc;
    jq.init = S;
    jk.init = jv.init = E;
  } else {
    jq.init = p->initial_state;
    jk.init = jv.init = d_final;
    jv.fin = d_initial;
    // (not by d_initial alone: gradients have the same bits whichever of them are asked for)
    jv.precise = p->initial_state != nullptr || d_initial != nullptr;
  }
  return launch<false>(*p, l, L, s);
}

extern "C" int ringrnn_linear_attention_step(const RingRnnLinearAttention* p, float* state, const unsigned char* active, void* out,
                                             void* stream) {
  if (p == nullptr) return RINGRNN_ERR_ARG;
  const int rc = check_linear(*p, true);
  if (rc != RINGRNN_OK) return rc;
  if (!p->q.data || !p->k.data || !p->v.data || !p->log_decay || !out || !state) return RINGRNN_ERR_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const LaOperand q = operand(p->q), k = operand(p->k), v = operand(p->v);
  return p->dtype == RINGRNN_F32    ? step_launch<float>(*p, q, k, v, state, active, out, s)
         : p->dtype == RINGRNN_BF16 ? step_launch<__nv_bfloat16>(*p, q, k, v, state, active, out, s)
                                    : step_launch<__half>(*p, q, k, v, state, active, out, s);
}
