// Linear attention with decay on tensor cores: bf16, widths up to 128 (padded to 64 or 128), chunks of 128 tokens.
//
// One CTA takes a (job, sequence, head, segment) and goes through its chunks with the state at hand; what a job is stands in
// linear_attention.cuh.  Everything is computed transposed, outer columns on the tensor-memory lanes, so that the state never
// leaves them (c: this chunk of n tokens; t, s: tokens in it; weights as in the forward, "reverse" mirrors them):
//
//   scores   [t x s]      = Q K^T                                     both from shared memory
//   inter^T  [outer x t]  = S^T Q^T        S^T = hi + lo: two bf16 numbers per element, in tensor memory
//   delta^T  [outer x in] = V^T K'         K'_s = g^(n-1-s) k_s = hi + lo, beside each other in shared memory
//   intra^T  [outer x t]  = V^T P^T        P_ts = bf16(scale g^(t-s) scores_ts), s <= t
//   out_t    = row_scale g^(t+1) inter_t + intra_t                    S = g^n S + delta
//
// Precision: the state is fp32 (registers); as an operand it and the weighted keys are two bf16 numbers, 2^-16 of an element, so
// that states passed from call to call keep what fp32 is for; P alone is rounded to bf16, like the outputs.
//
// Roles (20 warps): 0 TMA; 1 MMA issue; 4-7 weight the keys (in place, the rest beside) and the scores; 8-11 write the outputs;
// 12-19 keep the state, half a row each.  The tensor pipe's order per chunk is inter, delta, intra, next scores: while the state
// warps work on delta, it has the last two to do.  Tensor memory: 4 x 128 columns, scores | inter | intra | state, where delta is
// read from the columns that then receive the next operand.
#include <string.h>

#include "linear_attention.cuh"
#include "tc_ptx.cuh"

namespace ringrnn {
namespace {

using namespace tc;

constexpr int C = LA_TC_CHUNK;
constexpr int TILE = C * 128;  // bytes of [128 tokens x 64 columns]
constexpr int LT_THREADS = 640;
constexpr uint32_t TM_SCORES = 0, TM_INTER = 128, TM_INTRA = 256, TM_STATE = 384, TM_COLS = 512;

template <int DI, int DO>
struct LtCfg {
  static constexpr int WIDE = DI > DO ? DI : DO;
  static constexpr int SLOT = TILE * (WIDE / 64);
  static constexpr int SLOTS = WIDE == 128 ? 5 : 8;
  // slots | scores (or, forming sums, a second buffer of keys) | keys' rest.  The last operand may be followed by what it reads
  // in place of rows that nobody uses, so another buffer stands behind the slots.
  static constexpr int P = SLOT * SLOTS, KL = P + 2 * TILE, BARS = KL + TILE * (DI / 64);
  static constexpr int TABLES = BARS + 256;  // 128 row factors, 32 powers
  static constexpr int SMEM = TABLES + 640 + 1024;
};

struct LtParams {
  LaLaunch L;
  int h_step[LA_MAX_JOBS][3], b_step[LA_MAX_JOBS][3];  // 0: a tensor that all heads / sequences share
  alignas(64) CUtensorMap map[LA_MAX_JOBS][3];
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int t, int h, int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(t), "r"(h), "r"(b)
      : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_of(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_of(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
// two fp32 as bf16, and what that leaves of them as bf16
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
  *hi = pack2(a, b);
  *lo = pack2(a - lo_of(*hi), b - hi_of(*hi));
}

template <int DI, int DO, bool STATES>
__global__ void __launch_bounds__(LT_THREADS, 1) la_tc_kernel(const __grid_constant__ LtParams A, volatile int* host_status) {
  using Cfg = LtCfg<DI, DO>;
  constexpr int NS = Cfg::SLOTS, TILES = STATES ? 2 : 3;  // tiles of a chunk: (q,) k, v
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  uint8_t* const mem = raw + (base - smem_u32(raw));
  __shared__ int dead, drain_dead[2];
  __shared__ uint32_t tmem_base;

  const LaLaunch& L = A.L;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ji = (int)(blockIdx.x % L.jobs);
  const LaJob& J = L.job[ji];
  const int at = (int)(blockIdx.x / L.jobs), seg = at % L.segments, bh = at / L.segments, h = bh % L.H, b = bh / L.H;
  const bool rev = J.reverse != 0;
  const int len = la_length(L, b), begin = seg * L.segment_tokens, stop = min(L.T, begin + L.segment_tokens), end = min(len, stop);
  const int chunks = end > begin ? (end - begin + C - 1) / C : 0;
  auto chunk_at = [&](int c) { return begin + (rev ? chunks - 1 - c : c) * C; };

  const uint32_t bars = base + Cfg::BARS;
  auto full = [&](int i) { return bars + 8u * i; };
  auto empty = [&](int i) { return bars + 8u * (NS + i); };
  const uint32_t one = bars + 16u * NS;
  const uint32_t scores_ready = one, keys_ready = one + 8, pairs_ready = one + 16, inter_done = one + 24, delta_ready = one + 32,
                 state_ready = one + 40, out_ready = one + 48, out_free = one + 56, all_done = one + 64;
  float* const row_factor = reinterpret_cast<float*>(mem + Cfg::TABLES);
  float* const powers = row_factor + C;

  if (warp == 0) {
    if (lane == 0) {
      dead = drain_dead[0] = drain_dead[1] = 0;
      for (int i = 0; i < NS; ++i) {
        mbar_init(full(i), 1);
        mbar_init(empty(i), 1);
      }
      mbar_init(scores_ready, 1);
      mbar_init(keys_ready, 128);
      mbar_init(pairs_ready, 128);
      mbar_init(inter_done, 1);
      mbar_init(delta_ready, 1);
      mbar_init(state_ready, 256);
      mbar_init(out_ready, 1);
      mbar_init(out_free, 128);
      mbar_init(all_done, 1);
      fence_mbar_init();
    }
  } else if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_base), TM_COLS);
  }
  const LaDecay g(L.log_decay[h]);
  if (warp == 2) powers[lane] = g.power(rev ? lane : 31 - lane);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tm = tmem_base;
  const WaitCtx w{&dead, nullptr, WAIT_LIMIT_CYCLES, host_status};
  const WaitCtx drain{&drain_dead[warp & 1], nullptr, WAIT_LIMIT_CYCLES, host_status};

  if (warp == 0) {
    // ---- loads: q, k, v of each chunk through a ring of slots
    if (lane == 0) {
      const CUtensorMap* maps = A.map[ji];
      int i = 0, round = 0;
      for (int c = 0; c < chunks; ++c) {
        const int t0 = chunk_at(c);
#pragma unroll
        for (int x = 3 - TILES; x < 3; ++x) {
          if (!mbar_wait(empty(i), (round & 1) ^ 1, w, 101)) break;
          const int blocks = (x == 2 ? DO : DI) / 64;
          mbar_arrive_expect_tx(full(i), blocks * TILE);
          for (int k = 0; k < blocks; ++k)
            tma_load_4d(base + i * Cfg::SLOT + k * TILE, maps + x, full(i), k * 64, t0, h * A.h_step[ji][x], b * A.b_step[ji][x]);
          if (++i == NS) i = 0, ++round;
        }
        if (*static_cast<volatile int*>(&dead)) break;
      }
      // where a wait was abandoned, what is on its way has to land before the block's shared memory goes to another
      if (*static_cast<volatile int*>(&dead)) {
        const int issued = round * NS + i, first = issued > NS ? issued - NS : 0;
        for (int x = first; x < issued; ++x) mbar_wait(full(x % NS), (x / NS) & 1, drain, 102);
      }
    }
  } else if (warp == 1) {
    // ---- MMAs, issued by the whole warp (see umma_ts_warp)
    const uint32_t lead = elect_one();
    constexpr uint32_t ID_SCORES = make_idesc_bf16(128, 128, 0, 0), ID_INTER = make_idesc_bf16(128, 128, 0, 0),
                       ID_DELTA = make_idesc_bf16(128, DI, 1, 1), ID_INTRA = make_idesc_bf16(128, 128, 1, 0);
    auto slot = [&](int tile) { return base + (tile % NS) * Cfg::SLOT; };
    auto loaded = [&](int tile, int code) { mbar_wait(full(tile % NS), (tile / NS) & 1, w, code); };
    // K-major operands: 16 of the 64 columns of a 128-byte row at a time
    auto k_major = [&](uint32_t tile, int ks) { return desc_sw128(desc_lo(tile + (ks >> 2) * TILE + (ks & 3) * 32, 0)); };
    // M/N-major ones: 16 rows, blocks of 64 columns a tile apart
    auto mn_major = [&](uint32_t tile, int ks) { return desc_sw128(desc_lo(tile + ks * 2048, TILE)); };
    auto scores = [&](int c) {
      const uint32_t q = slot(TILES * c), k = slot(TILES * c + 1);
      loaded(TILES * c, 110);
      loaded(TILES * c + 1, 111);
      for (int ks = 0; ks < DI / 16; ++ks) umma_ss_warp(tm + TM_SCORES, k_major(q, ks), k_major(k, ks), ID_SCORES, ks != 0, lead);
      if (lead) umma_commit(scores_ready);
      __syncwarp();
    };
    if (!STATES && chunks > 0) scores(0);
    for (int c = 0; c < chunks; ++c) {
      const int kt = TILES * c + TILES - 2, vt = kt + 1;
      const uint32_t k = slot(kt), v = slot(vt);
      if (!STATES) {
        const int qt = TILES * c;
        mbar_wait(state_ready, c & 1, w, 112);
        if (c > 0) mbar_wait(out_free, (c - 1) & 1, w, 113);
        tcgen05_fence_after();
        // the state's halves stand one behind the other, each as DI / 4 columns of hi and DI / 4 of lo
        for (int part = 0; part < 2; ++part)
          for (int ks = 0; ks < DI / 16; ++ks)
            umma_ts_warp(tm + TM_INTER, tm + TM_STATE + (ks / (DI / 32)) * (DI / 2) + part * (DI / 4) + (ks % (DI / 32)) * 8,
                         k_major(slot(qt), ks), ID_INTER, part + ks != 0, lead);
        if (lead) {
          umma_commit(inter_done);
          umma_commit(empty(qt % NS));
        }
        __syncwarp();
      }
      mbar_wait(keys_ready, c & 1, w, 114);
      loaded(vt, 115);
      // delta overwrites the columns that inter has just read: no order holds between MMAs of different accumulators
      if (!STATES) mbar_wait(inter_done, c & 1, w, 116);
      tcgen05_fence_after();
      const uint32_t rest = base + (STATES && (c & 1) ? Cfg::P : Cfg::KL);
      for (int part = 0; part < 2; ++part)
        for (int ks = 0; ks < C / 16; ++ks)
          umma_ss_warp(tm + TM_STATE, mn_major(v, ks), mn_major(part ? rest : k, ks), ID_DELTA, (STATES && c > 0) || part + ks != 0, lead);
      if (lead) {
        if (STATES) umma_commit(c & 1 ? out_ready : inter_done);  // one barrier for even chunks, one for odd ones
        if (!STATES || c == chunks - 1) umma_commit(delta_ready);
        umma_commit(empty(kt % NS));
        if (STATES) umma_commit(empty(vt % NS));
      }
      __syncwarp();
      if (!STATES) {
        mbar_wait(pairs_ready, c & 1, w, 117);
        tcgen05_fence_after();
        for (int ks = 0; ks < C / 16; ++ks)
          umma_ss_warp(tm + TM_INTRA, mn_major(v, ks), k_major(base + Cfg::P, ks), ID_INTRA, ks != 0, lead);
        if (lead) {
          umma_commit(out_ready);
          umma_commit(empty(vt % NS));
        }
        __syncwarp();
        if (c + 1 < chunks) scores(c + 1);
      }
    }
    // tensor memory is given back below: nothing may still be writing it (at once, unless a wait was abandoned)
    if (lead) umma_commit(all_done);
    mbar_wait(all_done, 0, drain, 118);
  } else if (warp >= 4 && warp < 8) {
    // ---- keys weighted for the state, then scores weighted: a thread has row r of both
    const int r = tid - 128, q = warp - 4;
    if (!STATES) {  // blocks of 32 keys that no token of this warp's rows sees: zero once and for all
      for (int j = 0; j < 4; ++j)
        if (rev ? j < q : j > q)
          for (int i = 0; i < 4; ++i) sts128(base + Cfg::P + (j >> 1) * TILE + sw128_offset(r, (j & 1) * 32 + 8 * i), 0, 0, 0, 0);
    }
    for (int c = 0; c < chunks; ++c) {
      const int t0 = chunk_at(c), n = min(C, end - t0), kt = TILES * c + TILES - 2, vt = kt + 1;
      const uint32_t k = base + (kt % NS) * Cfg::SLOT, rest = base + (STATES && (c & 1) ? Cfg::P : Cfg::KL);
      if (STATES) {
        mbar_wait(full(kt % NS), (kt / NS) & 1, w, 120);
        // the sum of two chunks before has read its keys' rest
        if (c > 1) mbar_wait(c & 1 ? out_ready : inter_done, ((c >> 1) - 1) & 1, w, 121);
      } else {
        mbar_wait(scores_ready, c & 1, w, 122);
        tcgen05_fence_after();
      }
      const int steps = STATES ? (rev ? t0 + r - begin + 1 : end - 1 - t0 - r) : rev ? r + 1 : n - 1 - r;
      const float wk = r < n ? J.key_scale * g.power(steps) : 0.f;
#pragma unroll 4
      for (int i = 0; i < DI / 8; ++i) {
        const uint32_t o = (i >> 3) * TILE + sw128_offset(r, (i & 7) * 8);
        const uint4 x = lds128(k + o);
        uint4 hi, lo;
        split2(lo_of(x.x) * wk, hi_of(x.x) * wk, &hi.x, &lo.x);
        split2(lo_of(x.y) * wk, hi_of(x.y) * wk, &hi.y, &lo.y);
        split2(lo_of(x.z) * wk, hi_of(x.z) * wk, &hi.z, &lo.z);
        split2(lo_of(x.w) * wk, hi_of(x.w) * wk, &hi.w, &lo.w);
        if (r >= n) hi = lo = make_uint4(0, 0, 0, 0);  // whatever stands behind the sequence, a NaN included
        sts128(k + o, hi.x, hi.y, hi.z, hi.w);
        sts128(rest + o, lo.x, lo.y, lo.z, lo.w);
      }
      if (n < C) {
        mbar_wait(full(vt % NS), (vt / NS) & 1, w, 123);
        if (r >= n)
          for (int i = 0; i < DO / 8; ++i) sts128(base + (vt % NS) * Cfg::SLOT + (i >> 3) * TILE + sw128_offset(r, (i & 7) * 8), 0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      mbar_arrive(keys_ready);
      if (!STATES) {
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          if (rev ? j < q : j > q) continue;
          uint32_t x[32];
          tmem_ld32(tm + TM_SCORES + ((uint32_t)(q * 32) << 16) + j * 32, x);
          tmem_ld_wait();
          if (j == q) {
#pragma unroll
            for (int s = 0; s < 32; ++s) {
              const int far = rev ? s - lane : lane - s;
              x[s] = far >= 0 ? __float_as_uint(__uint_as_float(x[s]) * (J.pair_scale * exp2f(g.hi * (float)far))) : 0u;
            }
          } else {
            // g^(distance) as the distance to the block's near end times a power within it: both at most one
            const float f = J.pair_scale * g.power(rev ? 32 * j - r : r - 32 * j - 31);
#pragma unroll
            for (int s = 0; s < 32; s += 4) {
              const float4 p = *reinterpret_cast<const float4*>(powers + s);
              x[s] = __float_as_uint(__uint_as_float(x[s]) * (f * p.x));
              x[s + 1] = __float_as_uint(__uint_as_float(x[s + 1]) * (f * p.y));
              x[s + 2] = __float_as_uint(__uint_as_float(x[s + 2]) * (f * p.z));
              x[s + 3] = __float_as_uint(__uint_as_float(x[s + 3]) * (f * p.w));
            }
          }
          if (n < C)
#pragma unroll
            for (int s = 0; s < 32; ++s)
              if (32 * j + s >= n) x[s] = 0u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t* y = x + 8 * i;
            auto two = [&](int e) { return pack2(__uint_as_float(y[e]), __uint_as_float(y[e + 1])); };
            sts128(base + Cfg::P + (j >> 1) * TILE + sw128_offset(r, (j & 1) * 32 + 8 * i), two(0), two(2), two(4), two(6));
          }
        }
        fence_proxy_async_smem();
        tcgen05_fence_before();
        mbar_arrive(pairs_ready);
      }
    }
  } else if (warp >= 8 && warp < 12) {
    // ---- outputs: a thread has one outer column and the tokens of a chunk; neighbours trade tokens for columns, so that a store
    // is 4 bytes and covers 64 bytes of each of two tokens' rows
    if (!STATES) {
      const int q = warp - 8, o = q * 32 + lane, r = tid - 256;
      const size_t ld = (size_t)L.H * J.outer;
      __nv_bfloat16* const out = static_cast<__nv_bfloat16*>(J.out) + ((size_t)b * L.T * L.H + h) * J.outer;
      const bool pairs = (J.outer & 1) == 0 && (reinterpret_cast<uintptr_t>(J.out) & 3) == 0;
      const bool odd = lane & 1;
      int have = 0;
      for (int c = 0; c < chunks; ++c) {
        const int t0 = chunk_at(c), n = min(C, end - t0), rows = min(C, stop - t0);
        if (n != have) {  // factors of the rows: they change with the number of tokens only in reverse, and then once
          named_bar_sync(1, 128);
          row_factor[r] = r < n ? J.row_scale * g.power(rev ? n - 1 - r : r + 1) : 0.f;
          named_bar_sync(1, 128);
          have = n;
        }
        mbar_wait(out_ready, c & 1, w, 130);
        tcgen05_fence_after();
        if (q * 32 < DO) {
#pragma unroll 1
          for (int i = 0; i < C; i += 16) {
            uint32_t x[16], y[16];
            tmem_ld16(tm + TM_INTER + ((uint32_t)(q * 32) << 16) + i, x);
            tmem_ld16(tm + TM_INTRA + ((uint32_t)(q * 32) << 16) + i, y);
            tmem_ld_wait();
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const float4 f = *reinterpret_cast<const float4*>(row_factor + i + e);
              const float a0 = fmaf(f.x, __uint_as_float(x[e]), __uint_as_float(y[e]));
              const float a1 = fmaf(f.y, __uint_as_float(x[e + 1]), __uint_as_float(y[e + 1]));
              const float a2 = fmaf(f.z, __uint_as_float(x[e + 2]), __uint_as_float(y[e + 2]));
              const float a3 = fmaf(f.w, __uint_as_float(x[e + 3]), __uint_as_float(y[e + 3]));
              v[e / 2] = pack2(a0, a1);
              v[e / 2 + 1] = pack2(a2, a3);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int t = i + 2 * e;  // this thread's column at tokens t (low half) and t + 1
              if (n < C) {
                if (t >= n) v[e] &= 0xffff0000u;
                if (t + 1 >= n) v[e] &= 0x0000ffffu;
              }
              if (pairs) {
                const uint32_t other = __shfl_xor_sync(0xffffffffu, v[e], 1);
                const uint32_t z = odd ? __byte_perm(other, v[e], 0x7632) : __byte_perm(v[e], other, 0x5410);
                const int tt = t + odd;
                if (tt < rows && o < J.outer) *reinterpret_cast<uint32_t*>(out + (size_t)(t0 + tt) * ld + (o & ~1)) = z;
              } else if (o < J.outer) {
                if (t < rows) out[(size_t)(t0 + t) * ld + o] = __ushort_as_bfloat16((unsigned short)v[e]);
                if (t + 1 < rows) out[(size_t)(t0 + t + 1) * ld + o] = __ushort_as_bfloat16((unsigned short)(v[e] >> 16));
              }
            }
          }
        }
        tcgen05_fence_before();
        mbar_arrive(out_free);
      }
      // tokens behind the sequence, beyond its last chunk
      for (int t = begin + chunks * C; t < stop; ++t)
        if (o < J.outer) out[(size_t)t * ld + o] = __float2bfloat16_rn(0.f);
    }
  } else if (warp >= 12) {
    // ---- the state: a thread has half a row of S^T
    constexpr int N = DI / 2;
    const int q = warp & 3, half = (warp - 12) >> 2, o = q * 32 + lane, i0 = half * N;
    const uint32_t mine = tm + TM_STATE + ((uint32_t)(q * 32) << 16) + half * N;
    const size_t mat = (size_t)at * J.inner * J.outer;
    float S[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      S[i] = !STATES && J.init != nullptr && o < J.outer && i0 + i < J.inner ? J.init[mat + (size_t)(i0 + i) * J.s_in + (size_t)o * J.s_out] : 0.f;
    auto publish = [&]() {
#pragma unroll
      for (int i = 0; i < N; i += 16) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) split2(S[i + 2 * e], S[i + 2 * e + 1], hi + e, lo + e);
        tmem_st8(mine + i / 2, hi);
        tmem_st8(mine + N / 2 + i / 2, lo);
      }
      tmem_st_wait();
      tcgen05_fence_before();
      mbar_arrive(state_ready);
    };
    if (!STATES && chunks > 0) publish();
    if (STATES) {
      if (chunks > 0) {
        mbar_wait(delta_ready, 0, w, 140);
        tcgen05_fence_after();
#pragma unroll
        for (int i = 0; i < N; i += 16) {
          uint32_t x[16];
          tmem_ld16(mine + i, x);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) S[i + e] = __uint_as_float(x[e]);
        }
      }
    } else {
      const LaFactor whole(L.log_decay[h], C);
      for (int c = 0; c < chunks; ++c) {
        const int n = min(C, end - chunk_at(c));
        const LaFactor gn = n == C ? whole : LaFactor(L.log_decay[h], n);
        mbar_wait(delta_ready, c & 1, w, 141);
        tcgen05_fence_after();
#pragma unroll
        for (int i = 0; i < N; i += 16) {
          uint32_t x[16];
          tmem_ld16(mine + i, x);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) S[i + e] = gn.times(S[i + e], __uint_as_float(x[e]));
        }
        if (c + 1 < chunks) publish();
      }
    }
    if (J.fin != nullptr && o < J.outer) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i0 + i < J.inner) J.fin[mat + (size_t)(i0 + i) * J.s_in + (size_t)o * J.s_out] = S[i];
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tm, TM_COLS);
}

bool make_map(CUtensorMap* m, const LaOperand& o, int width, int B, int T, int H, int* h_step, int* b_step) {
  *h_step = H > 1 && o.sh != 0;
  *b_step = B > 1 && o.sb != 0;
  const uint64_t dims[4] = {(uint64_t)width, (uint64_t)T, (uint64_t)(*h_step ? H : 1), (uint64_t)(*b_step ? B : 1)};
  // strides of dimensions of one entry are not used: any valid one
  const uint64_t strides[3] = {(uint64_t)(T > 1 ? o.st * 2 : 16), (uint64_t)(*h_step ? o.sh * 2 : 16), (uint64_t)(*b_step ? o.sb * 2 : 16)};
  const uint32_t box[4] = {64, C, 1, 1};
  return make_tmap_bf16_4d(m, o.p, dims, strides, box);
}

template <int DI, int DO, bool STATES>
int launch(const LtParams& P, cudaStream_t s) {
  using Cfg = LtCfg<DI, DO>;
  volatile int* host = nullptr;
  const int rc = host_status_word(&host);
  if (rc != RINGRNN_OK) return rc;
  RINGRNN_CUDA_TRY(cudaFuncSetAttribute(la_tc_kernel<DI, DO, STATES>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
  LaunchScope ls(K_LAYER, s);
  la_tc_kernel<DI, DO, STATES><<<P.L.B * P.L.H * P.L.segments * P.L.jobs, LT_THREADS, Cfg::SMEM, s>>>(P, host);
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}

}  // namespace

bool la_tc_operand_ok(const LaOperand& o, int B, int T, int H) {
  const bool t = T == 1 || (o.st > 0 && o.st % 8 == 0 && o.st < (1LL << 38));
  const bool h = H == 1 || (o.sh >= 0 && o.sh % 8 == 0 && o.sh < (1LL << 38));
  const bool b = B == 1 || (o.sb >= 0 && o.sb % 8 == 0 && o.sb < (1LL << 38));
  return t && h && b && (reinterpret_cast<uintptr_t>(o.p) & 15) == 0;
}

int la_tc_launch(const LaLaunch& L, bool states_only, cudaStream_t s) {
  // jobs of one shape together
  for (int shape = 0; shape < 4; ++shape) {
    const int di = shape & 1 ? 128 : 64, d_o = shape & 2 ? 128 : 64;
    LtParams P;
    memset(&P, 0, sizeof(P));
    P.L = L;
    P.L.jobs = 0;
    for (int j = 0; j < L.jobs; ++j) {
      const LaJob& J = L.job[j];
      if ((J.inner <= 64 ? 64 : 128) != di || (J.outer <= 64 ? 64 : 128) != d_o) continue;
      const int to = P.L.jobs++;
      P.L.job[to] = J;
      const LaOperand* ops[3] = {&J.q, &J.k, &J.v};
      for (int x = states_only ? 1 : 0; x < 3; ++x)
        if (!make_map(&P.map[to][x], *ops[x], x == 2 ? J.outer : J.inner, L.B, L.T, L.H, &P.h_step[to][x], &P.b_step[to][x]))
          return RINGRNN_ERR_CUDA;
    }
    if (P.L.jobs == 0) continue;
    int rc;
    switch (shape * 2 + (states_only ? 1 : 0)) {
      case 0: rc = launch<64, 64, false>(P, s); break;
      case 1: rc = launch<64, 64, true>(P, s); break;
      case 2: rc = launch<128, 64, false>(P, s); break;
      case 3: rc = launch<128, 64, true>(P, s); break;
      case 4: rc = launch<64, 128, false>(P, s); break;
      case 5: rc = launch<64, 128, true>(P, s); break;
      case 6: rc = launch<128, 128, false>(P, s); break;
      default: rc = launch<128, 128, true>(P, s); break;
    }
    if (rc != RINGRNN_OK) return rc;
  }
  return RINGRNN_OK;
}

}  // namespace ringrnn
