// Linear attention with decay on tensor cores: bf16, widths up to 128 (padded to 64 or 128), chunks of 128 tokens.
//
// One CTA takes a (job, sequence, head, segment) and goes through its chunks with the state at hand; what a job is stands in
// linear_attention.cuh.  Everything is computed transposed, outer columns on the tensor-memory lanes, so that the state never
// leaves them (c: this chunk of n tokens; t, s: tokens in it; weights as in the forward, "reverse" mirrors them):
//
//   scores   [t x s]      = Q K^T                                     both from shared memory
//   inter^T  [outer x t]  = bf16(S^T) Q^T  S in tensor memory
//   intra^T  [outer x t]  = V^T P^T        P_ts = bf16(scale g^(t-s) scores_ts), s <= t
//   delta^T  [outer x in] = V^T K'         K'_s = g^(n-1-s) k_s = hi + lo, two bf16 numbers, beside each other in shared memory
//   out_t    = row_scale g^(t+1) inter_t + intra_t                    S = g^n S + delta
//
// Precision: the state is fp32 (registers) and what is added to it keeps sixteen bits, so that states passed from call to call
// and their gradients are good for what fp32 is for: 2e-6 of their size, where keys rounded to bf16 would leave 2e-3.  Where it
// only goes into bf16 outputs the state is rounded to bf16, like P: next to the outputs' own rounding that costs a factor of 1.4
// in their error, a second product for the rest of the state would make it 1.1 and take 512 of a chunk's cycles.
//
// Roles (28 warps): 0 TMA loads; 1 MMA issue; 2 TMA stores; 4-11 weight the scores and the keys (in place, the rest where q was);
// 12-19 bring the outputs to shared memory (where P was); 20-27 keep the state, half a row each.  A scheduler has two warps of a
// role at a time, each at its own place in the code, and waits for instructions more than for anything else
// once that outgrows the instruction cache (13 cycles for each instruction, with everything unrolled: 96 us instead of 82 for
// 8 x 2048 tokens of 16 heads): loops stay rolled, pairs of fp32 are computed as such, and what only a partial chunk needs is done
// apart.  The tensor pipe's order is inter and intra of a chunk, the next one's scores, delta: the weights of the next
// scores and keys are then formed while delta and the state follow.  Tensor memory: 4 x 128 columns, scores | inter | intra | state, where delta
// is read from the columns that then receive the next operand.
#include <string.h>

#include "linear_attention.cuh"
#include "tc_ptx.cuh"

namespace ringrnn {
namespace {

using namespace tc;

constexpr int C = LA_TC_CHUNK;
constexpr int TILE = C * 128;  // bytes of [128 tokens x 64 columns]
constexpr int LT_THREADS = 896;
// registers of warps 0-3, 4-11, 12-19, 20-27 (setmaxnreg): no more than the block is launched with
constexpr int REGS_ISSUE = 32, REGS_WEIGHT = 72, REGS_OUT = 64, REGS_STATE = 96;
static_assert((4 * REGS_ISSUE + 8 * REGS_WEIGHT + 8 * REGS_OUT + 8 * REGS_STATE) * 32 <= 65536 / LT_THREADS / 8 * 8 * LT_THREADS, "registers");
constexpr uint32_t TM_SCORES = 0, TM_INTER = 128, TM_INTRA = 256, TM_STATE = 384, TM_COLS = 512;

template <int DI, int DO>
struct LtCfg {
  static constexpr int WIDE = DI > DO ? DI : DO;
  static constexpr int SLOT = TILE * (WIDE / 64);
  static constexpr int SLOTS = WIDE == 128 ? 6 : 12;  // two chunks' q, k and v or four's: what it takes to keep the memory busy
  // slots | P, then the outputs on their way.  The last v may be followed by what the MMAs read in place of rows that nobody uses,
  // so another buffer stands behind the slots.
  static constexpr int P = SLOT * SLOTS, BARS = P + 2 * TILE;
  static constexpr int TABLES = BARS + (2 * SLOTS + 12) * 8 + 32;  // 128 row factors, 32 powers
  static_assert(TABLES % 16 == 0, "alignment");
  static constexpr int FLAGS = TABLES + 640;
  static constexpr int SMEM = FLAGS + 16;
  static_assert(SMEM <= 232448, "shared memory of a block");
};

struct LtParams {
  LaLaunch L;
  int h_step[LA_MAX_JOBS][3], b_step[LA_MAX_JOBS][3];  // 0: a tensor that all heads / sequences share
  int store[LA_MAX_JOBS];  // out can be written by TMA
  alignas(64) CUtensorMap map[LA_MAX_JOBS][4];  // q, k, v, out
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int t, int h, int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(t), "r"(h), "r"(b)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, uint32_t src, int x, int t, int h, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(src), "r"(x), "r"(t), "r"(h), "r"(b)
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
__device__ __forceinline__ uint32_t pack2(f32x2 v) {
  float a, b;
  upk2(v, a, b);
  return pack2(a, b);
}
template <int REGS>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }

template <int DI, int DO, bool STATES>
__global__ void __launch_bounds__(LT_THREADS, 1) la_tc_kernel(const __grid_constant__ LtParams A, volatile int* host_status) {
  using Cfg = LtCfg<DI, DO>;
  // Tiles of a chunk: (q,) k, v.  What the weighted keys leave goes where q was; forming sums, to P and the last slot in turn.
  constexpr int NS = Cfg::SLOTS - (STATES ? 1 : 0), TILES = STATES ? 2 : 3;
  // (nothing else is in shared memory, so that this starts on a boundary of the swizzle's period; there is no room to move it)
  extern __shared__ __align__(1024) uint8_t mem[];
  const uint32_t base = smem_u32(mem);
  if ((base & 1023u) != 0) {
    if (threadIdx.x == 0) report_abandoned(WaitCtx{nullptr, nullptr, 0, host_status}, 100);
    return;
  }
  int* const flags = reinterpret_cast<int*>(mem + Cfg::FLAGS);  // dead; one each for the two roles that drain; tensor memory

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
                 state_ready = one + 40, out_ready = one + 48, out_free = one + 56, all_done = one + 64, tail_ready = one + 72, staged = one + 80, stored = one + 88;
  // A barrier's waiter can only tell one phase from the next.  Two barriers in turn where the other side can be a chunk ahead.
  auto sum_keys_ready = [&](int c) { return c & 1 ? pairs_ready : keys_ready; };  // forming sums: keys two chunks ahead at most
  auto sum_done = [&](int c) { return c & 1 ? out_ready : inter_done; };          // and what they were added to
  float* const row_factor = reinterpret_cast<float*>(mem + Cfg::TABLES);
  float* const powers = row_factor + C;

  if (warp == 0) {
    if (lane == 0) {
      flags[0] = flags[1] = flags[2] = 0;
      for (int i = 0; i < NS; ++i) {
        mbar_init(full(i), 1);
        mbar_init(empty(i), 1);
      }
      mbar_init(scores_ready, 1);
      mbar_init(keys_ready, 256);
      mbar_init(pairs_ready, 256);
      mbar_init(inter_done, 1);
      mbar_init(delta_ready, 1);
      mbar_init(state_ready, 256);
      mbar_init(out_ready, 1);
      mbar_init(out_free, 256);
      mbar_init(all_done, 1);
      mbar_init(tail_ready, 256);
      mbar_init(staged, 256);
      mbar_init(stored, 1);
      fence_mbar_init();
    }
  } else if (warp == 1) {
    tmem_alloc(base + Cfg::FLAGS + 12, TM_COLS);
  }
  const LaDecay g(L.log_decay[h]);
  if (warp == 2) powers[lane] = g.power(rev ? lane : 31 - lane);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tm = *reinterpret_cast<volatile uint32_t*>(flags + 3);
  const WaitCtx w{flags, nullptr, WAIT_LIMIT_CYCLES, host_status};
  const WaitCtx drain{flags + 1 + (warp & 1), nullptr, WAIT_LIMIT_CYCLES, host_status};

  if (warp < 4) regs_down<REGS_ISSUE>();
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
        if (*static_cast<volatile int*>(flags)) break;
      }
      // where a wait was abandoned, what is on its way has to land before the block's shared memory goes to another
      if (*static_cast<volatile int*>(flags)) {
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
    // inter(c - 1), intra(c - 1), scores(c), delta(c - 1); loops are left rolled where their instructions keep up (see above)
#pragma unroll 1
    for (int i = STATES ? 1 : 0; i <= chunks; ++i) {
      const int c = i - 1, kt = TILES * c + TILES - 2, vt = kt + 1;  // of the chunk before
      if (!STATES && i > 0) {
        mbar_wait(state_ready, c & 1, w, 112);
        if (c > 0) mbar_wait(out_free, (c - 1) & 1, w, 113);
        tcgen05_fence_after();
        // the state's halves stand one behind the other, DI / 4 of DI / 2 columns each
#pragma unroll 2
        for (int ks = 0; ks < DI / 16; ++ks)
          umma_ts_warp(tm + TM_INTER, tm + TM_STATE + (ks / (DI / 32)) * (DI / 2) + (ks % (DI / 32)) * 8, k_major(slot(kt - 1), ks), ID_INTER,
                       ks != 0, lead);
        if (lead) umma_commit(inter_done);
        __syncwarp();
        loaded(vt, 115);
        mbar_wait(pairs_ready, c & 1, w, 117);
        tcgen05_fence_after();
#pragma unroll 2
        for (int ks = 0; ks < C / 16; ++ks)
          umma_ss_warp(tm + TM_INTRA, mn_major(slot(vt), ks), k_major(base + Cfg::P, ks), ID_INTRA, ks != 0, lead);
        if (lead) umma_commit(out_ready);
        __syncwarp();
      }
      if (!STATES && i < chunks) {
        const uint32_t q = slot(TILES * i), k = slot(TILES * i + 1);
        loaded(TILES * i, 110);
        loaded(TILES * i + 1, 111);
        if (chunk_at(i) + C > end) mbar_wait(tail_ready, 0, w, 119);
        tcgen05_fence_after();
#pragma unroll 2
        for (int ks = 0; ks < DI / 16; ++ks) umma_ss_warp(tm + TM_SCORES, k_major(q, ks), k_major(k, ks), ID_SCORES, ks != 0, lead);
        if (lead) umma_commit(scores_ready);
        __syncwarp();
      }
      if (i > 0) {
        if (STATES) {
          loaded(vt, 115);
          mbar_wait(sum_keys_ready(c), (c >> 1) & 1, w, 114);
        } else {
          mbar_wait(keys_ready, c & 1, w, 114);
          // delta overwrites the columns that inter has read: no order holds between MMAs of different accumulators
          mbar_wait(inter_done, c & 1, w, 116);
        }
        tcgen05_fence_after();
        const uint32_t k = slot(kt), v = slot(vt), rest = STATES ? base + (c & 1 ? NS * Cfg::SLOT : Cfg::P) : slot(kt - 1);
#pragma unroll 2
        for (int x = 0; x < C / 8; ++x)
          umma_ss_warp(tm + TM_STATE, mn_major(v, x >> 1), mn_major(x & 1 ? rest : k, x >> 1), ID_DELTA, (STATES && c > 0) || x != 0, lead);
        if (lead) {
          if (STATES) umma_commit(sum_done(c));
          if (!STATES || c == chunks - 1) umma_commit(delta_ready);
          umma_commit(empty(kt % NS));
          umma_commit(empty(vt % NS));
          if (!STATES) umma_commit(empty((kt - 1) % NS));
        }
        __syncwarp();
      }
    }
    // tensor memory is given back below: nothing may still be writing it (at once, unless a wait was abandoned)
    if (lead) umma_commit(all_done);
    mbar_wait(all_done, 0, drain, 118);
  } else if (warp == 2) {
    // ---- stores: outputs from where P was
    if (!STATES && lane == 0) {
      for (int c = 0; c < chunks; ++c) {
        if (!mbar_wait(staged, c & 1, w, 150)) break;
        if (A.store[ji]) {
          for (int k = 0; k < DO / 64; ++k) tma_store_4d(A.map[ji] + 3, base + Cfg::P + k * TILE, k * 64, chunk_at(c), h, b);
          bulk_commit();
          bulk_wait_read<0>();
        }
        mbar_arrive(stored);
      }
      bulk_wait_all<0>();
    }
  } else if (warp >= 4 && warp < 12) {
    // ---- keys weighted for the state, then scores weighted: a thread has half of row r of both
    regs_down<REGS_WEIGHT>();
    const int q = warp & 3, half = (warp - 4) >> 2, r = q * 32 + lane;
    // a block of 32 keys is seen by all, some or none of this warp's 32 tokens: j to q's one side, j == q, the other side
    auto pair_at = [&](int j) { return base + Cfg::P + (j >> 1) * TILE; };
    const int col = half * 16;  // of each block
    // Weights of scores, the same in every chunk.  The diagonal block's stand in registers.  Another block's are the power up to
    // its near end, a factor per token (32 tokens more: times g^32), times one within the block: all at most one.
    f32x2 diagonal[8];
    const float near = J.pair_scale * g.power(rev ? 32 - lane : lane + 1), g32 = g.power(32);
#pragma unroll
    for (int s = 0; s < 16; s += 2) {
      const int far = rev ? col + s - lane : lane - col - s, far1 = rev ? far + 1 : far - 1;
      diagonal[s / 2] = pk2(far >= 0 ? J.pair_scale * g.power(far) : 0.f, far1 >= 0 ? J.pair_scale * g.power(far1) : 0.f);
    }
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
      const int t0 = chunk_at(c), n = min(C, end - t0), kt = TILES * c + TILES - 2, vt = kt + 1;
      const uint32_t k = base + (kt % NS) * Cfg::SLOT, rest = base + (STATES ? (c & 1 ? NS * Cfg::SLOT : Cfg::P) : ((kt - 1) % NS) * Cfg::SLOT);
      const int steps = STATES ? (rev ? t0 + r - begin + 1 : end - 1 - t0 - r) : rev ? r + 1 : n - 1 - r;
      const float wk = r < n ? J.key_scale * g.power(steps) : 0.f;
      if (n < C) {
        // what stands behind the sequence, a NaN included, becomes zero before anybody reads it
        mbar_wait(full(kt % NS), (kt / NS) & 1, w, 120);
        mbar_wait(full(vt % NS), (vt / NS) & 1, w, 123);
        if (r >= n) {
          const uint32_t v = base + (vt % NS) * Cfg::SLOT;
          for (int i = half; i < DI / 8; i += 2) sts128(k + (i >> 3) * TILE + sw128_offset(r, (i & 7) * 8), 0, 0, 0, 0);
          for (int i = half; i < DO / 8; i += 2) sts128(v + (i >> 3) * TILE + sw128_offset(r, (i & 7) * 8), 0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        if (!STATES) mbar_arrive(tail_ready);
        else named_bar_sync(2, 256);
      }
      if (STATES) {
        mbar_wait(full(kt % NS), (kt / NS) & 1, w, 120);
        // the sum of two chunks before has read its keys' rest
        if (c > 1) mbar_wait(sum_done(c), ((c >> 1) - 1) & 1, w, 121);
      } else {
        mbar_wait(scores_ready, c & 1, w, 122);
        tcgen05_fence_after();
        if (c > 0) mbar_wait(stored, (c - 1) & 1, w, 124);
      }
      if (!STATES) {
        const uint32_t from = tm + TM_SCORES + ((uint32_t)(q * 32) << 16) + col;
        auto put = [&](int j, const f32x2* y) {
#pragma unroll
          for (int e = 0; e < 8; e += 4)
            sts128(pair_at(j) + sw128_offset(r, (j & 1) * 32 + col + 2 * e), pack2(y[e]), pack2(y[e + 1]), pack2(y[e + 2]), pack2(y[e + 3]));
        };
        uint32_t x[16];
        f32x2 y[8];
        tmem_ld16(from + q * 32, x);
#pragma unroll 1
        for (int j = rev ? q - 1 : q + 1; rev ? j >= 0 : j < 4; j += rev ? -1 : 1)  // blocks that none of this warp's tokens see
          for (int e = 0; e < 16; e += 8) sts128(pair_at(j) + sw128_offset(r, (j & 1) * 32 + col + e), 0, 0, 0, 0);
        tmem_ld_wait();
#pragma unroll
        for (int s = 0; s < 8; ++s) y[s] = mul2(pk2u(x[2 * s], x[2 * s + 1]), diagonal[s]);
        put(q, y);
        float f = near;
#pragma unroll 1
        for (int j = rev ? q + 1 : q - 1; rev ? j < 4 : j >= 0; j += rev ? 1 : -1) {
          tmem_ld16(from + j * 32, x);
          const f32x2 f2 = pk2(f, f);
          f *= g32;
#pragma unroll
          for (int s = 0; s < 8; s += 2) {
            const float4 p = *reinterpret_cast<const float4*>(powers + col + 2 * s);
            y[s] = mul2(f2, pk2(p.x, p.y));
            y[s + 1] = mul2(f2, pk2(p.z, p.w));
          }
          tmem_ld_wait();
#pragma unroll
          for (int s = 0; s < 8; ++s) y[s] = mul2(pk2u(x[2 * s], x[2 * s + 1]), y[s]);
          put(j, y);
        }
        fence_proxy_async_smem();
        tcgen05_fence_before();
        mbar_arrive(pairs_ready);
      }
      if (!STATES) mbar_wait(inter_done, c & 1, w, 125);  // q has been read for the last time: the keys' rest goes there
      // k w = hi + lo with w = w_hi + w_lo, all bf16: hi = k w_hi rounded, what that leaves is exact in bf16 (eight bits of the
      // sixteen), lo = k w_lo + that, rounded.  Three instructions for two elements, where the way through fp32 takes eight.
      const __nv_bfloat16 w_hi = __float2bfloat16_rn(wk);
      const __nv_bfloat162 wh = __bfloat162bfloat162(w_hi), wl = __bfloat162bfloat162(__float2bfloat16_rn(wk - __bfloat162float(w_hi)));
#pragma unroll 1
      for (int i = half * (DI / 16); i < (half + 1) * (DI / 16); i += 2) {
        const uint32_t o0 = (i >> 3) * TILE + sw128_offset(r, (i & 7) * 8), o1 = (i >> 3) * TILE + sw128_offset(r, (i & 7) * 8 + 8);
        const uint4 x0 = lds128(k + o0), x1 = lds128(k + o1);
        const uint32_t x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const __nv_bfloat162 y = *reinterpret_cast<const __nv_bfloat162*>(x + e), h2 = __hmul2_rn(y, wh);
          const __nv_bfloat162 l2 = __hfma2(y, wl, __hfma2(y, wh, __hneg2(h2)));
          hi[e] = *reinterpret_cast<const uint32_t*>(&h2);
          lo[e] = *reinterpret_cast<const uint32_t*>(&l2);
        }
        sts128(k + o0, hi[0], hi[1], hi[2], hi[3]);
        sts128(k + o1, hi[4], hi[5], hi[6], hi[7]);
        sts128(rest + o0, lo[0], lo[1], lo[2], lo[3]);
        sts128(rest + o1, lo[4], lo[5], lo[6], lo[7]);
      }
      fence_proxy_async_smem();
      mbar_arrive(STATES ? sum_keys_ready(c) : keys_ready);
    }
  } else if (warp >= 12 && warp < 20) {
    // ---- outputs: fragments of 32 columns by 16 tokens, turned by the matrix stores: [token][column] tiles where P was;
    // each of two warps with the same columns takes half of the tokens
    regs_down<REGS_OUT>();
    if (!STATES) {
      const int q = warp & 3, half = (warp - 12) >> 2, r = tid - 384, i0 = half * (C / 2);
      const size_t ld = (size_t)L.H * J.outer;
      __nv_bfloat16* const out = static_cast<__nv_bfloat16*>(J.out) + ((size_t)b * L.T * L.H + h) * J.outer;
      const uint32_t from = tm + ((uint32_t)(q * 32) << 16);
      const uint32_t put = base + Cfg::P + (q >> 1) * TILE + sw128_offset(lane & 7, (q & 1) * 32 + (lane >> 3) * 8);
      int have = 0;
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        const int t0 = chunk_at(c), n = min(C, end - t0);
        if (n != have) {  // factors of the rows: they change with the number of tokens only in reverse, and then once
          named_bar_sync(1, 256);
          if (r < C) row_factor[r] = r < n ? J.row_scale * g.power(rev ? n - 1 - r : r + 1) : 0.f;
          named_bar_sync(1, 256);
          have = n;
        }
        mbar_wait(out_ready, c & 1, w, 130);
        tcgen05_fence_after();
        if (q * 32 < DO) {
          uint32_t x[16], y[16];
          auto fetch = [&](int i) {
            tmem_ld_frag2(from + TM_INTER + i, x);
            tmem_ld_frag2(from + (16u << 16) + TM_INTER + i, x + 8);
            tmem_ld_frag2(from + TM_INTRA + i, y);
            tmem_ld_frag2(from + (16u << 16) + TM_INTRA + i, y + 8);
          };
          fetch(i0);
#pragma unroll 1
          for (int i = i0; i < i0 + C / 2; i += 16) {
            const f32x2 f0 = *reinterpret_cast<const f32x2*>(row_factor + i + 2 * (lane & 3)),
                        f1 = *reinterpret_cast<const f32x2*>(row_factor + i + 8 + 2 * (lane & 3));
            tmem_ld_wait();
            uint32_t v[8];  // of 16 columns (half), 8 tokens, 8 columns: half * 4 + tokens * 2 + columns
#pragma unroll
            for (int e = 0; e < 8; ++e)
              v[e] = pack2(fma2((e >> 1) & 1 ? f1 : f0, pk2u(x[2 * e], x[2 * e + 1]), pk2u(y[2 * e], y[2 * e + 1])));
            if (i + 16 < i0 + C / 2) {
              fetch(i + 16);
            } else {  // all of it is in registers
              tcgen05_fence_before();
              mbar_arrive(out_free);
            }
            if (i + 16 > n) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int t = i + ((e >> 1) & 1) * 8 + 2 * (lane & 3);
                if (t >= n) v[e] &= 0xffff0000u;
                if (t + 1 >= n) v[e] &= 0x0000ffffu;
              }
            }
            stmatrix_x4_trans(put + i * 128, v[0], v[1], v[4], v[5]);
            stmatrix_x4_trans(put + i * 128 + 1024, v[2], v[3], v[6], v[7]);
          }
        } else {
          mbar_arrive(out_free);
        }
        if (!A.store[ji]) {  // widths and addresses that TMA does not take: element by element
          named_bar_sync(1, 256);
          const int o = r & 127;
#pragma unroll 1
          for (int t = r >> 7; t < C && t0 + t < stop; t += 2)
            if (o < J.outer)
              out[(size_t)(t0 + t) * ld + o] = *reinterpret_cast<const __nv_bfloat16*>(mem + Cfg::P + (o >> 6) * TILE + sw128_offset(t, o & 63));
        }
        fence_proxy_async_smem();
        mbar_arrive(staged);
      }
      // tokens behind the sequence, beyond its last chunk
#pragma unroll 1
      for (int t = begin + chunks * C + (r >> 7); t < stop; t += 2)
        if ((r & 127) < J.outer) out[(size_t)t * ld + (r & 127)] = __float2bfloat16_rn(0.f);
    }
  } else if (warp >= 20) {
    // ---- the state: a thread has half a row of S^T
    regs_up<REGS_STATE>();
    constexpr int N = DI / 2;
    const int q = warp & 3, half = (warp - 20) >> 2, o = q * 32 + lane, i0 = half * N;
    const uint32_t mine = tm + TM_STATE + ((uint32_t)(q * 32) << 16) + half * N;
    const size_t mat = (size_t)at * J.inner * J.outer;
    f32x2 S[N / 2];
    {
      const float* from = J.init + mat + (size_t)o * J.s_out;
      const bool given = !STATES && J.init != nullptr && o < J.outer;
#pragma unroll
      for (int i = 0; i < N; i += 2)
        S[i / 2] = pk2(given && i0 + i < J.inner ? from[(size_t)(i0 + i) * J.s_in] : 0.f,
                       given && i0 + i + 1 < J.inner ? from[(size_t)(i0 + i + 1) * J.s_in] : 0.f);
    }
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
          for (int e = 0; e < 8; ++e) S[i / 2 + e] = pk2u(x[2 * e], x[2 * e + 1]);
        }
      }
    } else {
      const int part = (end - begin) % C;  // tokens of the one chunk that is not whole, 0: there is none
      const LaFactor whole(L.log_decay[h], C), rest(L.log_decay[h], part);
#pragma unroll 1
      for (int c = 0; c <= chunks && chunks > 0; ++c) {
        if (c > 0) {
          const bool all = part == 0 || chunk_at(c - 1) + C <= end;
          const f32x2 g_hi = all ? pk2(whole.hi, whole.hi) : pk2(rest.hi, rest.hi), g_lo = all ? pk2(whole.lo, whole.lo) : pk2(rest.lo, rest.lo);
          mbar_wait(delta_ready, (c - 1) & 1, w, 141);
          tcgen05_fence_after();
#pragma unroll
          for (int i = 0; i < N; i += 16) {
            uint32_t y[16];
            tmem_ld16(mine + i, y);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; ++e) S[i / 2 + e] = fma2(g_hi, S[i / 2 + e], fma2(g_lo, S[i / 2 + e], pk2u(y[2 * e], y[2 * e + 1])));
          }
        }
        if (c < chunks) {  // the next operand
#pragma unroll
          for (int i = 0; i < N; i += 16) {
            uint32_t x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = pack2(S[i / 2 + e]);
            tmem_st8(mine + i / 2, x);
          }
          tmem_st_wait();
          tcgen05_fence_before();
          mbar_arrive(state_ready);
        }
      }
    }
    if (J.fin != nullptr && o < J.outer) {
      float* to = J.fin + mat + (size_t)o * J.s_out;
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        float x, y;
        upk2(S[i / 2], x, y);
        if (i0 + i < J.inner) to[(size_t)(i0 + i) * J.s_in] = x;
        if (i0 + i + 1 < J.inner) to[(size_t)(i0 + i + 1) * J.s_in] = y;
      }
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
      int unused[2];
      const LaOperand out{J.out, (long long)L.T * L.H * J.outer, (long long)L.H * J.outer, J.outer};
      P.store[to] = !states_only && J.outer % 8 == 0 && (reinterpret_cast<uintptr_t>(J.out) & 15) == 0;
      if (P.store[to] && !make_map(&P.map[to][3], out, J.outer, L.B, L.T, L.H, unused, unused + 1)) return RINGRNN_ERR_CUDA;
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
