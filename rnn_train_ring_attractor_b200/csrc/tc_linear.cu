// Linear attention with decay on tensor cores: bf16 or fp16, widths up to 128 (padded to 64 or 128), chunks of 128 tokens.
//
// One CTA takes a (job, sequence, head, segment) and goes through its chunks with the state at hand; what a job is stands in
// linear_attention.cuh.  A chunk of n tokens (t, s: tokens in it; weights as in the forward, "reverse" mirrors them):
//
//   scores [t x s]      = Q K^T            both from shared memory
//   inter  [t x outer]  = Q b(S)           S copied to shared memory; its rows are then scaled by row_scale g^(t+1), in place
//   out    [t x outer] += P V              P_ts = b(scale g^(t-s) scores_ts), s <= t, in tensor memory where the scores were
//   delta  [in x outer] = K'^T V           K'_s = g^(n-1-s) k_s = hi + lo, two numbers, transposed into tensor memory (+ the rest)
//   S = g^n S + delta                      b(): rounded to the tensors' type
//
// Precision (of bf16): the state is fp32, in registers, and chunks are added to it there.  hi and lo keep sixteen bits of what is
// added, which is plenty where a state only goes into bf16 outputs (it is rounded to bf16 for those, like P: next to the outputs' own
// rounding that costs a factor of 1.4 in their error; a second product for the rest of the state would make it 1.1 and take 512
// of a chunk's cycles).  A state that a caller sees, or that sums of segments make, is good for what fp32 is for: there a third part of
// K' follows, so that all 24 bits of the product count.  Measured against 64 bits: 6e-7 of the state's size instead of 3.8e-6,
// for 65 us instead of 58 (forward of 8 x 2048 x 16 heads of 128; nothing at widths of 64 or where segments are summed).
// fp16 has three bits more and little range: what is rounded to it is multiplied by a power of two first that brings a chunk's largest
// number just below 2^15, and its product divided by it again.  The state's largest element; that of the keys times their weights, by
// way of fp32 (hi and lo keep 22 bits, and what is 2^-17 of the largest or less a share of 2^-39 of it); for scores their bound, the width
// times the largest elements of rows and keys.  Two passes over the operands in shared memory find those.  Forward and gradients of
// 8 x 2048 x 16 heads of 128: 64 and 160 us, without the powers of keys and scores 58 and 143, but small numbers lost their bits (keys
// of 1e-3: state off by 5e-5; gradients of 1e-5: by 2e-2) and scores from 65520 on were infinite.
//
// What bounds it: at widths of 128 the memory's share (a chunk is 128 KB, 5500 cycles of an SM's share at 6.5 TB/s when all SMs
// read), then shared memory's 128 bytes per cycle, which products with both operands there use up.  P and K' therefore live in tensor
// memory, and V is all that is read beside them: 3600 cycles of shared memory per chunk (4500 with K' in three parts), where the
// transposed arrangement (columns on the lanes, so that the state is the operand in tensor memory, P and K' in shared memory) took
// 5200 and was bound by that.  What a chunk takes is 5500 cycles (6100), the chain from one state to the next: products wait for
// shared memory, and the roles for one another's instructions.
//
// Roles (28 warps): 0 TMA loads; 1 MMA issue; 2 TMA stores; 4-11 weight the keys and the scores; 12-19 scale inter and bring the
// outputs to shared memory (where q was); 20-27 keep the state, half a row each.  A scheduler has two warps of a role at a time,
// each at its own place in the code, and waits for instructions more than for anything else once that outgrows the instruction
// cache (13 cycles for each instruction, with everything unrolled): loops stay rolled, pairs of fp32 are computed as such, and
// what only a partial chunk needs is done apart.  The tensor pipe's order is inter, delta, out, the next scores: the chain of a
// chunk is inter, delta, state, and the rest fills its gaps.
#include <cuda_fp16.h>
#include <string.h>

#include "linear_attention.cuh"
#include "tc_ptx.cuh"

namespace ringrnn {
namespace {

using namespace tc;

constexpr int C = LA_TC_CHUNK;
constexpr int TILE = C * 128;  // bytes of [128 rows x 64 columns]
constexpr int LT_THREADS = 896;
// registers of warps 0-3, 4-11, 12-19, 20-27 (setmaxnreg): no more than the block is launched with
constexpr int REGS_ISSUE = 32, REGS_WEIGHT = 72, REGS_OUT = 64, REGS_STATE = 96;
static_assert((4 * REGS_ISSUE + 8 * REGS_WEIGHT + 8 * REGS_OUT + 8 * REGS_STATE) * 32 <= 65536 / LT_THREADS / 8 * 8 * LT_THREADS, "registers");
// tensor memory: scores, of each 16 columns the first 8 then P; inter and outputs; delta; K' (hi, lo)
constexpr uint32_t TM_SCORES = 0, TM_OUT = 128, TM_DELTA = 256, TM_KEYS = 384, TM_COLS = 512;
// forming sums: K' (hi, lo, rest) in turn at two places, and delta
constexpr uint32_t TM_SUM_KEYS = 192, TM_SUM_DELTA = 384;

template <int DI, int DO>
struct LtCfg {
  static constexpr int WIDE = DI > DO ? DI : DO;
  static constexpr int SLOT = TILE * (WIDE / 64);
  static constexpr int SLOTS = WIDE == 128 ? 6 : 12;  // two chunks' q, k and v or four's: what it takes to keep the memory busy
  // slots | the state as operand | barriers and tables.  A product reads 128 rows of K' whatever DI is; nobody uses what it makes of the others.
  static constexpr int STATE = SLOT * SLOTS, BARS = STATE + 2 * TILE;
  static constexpr int TABLES = BARS + (2 * SLOTS + 15) * 8 + 8;  // 32 powers; key weights of 64 pairs of tokens, twice
  static_assert(TABLES % 16 == 0, "alignment");
  static constexpr int FLAGS = TABLES + 128 + 512 + 512;
  // fp16: the state's largest element by warp, and what it was divided by, of two chunks; the same of keys and rows (three by warp, in
  // turn at two places); what weighted keys were multiplied by, inverse, of four chunks; and scores, of two chunks' two steps
  static constexpr int RANGE = FLAGS + 16, TOPS = RANGE + 48, KEY_DOWN = TOPS + 256, SCORE_UP = KEY_DOWN + 16;
  static constexpr int SMEM = SCORE_UP + 16;
  static_assert(SMEM <= 232448, "shared memory of a block");
};

struct LtParams {
  LaLaunch L;
  int h_step[LA_MAX_JOBS][3], b_step[LA_MAX_JOBS][3];  // 0: a tensor that all heads / sequences share
  int store[LA_MAX_JOBS];                              // out can be written by TMA
  alignas(64) CUtensorMap map[LA_MAX_JOBS][4];         // q, k, v, out
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
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t a, uint32_t* x) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(a) : "memory");
}
// what differs between the types: pairs of elements, and the bits of an instruction descriptor that name them
template <class E>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  typedef __nv_bfloat162 type;
  static constexpr uint32_t IDESC = 0;
  static __device__ __forceinline__ type from(float a, float b) { return __floats2bfloat162_rn(a, b); }
  static __device__ __forceinline__ float kept(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
};
template <>
struct Pair<__half> {
  typedef __half2 type;
  static constexpr uint32_t IDESC = (1u << 7) | (1u << 10);  // taken from the bf16 descriptor
  static __device__ __forceinline__ type from(float a, float b) { return __floats2half2_rn(a, b); }
  static __device__ __forceinline__ float kept(float x) { return __half2float(__float2half_rn(x)); }
};
template <class E2>
__device__ __forceinline__ uint32_t bits(E2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
template <class E>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return bits(Pair<E>::from(lo, hi));
}
// two bf16 as fp32
__device__ __forceinline__ f32x2 wide(uint32_t pair) { return pk2u(pair << 16, pair & 0xffff0000u); }
template <class E>
__device__ __forceinline__ uint32_t pack2(f32x2 v) {
  float a, b;
  upk2(v, a, b);
  return pack2<E>(a, b);
}
__device__ __forceinline__ f32x2 wide_half(uint32_t pair) {
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&pair));
  return pk2(x.x, x.y);
}
// The power of two, of at most 2^most, that brings a number below 2^15 but not below 2^14; one for zero.
__device__ __forceinline__ float below_2_15(float top, int most) {
  int up = __float_as_uint(top) < 0x800000u ? 0 : 127 + 14 - (int)(__float_as_uint(top) >> 23);
  up = up > most ? most : up < -100 ? -100 : up;
  return __uint_as_float((uint32_t)(127 + up) << 23);
}
// 32 bytes: a whole sector of each lane's own row
__device__ __forceinline__ void ldg8(const float* p, float* x) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
               : "l"(p));
}
__device__ __forceinline__ void stg8(float* p, const float* x) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]),
               "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}
template <int REGS>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }

// What a block does with its chunks: outputs of a job; the sums of a segment; or the outputs of two jobs that share a state.
//
// The last is for gradients: dV (rows K, keys Q, values dO) and dK (rows V, keys dO, values Q) need the same E, the one as
// K E and the other as V E^T.  A chunk of theirs is loaded once instead of one and a half times, its keys are weighted and added
// to the state once instead of twice, and what is left, two products of scores, of state and of values, goes through the same
// places one after the other: step 2c is dV of chunk c, step 2c + 1 is dK.
// Such a block takes 1.55 times as long as one job's.  Measured: gradients of 8 x 2048 x 16 heads of 128, 150 us -> 137; what is left
// of a second round is a dQ block's 57 on most processors (128 pairs and 128 dQ on 148).
enum Mode { OUTPUTS, SUMS, GRADIENT_PAIR };

template <class E, int DI, int DO, int MODE, bool PRECISE>
__device__ __forceinline__ void la_tc_block(const LtParams& A, const int ji, const int at, volatile int* host_status) {
  using Cfg = LtCfg<DI, DO>;
  constexpr bool STATES = MODE == SUMS, PAIR = MODE == GRADIENT_PAIR;
  constexpr int STEPS = PAIR ? 2 : 1;  // of a chunk
  typedef typename Pair<E>::type E2;
  constexpr bool HALF = Pair<E>::IDESC != 0;
  // Tiles of a chunk: rows, keys, values, and for a pair the second rows; forming sums keys and values.
  constexpr int NS = Cfg::SLOTS, TILES = STATES ? 2 : PAIR ? 4 : 3, KEYS = PAIR ? 1 : 0, ROWS = PAIR ? 0 : 1, VALUES = STATES ? 1 : 2;
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
  const LaJob& J = L.job[ji];  // a pair's second is the next one
  const int seg = at % L.segments, bh = at / L.segments, h = bh % L.H, b = bh / L.H;
  const bool rev = J.reverse != 0;
  const int len = la_length(L, b), begin = seg * L.segment_tokens, stop = min(L.T, begin + L.segment_tokens), end = min(len, stop);
  const int chunks = end > begin ? (end - begin + C - 1) / C : 0;
  auto chunk_at = [&](int c) { return begin + (rev ? chunks - 1 - c : c) * C; };

  const bool rest = PRECISE && !HALF && !PAIR && (STATES || J.precise);  // K' in three parts
  auto out_tile = [&](int u) { return PAIR ? TILES * (u >> 1) + 3 * (u & 1) : TILES * u + ROWS; };  // whose place a step's outputs take

  const uint32_t bars = base + Cfg::BARS;
  auto full = [&](int i) { return bars + 8u * i; };
  auto empty = [&](int i) { return bars + 8u * (NS + i); };
  const uint32_t one = bars + 16u * NS;
  const uint32_t scores_ready = one, keys_ready = one + 8, pairs_ready = one + 16, inter_done = one + 24, delta_ready = one + 32,
                 state_ready = one + 40, out_ready = one + 48, out_free = one + 56, all_done = one + 64, tail_ready = one + 72,
                 staged = one + 80, scaled = one + 88, taken = one + 96, rest_ready = one + 104, keys_free = one + 112;
  // A barrier's waiter can only tell one phase from the next.  Two barriers in turn where the other side can be a chunk ahead.
  auto sum_keys_ready = [&](int c) { return c & 1 ? pairs_ready : keys_ready; };  // forming sums: keys two chunks ahead at most
  auto sum_done = [&](int c) { return c & 1 ? out_ready : inter_done; };          // and what they were added to
  auto sum_keys = [&](int c) { return (c & 1) * TM_SUM_KEYS; };
  float* const powers = reinterpret_cast<float*>(mem + Cfg::TABLES);
  uint2* const key_weights = reinterpret_cast<uint2*>(powers + 32);  // of tokens 2i and 2i + 1: what bf16 keeps of them, the rest
  float* const key_weights32 = reinterpret_cast<float*>(key_weights + 64);

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
      mbar_init(scaled, 256);
      mbar_init(taken, 1);
      mbar_init(rest_ready, 256);
      mbar_init(keys_free, 1);
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
    // ---- loads: each chunk's tiles through a ring of slots
    if (lane == 0) {
      int i = 0, round = 0;
      for (int c = 0; c < chunks; ++c) {
        const int t0 = chunk_at(c);
#pragma unroll
        for (int x = 0; x < TILES; ++x) {
          if (!mbar_wait(empty(i), (round & 1) ^ 1, w, 101)) break;
          const int blocks = (x >= VALUES ? DO : DI) / 64, from = x == 3 ? ji + 1 : ji, tensor = x == KEYS ? 1 : x == VALUES ? 2 : 0;
          mbar_arrive_expect_tx(full(i), blocks * TILE);
          for (int k = 0; k < blocks; ++k)
            tma_load_4d(base + i * Cfg::SLOT + k * TILE, &A.map[from][tensor], full(i), k * 64, t0, h * A.h_step[from][tensor],
                        b * A.b_step[from][tensor]);
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
    // (M, N, whether A and B have their rows along K)
    constexpr uint32_t ID_SCORES = make_idesc_bf16(128, 128, 0, 0) - Pair<E>::IDESC, ID_OUT = make_idesc_bf16(128, DO, 0, 1) - Pair<E>::IDESC,
                       ID_OUT2 = make_idesc_bf16(128, DI, 0, 1) - Pair<E>::IDESC, ID_INTER2 = make_idesc_bf16(128, DI, 0, 0) - Pair<E>::IDESC,
                       ID_REST = make_idesc_bf16(128, DO, 1, 1) - Pair<E>::IDESC;
    auto slot = [&](int tile) { return base + (tile % NS) * Cfg::SLOT; };
    auto loaded = [&](int tile, int code) { mbar_wait(full(tile % NS), (tile / NS) & 1, w, code); };
    // K-major operands: 16 of the 64 columns of a 128-byte row at a time
    auto k_major = [&](uint32_t tile, int ks) { return desc_sw128(desc_lo(tile + (ks >> 2) * TILE + (ks & 3) * 32, 0)); };
    // M/N-major ones: 16 rows, blocks of 64 columns a tile apart
    auto mn_major = [&](uint32_t tile, int ks) { return desc_sw128(desc_lo(tile + ks * 2048, TILE)); };
    // inter, (delta,) out of step u, scores of the next; loops are left rolled where their instructions keep up (see above)
#pragma unroll 1
    for (int i = STATES ? 1 : 0; i <= chunks * STEPS; ++i) {
      const int u = i - 1, c = PAIR ? u >> 1 : u, tile = TILES * c;
      const bool second = PAIR && (u & 1);
      if (i > 0) {
        if (!STATES) {
          if (!second) mbar_wait(state_ready, c & 1, w, 112);
          if (u > 0) mbar_wait(out_free, (u - 1) & 1, w, 113);
          tcgen05_fence_after();
          if (!second) {
#pragma unroll 2
            for (int ks = 0; ks < DI / 16; ++ks)
              umma_ss_warp(tm + TM_OUT, k_major(slot(tile + ROWS), ks), mn_major(base + Cfg::STATE, ks), ID_OUT, ks != 0, lead);
          } else {
#pragma unroll 2
            for (int ks = 0; ks < DO / 16; ++ks)
              umma_ss_warp(tm + TM_OUT, k_major(slot(tile + 3), ks), k_major(base + Cfg::STATE, ks), ID_INTER2, ks != 0, lead);
          }
          if (lead) umma_commit(inter_done);
          __syncwarp();
        }
        loaded(tile + VALUES, 115);
        const uint32_t v = slot(tile + VALUES);
        const bool add = !PAIR || second;
        const uint32_t delta = tm + (STATES ? TM_SUM_DELTA : TM_DELTA);
        if (add) {
          if (STATES) {
            mbar_wait(sum_keys_ready(c), (c >> 1) & 1, w, 114);
            if (c > 0) mbar_wait(state_ready, (c - 1) & 1, w, 112);
          } else {
            mbar_wait(keys_ready, c & 1, w, 114);
          }
          tcgen05_fence_after();
          const uint32_t keys = tm + (STATES ? sum_keys(c) : TM_KEYS);
#pragma unroll 2
          for (int x = 0; x < C / 8; ++x)
            umma_ts_warp(delta, keys + (x & 1) * 64 + (x >> 1) * 8, mn_major(v, x >> 1), ID_OUT, x != 0, lead);
          if (STATES && rest) {
#pragma unroll 2
            for (int ks = 0; ks < C / 16; ++ks) umma_ts_warp(delta, keys + 128 + ks * 8, mn_major(v, ks), ID_OUT, true, lead);
          }
          if (lead) {
            if (STATES) {
              umma_commit(sum_done(c));
              umma_commit(empty((tile + KEYS) % NS));
              umma_commit(empty((tile + VALUES) % NS));
            } else {
              umma_commit(keys_free);
              if (!rest) umma_commit(delta_ready);
            }
          }
          __syncwarp();
        }
        if (!STATES) {
          mbar_wait(scaled, u & 1, w, 116);
          mbar_wait(pairs_ready, u & 1, w, 117);
          tcgen05_fence_after();
          const uint32_t values = second ? slot(tile + KEYS) : v;
#pragma unroll 2
          for (int ks = 0; ks < C / 16; ++ks)
            umma_ts_warp(tm + TM_OUT, tm + TM_SCORES + 16 * ks, mn_major(values, ks), second ? ID_OUT2 : ID_OUT, true, lead);
          if (lead) umma_commit(out_ready);
          __syncwarp();
          if (rest) {
            mbar_wait(rest_ready, c & 1, w, 114);
            tcgen05_fence_after();
#pragma unroll 2
            for (int ks = 0; ks < C / 16; ++ks) umma_ss_warp(delta, mn_major(slot(tile + KEYS), ks), mn_major(v, ks), ID_REST, true, lead);
            if (lead) umma_commit(delta_ready);
            __syncwarp();
          }
          if (add && lead) {
            umma_commit(empty((tile + KEYS) % NS));
            umma_commit(empty((tile + VALUES) % NS));
          }
          __syncwarp();
        }
      }
      if (!STATES && i < chunks * STEPS) {
        const int n = PAIR ? i >> 1 : i;
        const bool two = PAIR && (i & 1);
        const int rows = TILES * n + (two ? 3 : ROWS), keys = TILES * n + (two ? VALUES : KEYS);
        loaded(rows, 110);
        loaded(keys, 111);
        if (chunk_at(n) + C > end) mbar_wait(tail_ready, 0, w, 119);
        // the scores go where out has just read P: no order holds between MMAs of different accumulators
        if (i > 0) mbar_wait(out_ready, u & 1, w, 118);
        tcgen05_fence_after();
#pragma unroll 2
        for (int ks = 0; ks < (two ? DO : DI) / 16; ++ks)
          umma_ss_warp(tm + TM_SCORES, k_major(slot(rows), ks), k_major(slot(keys), ks), ID_SCORES, ks != 0, lead);
        if (lead) umma_commit(scores_ready);
        __syncwarp();
      }
    }
    // tensor memory is given back below: nothing may still be writing it (at once, unless a wait was abandoned)
    if (lead) umma_commit(all_done);
    mbar_wait(all_done, 0, drain, 118);
  } else if (warp == 2) {
    // ---- stores: outputs from the slot that held the rows, which is free after that
    if (!STATES && lane == 0) {
      for (int u = 0; u < chunks * STEPS; ++u) {
        const int c = PAIR ? u >> 1 : u, job = PAIR ? ji + (u & 1) : ji, slot = out_tile(u) % NS;
        if (!mbar_wait(staged, u & 1, w, 150)) break;
        mbar_arrive(taken);
        if (A.store[job]) {
          for (int k = 0; k < (PAIR && (u & 1) ? DI : DO) / 64; ++k)
            tma_store_4d(&A.map[job][3], base + slot * Cfg::SLOT + k * TILE, k * 64, chunk_at(c), h, b);
          bulk_commit();
          bulk_wait_read<0>();
        }
        mbar_arrive(empty(slot));
      }
      bulk_wait_all<0>();
    }
  } else if (warp >= 4 && warp < 12) {
    // ---- keys, transposed and weighted for the state, then scores weighted
    regs_down<REGS_WEIGHT>();
    const int q = warp & 3, half = (warp - 4) >> 2, r = q * 32 + lane, a = tid - 128;
    const int col = half * 16;  // scores: a thread has row r and these 16 of each 32 columns
    // Weights of scores, the same in every chunk.  The diagonal block's stand in registers.  Another block's are the power up to
    // its near end, a factor per token (32 tokens more: times g^32), times one within the block: all at most one.
    f32x2 diagonal[8];
    const float near = J.pair_scale * g.power(rev ? 32 - lane : lane + 1), g32 = g.power(32);
#pragma unroll
    for (int s = 0; s < 16; s += 2) {
      const int far = rev ? col + s - lane : lane - col - s, far1 = rev ? far + 1 : far - 1;
      diagonal[s / 2] = pk2(far >= 0 ? J.pair_scale * g.power(far) : 0.f, far1 >= 0 ? J.pair_scale * g.power(far1) : 0.f);
    }
    int have = 0, turn = 0;
    // fp16: the largest element of this thread's half of row r (an infinity has no part in what the others are scaled by)
    auto row_top = [&](int tile, int width, int n) {
      mbar_wait(full(tile % NS), (tile / NS) & 1, w, 124);
      const uint32_t from = base + (tile % NS) * Cfg::SLOT;
      __half2 top = __float2half2_rn(0.f);
      if (r < n)
#pragma unroll 4
        for (int i = half; i < width / 8; i += 2) {
          uint32_t x[4];
          lds128(from + (i >> 3) * TILE + sw128_offset(r, (i & 7) * 8), x);
#pragma unroll
          for (int e = 0; e < 4; ++e) top = __hmax2(top, __habs2(*reinterpret_cast<const __half2*>(x + e)));
        }
      const float x = __half2float(__hmax(__low2half(top), __high2half(top)));
      return x < 65536.f ? x : 0.f;
    };
    // the largest of all threads' numbers (not negative: their order is that of their bits)
    auto largest = [&](float x, float y, float z) {
      uint4* const tops = reinterpret_cast<uint4*>(mem + Cfg::TOPS) + turn;
      turn ^= 8;
      auto top = [](uint32_t bits) { return __reduce_max_sync(0xffffffffu, bits); };
      const uint4 mine = make_uint4(top(__float_as_uint(x)), top(__float_as_uint(y)), top(__float_as_uint(z)), 0u);
      if (lane == 0) tops[warp - 4] = mine;
      named_bar_sync(1, 256);
      const uint4 all = tops[lane & 7];
      return make_float3(__uint_as_float(top(all.x)), __uint_as_float(top(all.y)), __uint_as_float(top(all.z)));
    };
    const float grows = fmaxf(1.f, g.power(C - 1));
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
      const int t0 = chunk_at(c), n = min(C, end - t0), kt = TILES * c + KEYS, vt = TILES * c + VALUES;
      const uint32_t k = base + (kt % NS) * Cfg::SLOT;
      mbar_wait(full(kt % NS), (kt / NS) & 1, w, 120);
      if (n < C) {
        // what stands behind the sequence, a NaN included, becomes zero before anybody reads it
        mbar_wait(full(vt % NS), (vt / NS) & 1, w, 123);
        if (r >= n) {
          const uint32_t v = base + (vt % NS) * Cfg::SLOT;
          for (int i = half; i < DI / 8; i += 2) sts128(k + (i >> 3) * TILE + sw128_offset(r, (i & 7) * 8), 0, 0, 0, 0);
          for (int i = half; i < DO / 8; i += 2) sts128(v + (i >> 3) * TILE + sw128_offset(r, (i & 7) * 8), 0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        if (!STATES) mbar_arrive(tail_ready);
      }
      if (STATES || n != have) {  // the keys' weights: they change with the number of tokens, and towards a segment's end
        named_bar_sync(1, 256);
        if (a < 64) {
          float x[2], left[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int s = 2 * a + e;
            const int steps = STATES ? (rev ? t0 + s - begin + 1 : end - 1 - t0 - s) : rev ? s + 1 : n - 1 - s;
            x[e] = s < n ? J.key_scale * g.power(steps) : 0.f;
            left[e] = x[e] - Pair<E>::kept(x[e]);
          }
          if (!HALF) key_weights[a] = make_uint2(pack2<E>(x[0], x[1]), pack2<E>(left[0], left[1]));
          key_weights32[2 * a] = x[0], key_weights32[2 * a + 1] = x[1];
        }
        named_bar_sync(1, 256);
        have = n;
      }
      float keys_up = 1.f, keys_top = 0.f, rows_top = 0.f;
      if constexpr (HALF) {
        const float top = row_top(kt, DI, n);
        const float3 all = largest(top * fabsf(key_weights32[r]), top, STATES ? 0.f : row_top(TILES * c + ROWS, DI, n));
        keys_up = below_2_15(all.x, 100);
        keys_top = all.y, rows_top = all.z;
        if (a == 0) reinterpret_cast<float*>(mem + Cfg::KEY_DOWN)[c & 3] = 1.f / keys_up;
      }
      // what read the last keys: the chunk before's delta; forming sums, of two chunks before
      if (STATES ? c > 1 : c > 0) {
        if (STATES) mbar_wait(sum_done(c), ((c >> 1) - 1) & 1, w, 121);
        else mbar_wait(keys_free, (c - 1) & 1, w, 121);
        tcgen05_fence_after();
      }
      // in fp32, of bf16 products: z w - hi - lo, rounded
      auto remains = [](uint32_t z, f32x2 w32, E2 hi, E2 lo) { return pack2<E>(add2(fma2(wide(z), w32, wide(bits(__hneg2(hi)))), wide(bits(__hneg2(lo))))); };
      if (q * 32 < DI) {
        // bf16: k w = hi + lo with w = w_hi + w_lo, all of the tensors' type: hi = k w_hi rounded, what that leaves is exact (half of the
        // product's bits), lo = k w_lo + that, rounded.  Three instructions for two elements, where the way through fp32 takes eight.
        const int row = half * 64 + (lane >> 4) * 8 + (lane & 7), in = (q & 1) * 32 + ((lane >> 3) & 1) * 8;  // matrices: two of tokens by two of columns
        const uint32_t from = k + (q >> 1) * TILE, to = tm + (STATES ? sum_keys(c) : TM_KEYS) + ((uint32_t)(q * 32) << 16) + half * 32;
        const uint2* kw = key_weights + half * 32 + (lane & 3);
#pragma unroll 1
        for (int j = 0; j < 2; ++j) {  // 32 tokens
          uint2 wt[4];
          f32x2 wt32[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (HALF) {
              const float2 x = *reinterpret_cast<const float2*>(key_weights32 + 2 * (half * 32 + (lane & 3) + (j * 4 + e) * 4));
              wt32[e] = mul2(pk2(x.x, x.y), pk2(keys_up, keys_up));
            } else {
              wt[e] = kw[(j * 4 + e) * 4];
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // 16 columns
            uint32_t hi[8], lo[8], left[8];
            ldmatrix_x4_trans(from + sw128_offset(row + j * 32, in + i * 16), lo);
            ldmatrix_x4_trans(from + sw128_offset(row + j * 32 + 16, in + i * 16), lo + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if constexpr (HALF) {
                // the type's small numbers have few bits, so by way of fp32, with the chunk's largest product just below 2^15
                const f32x2 p = mul2(wide_half(lo[e]), wt32[e >> 1]);
                hi[e] = pack2<E>(p);
                lo[e] = pack2<E>(fma2(wide_half(hi[e]), pk2(-1.f, -1.f), p));
                continue;
              }
              const E2 wh = *reinterpret_cast<const E2*>(&wt[e >> 1].x), wl = *reinterpret_cast<const E2*>(&wt[e >> 1].y),
                       z = *reinterpret_cast<const E2*>(lo + e), h2 = __hmul2_rn(z, wh), l2 = __hfma2(z, wl, __hfma2(z, wh, __hneg2(h2)));
              if (STATES && !HALF) {
                const float2 w32 = *reinterpret_cast<const float2*>(key_weights32 + 2 * (half * 32 + (lane & 3) + (j * 4 + (e >> 1)) * 4));
                left[e] = remains(lo[e], pk2(w32.x, w32.y), h2, l2);
              }
              hi[e] = bits(h2);
              lo[e] = bits(l2);
            }
            tmem_st_frag4(to + ((uint32_t)(i * 16) << 16) + j * 16, hi);
            tmem_st_frag4(to + ((uint32_t)(i * 16) << 16) + 64 + j * 16, lo);
            if (STATES && !HALF) tmem_st_frag4(to + ((uint32_t)(i * 16) << 16) + 128 + j * 16, left);
          }
        }
        tmem_st_wait();
        tcgen05_fence_before();
      }
      // What hi and lo leave of k w in fp32, in k's place, once nobody reads that any more (tensor memory has no room for it).
      auto leave_rest = [&] {
        named_bar_sync(1, 256);
#pragma unroll 2
        for (int at0 = 0; at0 < 128 * DI / 8; at0 += 256) {
          const int i = at0 + a;
          const int s = (i >> 3) & 127;  // eight elements of one token
          const uint32_t at = k + (i >> 10) * TILE + sw128_offset(s, (i & 7) * 8);
          const float x = key_weights32[s], kept = Pair<E>::kept(x);
          const uint32_t wh_bits = pack2<E>(kept, kept), wl_bits = pack2<E>(x - kept, x - kept);
          const E2 wh = *reinterpret_cast<const E2*>(&wh_bits), wl = *reinterpret_cast<const E2*>(&wl_bits);
          uint32_t y[4];
          lds128(at, y);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const E2 z = *reinterpret_cast<const E2*>(y + e), h2 = __hmul2_rn(z, wh), l2 = __hfma2(z, wl, __hfma2(z, wh, __hneg2(h2)));
            y[e] = remains(y[e], pk2(x, x), h2, l2);
          }
          sts128(at, y[0], y[1], y[2], y[3]);
        }
        fence_proxy_async_smem();
      };
      mbar_arrive(STATES ? sum_keys_ready(c) : keys_ready);
#pragma unroll 1
      for (int step = 0; step < (STATES ? 0 : STEPS); ++step) {
        float up = 1.f;
        if constexpr (HALF) {
          // Scores are brought below 2^15 by what bounds them: the width times the largest elements of rows and keys.
          if (step > 0) {
            const float3 all = largest(0.f, row_top(vt, DO, n), row_top(TILES * c + 3, DO, n));
            keys_top = all.y, rows_top = all.z;
          }
          up = below_2_15((step > 0 ? J.outer : J.inner) * rows_top * keys_top * fabsf(J.pair_scale) * grows, 64);
          if (a == 0) reinterpret_cast<float*>(mem + Cfg::SCORE_UP)[(c & 1) * 2 + step] = up;
        }
        mbar_wait(scores_ready, (c * STEPS + step) & 1, w, 122);
        tcgen05_fence_after();
        const uint32_t mine = tm + TM_SCORES + ((uint32_t)(q * 32) << 16) + col;
        uint32_t x[16];
        f32x2 y[8];
        auto put = [&](int j) {
          uint32_t z[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = pack2<E>(y[e]);
          tmem_st8(mine + j * 32, z);
        };
        tmem_ld16(mine + q * 32, x);
        tmem_ld_wait();
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          y[s] = mul2(pk2u(x[2 * s], x[2 * s + 1]), diagonal[s]);
          if (HALF) y[s] = mul2(y[s], pk2(up, up));
        }
        put(q);
        float f = HALF ? near * up : near;
#pragma unroll 1
        for (int j = rev ? q + 1 : q - 1; rev ? j < 4 : j >= 0; j += rev ? 1 : -1) {
          tmem_ld16(mine + j * 32, x);
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
          put(j);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0u;
#pragma unroll 1
        for (int j = rev ? q - 1 : q + 1; rev ? j >= 0 : j < 4; j += rev ? -1 : 1) tmem_st8(mine + j * 32, x);  // what none of these tokens sees
        tmem_st_wait();
        tcgen05_fence_before();
        mbar_arrive(pairs_ready);
      }
      if (PRECISE && !STATES && rest) {
        leave_rest();
        mbar_arrive(rest_ready);
      }
    }
  } else if (warp >= 12 && warp < 20) {
    // ---- outputs: a thread has token r and half of its columns.  Inter is scaled; later the sum goes to shared memory
    regs_down<REGS_OUT>();
    if (!STATES) {
      const int q = warp & 3, half = (warp - 12) >> 2, r = q * 32 + lane, a = tid - 384;
#pragma unroll 1
      for (int u = 0; u < chunks * STEPS; ++u) {
        const int c = PAIR ? u >> 1 : u, job = PAIR ? ji + (u & 1) : ji, N = (PAIR && (u & 1) ? DI : DO) / 2, o0 = half * N;
        const uint32_t mine = tm + TM_OUT + ((uint32_t)(q * 32) << 16) + o0;
        const int t0 = chunk_at(c), n = min(C, end - t0);
        const int slot = (out_tile(u) % NS) * Cfg::SLOT;
        float f = r < n ? J.row_scale * g.power(rev ? n - 1 - r : r + 1) : 0.f;
        mbar_wait(inter_done, u & 1, w, 130);
        tcgen05_fence_after();
        float down = 1.f;
        if (HALF) {
          mbar_wait(pairs_ready, u & 1, w, 133);  // (what the scores were multiplied by is known then)
          const float up = reinterpret_cast<const volatile float*>(mem + Cfg::SCORE_UP)[(c & 1) * 2 + u % STEPS];
          f *= reinterpret_cast<const volatile float*>(mem + Cfg::RANGE)[8 + (c & 1)] * up;
          down = 1.f / up;
        }
        const f32x2 f2 = pk2(f, f), down2 = pk2(down, down);
#pragma unroll 1
        for (int i = 0; i < N; i += 16) {
          uint32_t x[16];
          tmem_ld16(mine + i, x);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float y, z;
            upk2(mul2(f2, pk2u(x[e], x[e + 1])), y, z);
            x[e] = __float_as_uint(y), x[e + 1] = __float_as_uint(z);
          }
          tmem_st8(mine + i, x);
          tmem_st8(mine + i + 8, x + 8);
        }
        tmem_st_wait();
        tcgen05_fence_before();
        mbar_arrive(scaled);
        mbar_wait(out_ready, u & 1, w, 131);
        tcgen05_fence_after();
        const uint32_t to = base + slot + (o0 >> 6) * TILE;
#pragma unroll 1
        for (int i = 0; i < N; i += 16) {
          uint32_t x[16];
          tmem_ld16(mine + i, x);
          tmem_ld_wait();
          if (i + 16 == N) {  // all of it is in registers
            tcgen05_fence_before();
            mbar_arrive(out_free);
          }
          uint32_t y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const f32x2 z = pk2u(x[2 * e], x[2 * e + 1]);
            y[e] = r < n ? pack2<E>(HALF ? mul2(z, down2) : z) : 0u;
          }
          sts128(to + sw128_offset(r, (o0 & 63) + i), y[0], y[1], y[2], y[3]);
          sts128(to + sw128_offset(r, (o0 & 63) + i + 8), y[4], y[5], y[6], y[7]);
        }
        if (!A.store[job]) {  // widths and addresses that TMA does not take: as many elements at a time as they allow
          named_bar_sync(2, 256);
          const int outer = L.job[job].outer, rows = min(C, stop - t0);
          const size_t pitch = (size_t)L.H * outer;
          unsigned short* const out = static_cast<unsigned short*>(L.job[job].out) + (((size_t)b * L.T + t0) * L.H + h) * outer;
          auto copy = [&](auto word) {  // four rows' words under way at a time
            typedef decltype(word) P;
            constexpr int N = sizeof(P) / 2, LANES = 128 / N, PER = 256 / LANES;
            const int o = (a & (LANES - 1)) * N;
#pragma unroll 1
            for (int r0 = a / LANES; r0 < rows; r0 += 4 * PER) {
              P z[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (r0 + j * PER < rows && o < outer)
                  z[j] = *reinterpret_cast<const P*>(mem + slot + (o >> 6) * TILE + sw128_offset(r0 + j * PER, o & 63));
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (r0 + j * PER < rows && o < outer) *reinterpret_cast<P*>(out + (r0 + j * PER) * pitch + o) = z[j];
            }
          };
          // (odd widths by words, with the rows' two kinds of boundary told apart, took longer: forward of 8 x 2048 x 16 heads of 121
          // 306 us, so 176)
          const uintptr_t boundary = reinterpret_cast<uintptr_t>(L.job[job].out) | (uintptr_t)outer * 2;
          if (boundary % 8 == 0) copy(uint2());
          else if (boundary % 4 == 0) copy(uint32_t());
          else copy((unsigned short)0);
        }
        fence_proxy_async_smem();
        if (u > 0) mbar_wait(taken, (u - 1) & 1, w, 132);  // a store may wait for the memory longer than a chunk takes
        mbar_arrive(staged);
      }
      // tokens behind the sequence, beyond its last chunk
#pragma unroll 1
      for (int job = ji; job < ji + STEPS; ++job) {
        const int outer = L.job[job].outer, o = a & 127;
        unsigned short* const out = static_cast<unsigned short*>(L.job[job].out) + ((size_t)b * L.T * L.H + h) * outer + o;
#pragma unroll 1
        for (int t = begin + chunks * C + (a >> 7); t < stop; t += 2)
          if (o < outer) out[(size_t)t * L.H * outer] = 0;
      }
    }
  } else if (warp >= 20) {
    // ---- the state: a thread has half a row
    regs_up<REGS_STATE>();
    constexpr int N = DO / 2;
    const int q = warp & 3, half = (warp - 20) >> 2, in = q * 32 + lane, o0 = half * N;
    const uint32_t mine = tm + TM_DELTA + ((uint32_t)(q * 32) << 16) + o0;
    const uint32_t to = base + Cfg::STATE + (o0 >> 6) * TILE;
    const size_t mat = (size_t)at * J.inner * J.outer;
    // rows of a state in its own order are read and written a sector at a time (the transposed ones come lane by lane)
    auto rows_of_sectors = [&](const float* p) { return J.s_out == 1 && (J.outer & 7) == 0 && (reinterpret_cast<uintptr_t>(p) & 31) == 0; };
    f32x2 S[N / 2];
    {
      const float* from = J.init + mat + (size_t)in * J.s_in + (size_t)o0 * J.s_out;
      const bool given = !STATES && J.init != nullptr && in < J.inner, sectors = rows_of_sectors(J.init);
#pragma unroll
      for (int i = 0; i < N; i += 8) {
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (given && sectors) {
          if (o0 + i < J.outer) ldg8(from + i, x);
        } else if (given) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (o0 + i + e < J.outer) x[e] = from[(size_t)(i + e) * J.s_out];
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) S[(i + e) / 2] = pk2(x[e], x[e + 1]);
      }
    }
    if (STATES) {
      // (added up here and not by the tensor cores, which cut a sum off at 2^-24 of it, over hundreds of chunks)
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        mbar_wait(sum_done(c), (c >> 1) & 1, w, 140);
        tcgen05_fence_after();
        const uint32_t from = mine - TM_DELTA + TM_SUM_DELTA;
        const float times = HALF ? reinterpret_cast<const volatile float*>(mem + Cfg::KEY_DOWN)[c & 3] : 1.f;
#pragma unroll
        for (int i = 0; i < N; i += 16) {
          uint32_t x[16];
          tmem_ld16(from + i, x);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 8; ++e) S[i / 2 + e] = fma2(pk2(times, times), pk2u(x[2 * e], x[2 * e + 1]), S[i / 2 + e]);
        }
        tcgen05_fence_before();
        mbar_arrive(state_ready);
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
          const float times = HALF ? reinterpret_cast<const volatile float*>(mem + Cfg::KEY_DOWN)[(c - 1) & 3] : 1.f;
#pragma unroll
          for (int i = 0; i < N; i += 16) {
            uint32_t y[16];
            tmem_ld16(mine + i, y);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              f32x2 delta = pk2u(y[2 * e], y[2 * e + 1]);
              if (HALF) delta = mul2(delta, pk2(times, times));
              S[i / 2 + e] = fma2(g_hi, S[i / 2 + e], fma2(g_lo, S[i / 2 + e], delta));
            }
          }
        }
        if (c < chunks) {  // the next operand (delta of this chunk is behind inter, which has read the last one)
          float down = 1.f;
          if (HALF) {  // the largest element of all, and the power of two that brings it below 2^15 but not 2^14
            volatile float* const range = reinterpret_cast<volatile float*>(mem + Cfg::RANGE);
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
              float x, y;
              upk2(S[i], x, y);
              top = fmaxf(top, fmaxf(fabsf(x), fabsf(y)));
            }
            if (in >= DI) top = 0.f;
#pragma unroll
            for (int e = 16; e > 0; e >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
            named_bar_sync(3, 256);  // the last chunk's have been read
            if (lane == 0) range[warp - 20] = top;
            named_bar_sync(3, 256);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, range[e]);
            const int exponent = (int)(__float_as_uint(top) >> 23) - 127 - 14;
            if (exponent > -100 && exponent < 100) down = __uint_as_float((uint32_t)(127 - exponent) << 23);
            if (tid == 640) range[8 + (c & 1)] = 1.f / down;
          }
          if (in < DI) {
            const f32x2 down2 = pk2(down, down);
            auto two = [&](int i) { return pack2<E>(HALF ? mul2(S[i], down2) : S[i]); };
#pragma unroll
            for (int i = 0; i < N; i += 8) sts128(to + sw128_offset(in, (o0 & 63) + i), two(i / 2), two(i / 2 + 1), two(i / 2 + 2), two(i / 2 + 3));
          }
          fence_proxy_async_smem();
          tcgen05_fence_before();
          mbar_arrive(state_ready);
        }
      }
    }
    if (J.fin != nullptr && in < J.inner) {
      float* fin = J.fin + mat + (size_t)in * J.s_in + (size_t)o0 * J.s_out;
      const bool sectors = rows_of_sectors(J.fin);
#pragma unroll
      for (int i = 0; i < N; i += 8) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e += 2) upk2(S[(i + e) / 2], x[e], x[e + 1]);
        if (sectors) {
          if (o0 + i < J.outer) stg8(fin + i, x);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (o0 + i + e < J.outer) fin[(size_t)(i + e) * J.s_out] = x[e];
        }
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tm, TM_COLS);
}

template <class E, int DI, int DO, int MODE>
__global__ void __launch_bounds__(LT_THREADS, 1) la_tc_kernel(const __grid_constant__ LtParams A, volatile int* host_status) {
  la_tc_block<E, DI, DO, MODE, true>(A, (int)(blockIdx.x % A.L.jobs), (int)(blockIdx.x / A.L.jobs), host_status);
}
// Gradients: jobs dQ, dV, dK.  The longer blocks first, so that the others fill the last round: dV and dK of each sequence, head and
// segment together, then dQ (inner and outer widths exchanged).
template <class E, int DK, int DV>
__global__ void __launch_bounds__(LT_THREADS, 1) la_tc_gradients_kernel(const __grid_constant__ LtParams A, volatile int* host_status) {
  const int pairs = gridDim.x / 2;
  if ((int)blockIdx.x < pairs) la_tc_block<E, DK, DV, GRADIENT_PAIR, false>(A, 1, (int)blockIdx.x, host_status);
  else la_tc_block<E, DV, DK, OUTPUTS, false>(A, 0, (int)blockIdx.x - pairs, host_status);
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

int launch(void (*kernel)(LtParams, volatile int*), int smem, int blocks, const LtParams& P, cudaStream_t s) {
  volatile int* host = nullptr;
  const int rc = host_status_word(&host);
  if (rc != RINGRNN_OK) return rc;
  RINGRNN_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  LaunchScope ls(K_LAYER, s);
  kernel<<<blocks, LT_THREADS, smem, s>>>(P, host);
  RINGRNN_CUDA_TRY(cudaGetLastError());
  return RINGRNN_OK;
}
// all jobs of one shape; gradients: DI x DO is the state's shape
template <class E, int DI, int DO>
int launch(int mode, const LtParams& P, cudaStream_t s) {
  constexpr int smem = LtCfg<DI, DO>::SMEM;
  const int each = P.L.B * P.L.H * P.L.segments;
  switch (mode) {
    case OUTPUTS: return launch(la_tc_kernel<E, DI, DO, OUTPUTS>, smem, each * P.L.jobs, P, s);
    case SUMS: return launch(la_tc_kernel<E, DI, DO, SUMS>, smem, each * P.L.jobs, P, s);
    default: return launch(la_tc_gradients_kernel<E, DI, DO>, smem, each * 2, P, s);
  }
}
template <class E>
int launch(int di, int d_o, int mode, const LtParams& P, cudaStream_t s) {
  return di == 64 ? (d_o == 64 ? launch<E, 64, 64>(mode, P, s) : launch<E, 64, 128>(mode, P, s))
                  : (d_o == 64 ? launch<E, 128, 64>(mode, P, s) : launch<E, 128, 128>(mode, P, s));
}
int launch(int dtype, int di, int d_o, int mode, const LtParams& P, cudaStream_t s) {
  return dtype == RINGRNN_F16 ? launch<__half>(di, d_o, mode, P, s) : launch<__nv_bfloat16>(di, d_o, mode, P, s);
}
bool add_job(LtParams* P, const LaJob& J, bool sums) {
  const LaLaunch& L = P->L;
  const int to = P->L.jobs++;
  P->L.job[to] = J;
  const LaOperand* ops[3] = {&J.q, &J.k, &J.v};
  for (int x = sums ? 1 : 0; x < 3; ++x)
    if (!make_map(&P->map[to][x], *ops[x], x == 2 ? J.outer : J.inner, L.B, L.T, L.H, &P->h_step[to][x], &P->b_step[to][x])) return false;
  int unused[2];
  const LaOperand out{J.out, (long long)L.T * L.H * J.outer, (long long)L.H * J.outer, J.outer};
  P->store[to] = !sums && J.outer % 8 == 0 && (reinterpret_cast<uintptr_t>(J.out) & 15) == 0;
  return !P->store[to] || make_map(&P->map[to][3], out, J.outer, L.B, L.T, L.H, unused, unused + 1);
}
int padded(int width) { return width <= 64 ? 64 : 128; }

}  // namespace

bool la_tc_operand_ok(const LaOperand& o, int B, int T, int H) {
  const bool t = T == 1 || (o.st > 0 && o.st % 8 == 0 && o.st < (1LL << 38));
  const bool h = H == 1 || (o.sh >= 0 && o.sh % 8 == 0 && o.sh < (1LL << 38));
  const bool b = B == 1 || (o.sb >= 0 && o.sb % 8 == 0 && o.sb < (1LL << 38));
  return t && h && b && (reinterpret_cast<uintptr_t>(o.p) & 15) == 0;
}

int la_tc_launch(const LaLaunch& L, int dtype, bool sums, cudaStream_t s) {
  LtParams P;
  memset(&P, 0, sizeof(P));
  P.L = L;
  P.L.jobs = 0;
  const bool at_once = L.B * L.H * L.segments * L.jobs <= LA_TC_BLOCKS;
  if (!sums && L.jobs == 3 && !at_once && !L.job[2].precise) {  // (a pair needs its keys to the end of a chunk: no room for their rest)
    const int order[3] = {0, 2, 1};
    for (int j : order)
      if (!add_job(&P, L.job[j], false)) return RINGRNN_ERR_CUDA;
    return launch(dtype, padded(L.job[2].inner), padded(L.job[2].outer), GRADIENT_PAIR, P, s);
  }
  // Jobs of one shape together.  Where all of them fit the GPU at once, the largest shape does for all: its products take longer, a
  // second launch more (gradients of 5 x 777 x 6 heads of 64 and 104, 90 CTAs: 25 us instead of 44).  So do gradients job by job.
  int most_in = 64, most_out = 64;
  for (int j = 0; j < L.jobs; ++j) {
    most_in = padded(L.job[j].inner) > most_in ? padded(L.job[j].inner) : most_in;
    most_out = padded(L.job[j].outer) > most_out ? padded(L.job[j].outer) : most_out;
  }
  for (int shape = 0; shape < 4; ++shape) {
    const int di = shape & 1 ? 128 : 64, d_o = shape & 2 ? 128 : 64;
    P.L.jobs = 0;
    for (int j = 0; j < L.jobs; ++j)
      if (di == (at_once ? most_in : padded(L.job[j].inner)) && d_o == (at_once ? most_out : padded(L.job[j].outer)))
        if (!add_job(&P, L.job[j], sums)) return RINGRNN_ERR_CUDA;
    if (P.L.jobs == 0) continue;
    const int rc = launch(dtype, di, d_o, sums ? SUMS : OUTPUTS, P, s);
    if (rc != RINGRNN_OK) return rc;
  }
  return RINGRNN_OK;
}

}  // namespace ringrnn
