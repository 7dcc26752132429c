// frn_prompt_attention.cu -- causal grouped-query attention over packed
// prompts.
//
//   out[i, h, :] = sum_{j <= i} softmax_j(scale * q[i, h, :] . k[j, h / G, :]) v[j, h / G, :]
//
// for every token i of every sequence, j running over the tokens of the same
// sequence; the sequences lie one after the other in the token dimension,
// sequence b in rows [cu_seqlens[b], cu_seqlens[b + 1]).
//
// Work item: one KV head and 2 x TQ consecutive tokens of one sequence, TQ =
// 128 / G.  All G query heads of a token share its keys, so (token, head)
// pairs are the rows of the tile: row r of a 128-row tile is token r / G, head
// r % G, which a 4-D TMA box (d, head of the group, KV head, token) delivers
// in that order.  A short sequence thus fills its tiles G times as well, the
// causal edge is G times finer, and every K/V tile serves two row tiles.
// Items are numbered by falling length of their key range (the last blocks of
// the longest sequences first), so that the device ends evenly; KV heads whose
// keys and values would not fit L2 together come one group after the other.
//
// There is a CTA for each item; those that run take over the items of CTAs that
// have not been launched, in that order.  Two row tiles an item take turns on the
// tensor core:
//   S_s = Q_s K_j^T   (128 rows x 128 keys, operands in shared memory)
//   O_s += P_s V_j    (P_s from TMEM, where it overwrites S_s; V from shared
//                      memory as it lies, keys being the slow dimension)
// While one tile's S is exponentiated by its four warps (one row a thread, no
// shuffles), the other tile's two products run.  The MMAs of a row tile are
// issued by one thread in the order PV_s(j), S_s(j+1): a completed S_s(j+1)
// implies a completed PV_s(j), so the softmax warps need one barrier for both.
// After a tile's last PV comes its first S of the next item, so that the loads
// and first products of an item run under the end of the last.
//
// Roles: warps 0-3 and 4-7 the softmax of row tile 0 and 1, 8-11 the output of
// both, 12 loads Q and K, 13 and 14 issue the MMAs of tile 0 and 1, 15 finds the
// items and loads V (whose ring may be full while a K tile is needed).
//
// Softmax in base 2.  The maximum that scales the exponentials may lag the true
// running maximum by up to 2^8 (kLag); O in TMEM is only rescaled, by the
// warp whose rows need it, when the lag would grow beyond that.  The final
// division makes the result independent of it.  P is rounded to the input type
// for the second product; the row sums are of the unrounded values, in fp32.
//
// What bounds it.  Of a K/V tile and both row tiles the tensor core has 2048
// clocks of work (D = 128), the special-function units 2048; a round takes 3000
// (time x sampled clock over rounds an SM, 16384 to 65536 tokens): the way of one row
// tile from a finished S through its exponentials, the rest of PV and the next S,
// and two barriers.  One prompt of 8192 tokens, 32 / 8 heads of 128, bf16: 401 to 417
// us (1320 to 1370 TFLOP/s) in short runs at 1.73 GHz, 466 to 480 us (1150 to 1180
// TFLOP/s) without pause, where the power limit holds the clock at 1.5 GHz.  Short
// prompts lose as much between items: 24 packed ones of 16 to 1500 tokens take 95 to
// 98 us (680 to 700 TFLOP/s), 159 thousand clocks for 33 rounds and 8.5 items an SM,
// so some 7000 an item beside its rounds; MLA heads (192 / 128, 2700 clocks a round of
// 96 keys) of 500 to 2048 tokens 239 to 245 us (780 to 800 TFLOP/s), 366 thousand for
// 105 rounds and 9.9 items, 8400 an item.  In these are the start, the uneven end
// and the change of items; they were not told apart.  13% of the MLA products are
// masked parts of diagonal tiles.  Finding an item reads all lengths again where there
// are more than 32: 32, 64, 256 and 1024 prompts of 100 tokens, 32 / 8 heads, take 27,
// 49, 310 and 3930 us.  Heads of 64: 28 / 4 heads, 4096 tokens 92 us, 16384 1220 us
// (790 TFLOP/s; 3000 clocks a round again, with 1024 of work for the tensor core and
// 2048 for the special-function units).
// The instructions of a round should stay in cache: one copy of the tile code for
// whole and masked tiles, 16 KB less, took 500 us to 485.  Nor is there a register to
// spare: what all warps use is spilled when any of them needs more.
// Not adopted: a quarter or half of the exponentials by polynomial (no gain once
// the registers sufficed, 2.5% at D = 64), two threads a row (the maximum has to
// be agreed on: 611 us), spinning instead of suspended waits (3% slower).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "frn_internal.h"
#include "frn_ptx.cuh"
#include "frn_take_over.h"

namespace frn {

constexpr int kPromptThreads = 512;
constexpr int kRows = 128;   // rows of a tile
// Warps: 0-3 and 4-7 softmax of row tile 0 and 1, 8-11 output.
constexpr int kOut = 8, kLoadQK = 12, kMma = 13, kLoadV = 15;
constexpr int kAhead = 6;      // K/V tiles before its end that an item's successor is found
constexpr int kItemSlots = 4;  // items that the scheduler is ahead
constexpr float kLag = 8.f;    // log2 of the most that a probability may exceed 1
constexpr float kFar = 0x1p14f;   // scaled scores from which on differences are taken first
constexpr float kFloor = -FLT_MAX;  // least first maximum: scores of -inf alone are not one

// Two row tiles of one KV head: tokens from t0 on of the sequence in rows
// [first, first + len).  len = 0: no more items.
struct PromptItem {
  int32_t first, len, t0, kvh;
};

template <int DQK, int DV>
struct PromptCfg {
  static constexpr int QH = DQK / 64, VH = DV / 64;  // 64-column halves (128-byte rows)
  // Keys of a K/V tile.  With 192 columns 96 of them, so that K and V tiles fit
  // twice beside the two Q tiles (with 128 a second V tile does not, and every
  // tile waits for its V: 308 us for four sequences of 500 to 2048 tokens, 64
  // heads, 289 with 96, both before the later steps; with 64 a product takes 48
  // clocks of the tensor core where 32 would do, for its operands' shared-memory
  // reads).
  static constexpr int KEYS = DQK == 192 ? 96 : 128;
  static constexpr int MOST = KEYS - 32;             // keys whose P is announced before the rest
  static constexpr int QHALF = kRows * 128;          // bytes of 128 rows x 64 columns
  static constexpr int HALF = KEYS * 128;            // and of a K/V tile's
  static constexpr int Q_BYTES = QH * QHALF, K_BYTES = QH * HALF, V_BYTES = VH * HALF;
  // As many K and V tiles as fit.
  static constexpr int NK = DQK == 64 ? 5 : 2;
  static constexpr int NV = DQK == 64 ? 5 : 2;
  // Staging of an output warp: pieces of 32 rows x 32 columns.
  static constexpr int NOUT = DQK == 128 ? 4 : DQK == 192 ? 1 : 2;
  static constexpr int OFF_K = 2 * Q_BYTES;
  static constexpr int OFF_V = OFF_K + NK * K_BYTES;
  static constexpr int OFF_OUT = OFF_V + NV * V_BYTES;
  static constexpr int OFF_BAR = OFF_OUT + 4 * NOUT * 2048;
  static constexpr int OFF_ITEMS = OFF_BAR + (20 + 2 * NK + 2 * NV + 2 * kItemSlots) * 8;
  static constexpr int OFF_L = OFF_ITEMS + kItemSlots * 16 + 32;  // [parity][row tile][row] sums
  static constexpr int SMEM_BYTES = OFF_L + 2048;
  static_assert(SMEM_BYTES <= 232448, "shared memory of one SM");
  // TMEM columns: S_0, S_1 (P_s in the first half of S_s), O_0, O_1.
  static constexpr uint32_t TM_S = 0, TM_O = 256, TM_COLS = 512;
};

struct PromptParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;  // elements
  const int32_t* cu;
  int32_t batch, tokens, max_seqlen, group, hkv, tq, heads_at_once;
  float qscale;     // |scale| * log2(e), never zero
  uint32_t negate;  // scale < 0: S is computed with Q negated
  uint64_t timeout_ns;
};

// D(tmem) (+)= A(tmem, 16-bit pairs) * B(smem).
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Descriptor of a B operand whose rows run along the contraction (keys): rows
// of 64 columns (128 bytes, 128-byte swizzle), 8-row groups 1024 bytes apart
// (stride offset), the next 64 columns `half_bytes` further (leading offset).
__device__ __forceinline__ uint64_t make_smem_desc_mn_sw128(uint32_t smem_byte_addr,
                                                            uint32_t half_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_byte_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(half_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

// Two fp32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Asks for the number of a CTA of this grid that has not been launched yet, which
// then never will be; the 16-byte answer completes on `bar`.
__device__ __forceinline__ void take_cta(void* answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128"
      " [%0], [%1];" ::"r"(smem_addr(answer)),
      "r"(smem_addr(bar))
      : "memory");
}

// The answer: false if there was no such CTA (after which none may be asked for).
__device__ __forceinline__ bool taken_cta(const void* answer, uint32_t& cta) {
  uint32_t yes, x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 a;\n\t.reg .b32 y, z, w;\n\t"
      "mov.b32 %1, 0;\n\t"
      "ld.shared.b128 a, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, a;\n\t}"
      : "=&r"(yes), "=&r"(x)
      : "r"(smem_addr(answer))
      : "memory");
  cta = x;
  return yes != 0;
}

// Moves registers between the warpgroups: all warps of one execute it.
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// All N columns of this lane's row of scores: as many as `x` has room for.
template <int N>
__device__ __forceinline__ void tmem_ld_row(uint32_t taddr, float (&x)[N]) {
  static_assert(N % 32 == 0, "whole loads of 32 columns");
#pragma unroll
  for (int c = 0; c < N / 32; ++c)
    tmem_ld_32x32b_x32(taddr + c * 32, reinterpret_cast<uint32_t(&)[32]>(x[c * 32]));
}

__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* m, uint64_t* bar,
                                            int32_t c0, int32_t c1, int32_t c2, int32_t c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_addr(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_addr(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// True in one lane of a converged warp.  Unlike a test of the lane number this
// tells the compiler that the branch is for a single thread, so that the MMA's
// uniform operands need no loop over lanes: the eight MMAs of a PV are issued in
// 450 clocks instead of 770 (8192 tokens, without the later steps: 586 us instead of
// 669).
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0;
}

__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap* m, int32_t c0, int32_t c1,
                                                int32_t c2, int32_t c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, uint32_t smem_src, int32_t c0,
                                             int32_t c1, int32_t c2, int32_t c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::
          "l"(reinterpret_cast<uint64_t>(m)),
      "r"(smem_src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ float prompt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows [first, first + len) of sequence b, cut to the call's limits.
__device__ __forceinline__ void sequence_of(const PromptParams& p, int b, int32_t& first,
                                            int32_t& len) {
  const int64_t a = p.cu[b], e = p.cu[b + 1];
  int64_t a2 = a < 0 ? 0 : a, e2 = e > p.tokens ? p.tokens : e;
  if (e2 - a2 > p.max_seqlen) e2 = a2 + p.max_seqlen;
  if (a2 != a || e2 != e) atomicOr(&g_frn_device_error, kDevErrBadLength);
  first = static_cast<int32_t>(a2);
  len = e2 > a2 ? static_cast<int32_t>(e2 - a2) : 0;
}


// Finds the items of the CTA, in the order of falling block number, for a whole
// warp.  F(L) = items of block number >= L = sum_b max(0, blocks_b - L) falls
// with L; item number `index` has as its block the largest L with F(L) > index,
// and it is the (index - F(L + 1))-th sequence that has such a block.  32 levels
// are tried at a time, one a lane; the first 32 sequences stay in registers.
struct ItemFinder {
  int32_t first, blocks, len;  // this lane's of the first 32 sequences
  int32_t below;               // the level is below this: it falls as the number grows
  int32_t last;                // the last number looked for
  bool more;                   // more than 32 sequences

  __device__ __forceinline__ void look(const PromptParams& p, int b) {
    const int32_t per = 2 * p.tq;
    blocks = len = first = 0;
    if (b < p.batch) {
      sequence_of(p, b, first, len);
      blocks = (len + per - 1) / per;
    }
  }

  __device__ __forceinline__ int32_t most(const PromptParams& p) {
    return (p.max_seqlen + 2 * p.tq - 1) / (2 * p.tq);
  }

  __device__ __forceinline__ void start(const PromptParams& p) {
    below = most(p);
    last = 0;
    more = p.batch > 32;
    look(p, static_cast<int>(threadIdx.x & 31));
  }

  // F at this lane's level.
  __device__ __forceinline__ int32_t count(const PromptParams& p, int32_t level) {
    int32_t n = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      if (more) look(p, b0 + static_cast<int>(threadIdx.x & 31));
#pragma unroll 4
      for (int i = 0; i < min(32, p.batch - b0); ++i)
        n += max(0, __shfl_sync(0xffffffffu, blocks, i) - level);
    }
    return n;
  }

  __device__ __forceinline__ bool find(const PromptParams& p, int32_t index, PromptItem& item) {
    const int lane = static_cast<int>(threadIdx.x & 31);
    if (index < last) below = most(p);
    last = index;
    int32_t lo = 0, hi = below;  // F(lo) > index >= F(hi), if there is such an item
    int32_t above = 0;           // F(hi)
    bool first_round = true;
    while (hi - lo > 1 || first_round) {
      const int32_t step = (hi - lo + 31) / 32;
      const int32_t level = lo + lane * step;
      const int32_t n = count(p, min(level, hi));
      const uint32_t yes = __ballot_sync(0xffffffffu, level < hi && n > index);
      if (yes == 0) return false;
      const int top = 31 - __clz(yes);
      const int32_t next = __shfl_sync(0xffffffffu, n, min(top + 1, 31));
      if (top < 31 && lo + (top + 1) * step < hi) {
        above = next;
        hi = lo + (top + 1) * step;
      } else if (first_round) {
        above = count(p, hi);
      }
      lo += top * step;
      first_round = false;
    }
    below = lo + 1;
    int32_t k = index - above;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      if (more) look(p, b0 + lane);
      uint32_t mask = __ballot_sync(0xffffffffu, blocks > lo);
      if (k < __popc(mask)) {
        for (; k > 0; --k) mask &= mask - 1;
        const int src = __ffs(mask) - 1;
        item.first = __shfl_sync(0xffffffffu, first, src);
        item.len = __shfl_sync(0xffffffffu, len, src);
        item.t0 = lo * 2 * p.tq;
        return true;
      }
      k -= __popc(mask);
    }
    return false;
  }
};

// Two 16-bit elements: their exponents, all ones in one that is not finite.
template <typename T>
__device__ __forceinline__ uint32_t odd_halves(uint32_t pair) {
  constexpr uint32_t kExp = Elem16<T>::kUmmaFormat == 0u ? 0x7c00u : 0x7f80u;
  return ((pair & kExp) == kExp ? 0xffffu : 0u) |
         ((pair & (kExp << 16)) == kExp << 16 ? 0xffff0000u : 0u);
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t row_pair) {
  uint32_t t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(row_pair));
  return t;
}

// The rows of a warp whose product with V met a NaN or an infinity at a position
// that the row does not see (zero weight times that is not zero), computed once
// more by the warp alone: 8 rows and 64 columns of V at a time, 16 keys a step, on
// 16x8x16 MMAs (S^T = K Q^T, O^T += V^T P^T) whose operands come straight from
// memory (the contraction of Q and K takes the head dims in an order in which a
// lane's are 16 bytes).  Steps whose keys not every row sees take V without such
// values and then add those that a row does see by themselves.  `rows` are the
// lanes whose rows hold a value that is not finite, `tok` and `head` the lane's
// row; the warp's first row is token tok0.
// Bound by the latency of its loads.  One NaN in V at the end of a prompt makes 128
// rows a KV head do this: 8192 tokens, 32 / 8 heads of 128, 5.6 ms instead of 0.42;
// 65536 tokens, 4 heads of 64 on one, 18 instead of 2.6; an infinity in the same
// column of every token makes all rows do it, 37 ms for the first of these.  (A key
// at a time, in one chain, it would be some 450 clocks a key and row.)  16 rows at a
// time take more registers than the output warps have: values that all warps use
// are spilled for it, and 77 tokens with heads of 64 take 9.4 us instead of 7.7.
template <typename T, int DQK, int DV>
__device__ __noinline__ void redo_rows(const PromptParams& p, uint32_t rows, int32_t first,
                                       int32_t tok0, int32_t tok, int kvh, int head,
                                       int32_t covered, volatile uint32_t* abort_flag) {
  const int lane = static_cast<int>(threadIdx.x & 31), g = lane >> 2, tq = lane & 3;
  const T* k = static_cast<const T*>(p.k) + first * p.k_token + kvh * p.k_head + tq * 8;
  const T* v0 = static_cast<const T*>(p.v) + first * p.v_token + kvh * p.v_head;
  // The last position that the rows' products covered and that holds such a value.
  int32_t last = -1;
  for (int32_t i = lane; i < (covered - tok0 - 1) * (DV / 8); i += 32) {
    const int32_t j = tok0 + 1 + i / (DV / 8);
    const uint4 x =
        *reinterpret_cast<const uint4*>(v0 + j * p.v_token + i % (DV / 8) * 8);
    if (odd_halves<T>(x.x) | odd_halves<T>(x.y) | odd_halves<T>(x.z) | odd_halves<T>(x.w))
      last = j;
  }
  last = __reduce_max_sync(0xffffffffu, last);
  rows &= __ballot_sync(0xffffffffu, tok < last);  // the others' own keys gave the value
  const float qs = p.negate ? -p.qscale : p.qscale;
  constexpr float kUp = Elem16<T>::kUmmaFormat == 0u ? 15.f - kLag : 0.f;
  constexpr int NC = 2;  // 32-column pieces of V at a time
  while (rows) {
    // The 8 rows of a pass, the last one standing in for those that are missing: the
    // queries of row g, and the results of rows 2 tq and 2 tq + 1.
    const int most = __popc(rows) - 1;
    const int src = static_cast<int>(__fns(rows, 0, min(g, most) + 1));
    const int32_t my_row = __shfl_sync(0xffffffffu, tok, src);
    const int my_head = __shfl_sync(0xffffffffu, head, src);
    for (int i = 0; i < 8; ++i) rows &= rows - 1;
    const T* q = static_cast<const T*>(p.q) + (first + my_row) * p.q_token + my_head * p.q_head + tq * 8;
    const int32_t row[2] = {__shfl_sync(0xffffffffu, my_row, tq * 8),
                            __shfl_sync(0xffffffffu, my_row, tq * 8 + 4)};
    const int32_t seen_by_all = __reduce_min_sync(0xffffffffu, my_row) + 1;
    const int32_t end = __reduce_max_sync(0xffffffffu, my_row) + 1;
#pragma unroll 1
    for (int c0 = 0; c0 < DV; c0 += 32 * NC) {
      const T* v = v0 + c0 + tq * 8;
      float acc[2 * NC][4], m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2 * NC; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll 1
      for (int32_t j0 = 0; j0 < end; j0 += 16) {
        const bool masked = j0 + 16 > seen_by_all;
        float x[4] = {0.f, 0.f, 0.f, 0.f};  // key g (0, 1), g + 8 (2, 3) of rows 2 tq (0, 2), 2 tq + 1
        const int32_t ja = min(j0 + g, end - 1), jb = min(j0 + 8 + g, end - 1);
#pragma unroll 2
        for (int c = 0; c < DQK; c += 32) {
          const uint4 qa = *reinterpret_cast<const uint4*>(q + c);
          const uint4 ka = *reinterpret_cast<const uint4*>(k + ja * p.k_token + c);
          const uint4 kb = *reinterpret_cast<const uint4*>(k + jb * p.k_token + c);
          const uint32_t lo[4] = {ka.x, kb.x, ka.y, kb.y}, hi[4] = {ka.z, kb.z, ka.w, kb.w};
          mma_16816<T>(x, lo, qa.x, qa.y);
          mma_16816<T>(x, hi, qa.z, qa.w);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          x[r] = j0 + g <= row[r] ? x[r] * qs : -INFINITY;
          x[r + 2] = j0 + 8 + g <= row[r] ? x[r + 2] * qs : -INFINITY;
          float m_new = fmaxf(m[r], fmaxf(x[r], x[r + 2]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1)
            m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, o));
          const float c = exp2f(m[r] - m_new);
          m[r] = m_new;
          l[r] *= c;
#pragma unroll
          for (int i = 0; i < 2 * NC; ++i) {
            acc[i][r] *= c;
            acc[i][r + 2] *= c;
          }
          x[r] = exp2f((x[r] - m_new) + kUp);
          x[r + 2] = exp2f((x[r + 2] - m_new) + kUp);
          l[r] += x[r] + x[r + 2];
        }
        const uint32_t p0 = transpose_8x8(float2_to_pair<T>(x[0], x[1]));
        const uint32_t p1 = transpose_8x8(float2_to_pair<T>(x[2], x[3]));
        uint32_t odd = 0;  // of keys g (low half) and g + 8
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint4 va = *reinterpret_cast<const uint4*>(v + ja * p.v_token + c * 32);
          const uint4 vb = *reinterpret_cast<const uint4*>(v + jb * p.v_token + c * 32);
          uint32_t a[4] = {va.x, va.y, va.z, va.w}, b[4] = {vb.x, vb.y, vb.z, vb.w};
          if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t oa = odd_halves<T>(a[i]), ob = odd_halves<T>(b[i]);
              odd |= (oa ? 1u : 0u) | (ob ? 2u : 0u);
              a[i] &= ~oa;
              b[i] &= ~ob;
            }
          }
          // Rows of a product: 8 columns of each of two words.
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const uint32_t vt[4] = {transpose_8x8(a[i]), transpose_8x8(a[i + 1]),
                                    transpose_8x8(b[i]), transpose_8x8(b[i + 1])};
            mma_16816<T>(acc[c * 2 + i / 2], vt, p0, p1);
          }
        }
        if (masked) {
          const uint32_t lanes_a = __ballot_sync(0xffffffffu, odd & 1u);
          const uint32_t lanes_b = __ballot_sync(0xffffffffu, odd & 2u);
#pragma unroll 1
          for (int t = 0; t < 16 && j0 + t < end; ++t) {
            if (!((t < 8 ? lanes_a : lanes_b) >> ((t & 7) * 4) & 15u)) continue;
            // The weights of key t, from the lanes that hold them.
            const int from = (t & 7) * 4 + tq;
            const float w0 = __shfl_sync(0xffffffffu, t < 8 ? x[0] : x[2], from);
            const float w1 = __shfl_sync(0xffffffffu, t < 8 ? x[1] : x[3], from);
            // Results of this lane: column (g / 2) * 8 + 2 i + g % 2 of word i.
            const T* vr = v0 + c0 + (j0 + t) * p.v_token + (g >> 1) * 8 + (g & 1);
#pragma unroll
            for (int i = 0; i < 4 * NC; ++i) {
              const float y = static_cast<float>(vr[(i / 4) * 32 + (i % 4) * 2]);
              float* o = acc[i / 2] + (i & 1) * 2;
              if (!isfinite(y)) {
                if (j0 + t <= row[0]) o[0] = fmaf(w0, y, o[0]);
                if (j0 + t <= row[1]) o[1] = fmaf(w1, y, o[1]);
              }
            }
          }
        }
        bool lost = true;
#pragma unroll
        for (int i = 0; i < 2 * NC; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) lost &= isnan(acc[i][e]);
        if (__all_sync(0xffffffffu, lost)) break;  // NaN everywhere stays so
        if (__any_sync(0xffffffffu, *abort_flag)) return;
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
        const float inv = 1.f / l[r];
        T* out = static_cast<T*>(p.out) + (first + row[r]) * p.out_token +
                 __shfl_sync(0xffffffffu, my_head, tq * 8 + r * 4) * p.out_head + c0 +
                 (g >> 1) * 8 + (g & 1);
#pragma unroll
        for (int i = 0; i < 4 * NC; ++i)
          out[(i / 4) * 32 + (i % 4) * 2] = static_cast<T>(acc[i / 2][(i & 1) * 2 + r] * inv);
      }
    }
  }
}

template <typename T, int DQK, int DV>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_attention_kernel(const __grid_constant__ CUtensorMap tmap_q,
                            const __grid_constant__ CUtensorMap tmap_k,
                            const __grid_constant__ CUtensorMap tmap_v,
                            const __grid_constant__ CUtensorMap tmap_o,
                            const __grid_constant__ PromptParams p) {
  using C = PromptCfg<DQK, DV>;
  constexpr int kKeys = C::KEYS;
  extern __shared__ __align__(1024) uint8_t smem[];  // no room to align it here
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_empty = q_full + 2;
  uint64_t* k_full = q_empty + 2;
  uint64_t* k_empty = k_full + C::NK;
  uint64_t* v_full = k_empty + C::NK;
  uint64_t* v_empty = v_full + C::NV;
  uint64_t* s_full = v_empty + C::NV;
  uint64_t* p_ready = s_full + 2;
  uint64_t* p_most = p_ready + 2;
  uint64_t* o_full = p_most + 2;
  uint64_t* o_empty = o_full + 2;
  uint64_t* l_full = o_empty + 2;
  uint64_t* i_full = l_full + 4;
  uint64_t* i_empty = i_full + kItemSlots;
  uint64_t* answer_full = i_empty + kItemSlots;
  PromptItem* items = reinterpret_cast<PromptItem*>(smem + C::OFF_ITEMS);
  uint8_t* answer = smem + C::OFF_ITEMS + kItemSlots * 16;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(answer + 16);
  uint32_t* tmem_ptr = const_cast<uint32_t*>(abort_flag) + 1;

  const int warp = static_cast<int>(warp_id_in_cta()), lane = static_cast<int>(threadIdx.x & 31);
  const uint64_t to = p.timeout_ns;

  if (warp == kLoadQK && lane == 0) {
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
    prefetch_tmap(&tmap_o);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);  // the tile's softmax warps
      mbar_init(&p_most[i], 5);   // and the other tile's MMA warp, handing over
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 4);  // the output warps
      mbar_init(&l_full[i], 4);  // [row tile], then the second slots
      mbar_init(&l_full[2 + i], 4);
    }
    for (int i = 0; i < C::NK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);  // both MMA warps
    }
    for (int i = 0; i < C::NV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 2);
    }
    mbar_init(answer_full, 1);
    for (int i = 0; i < kItemSlots; ++i) {
      mbar_init(&i_full[i], 1);
      mbar_init(&i_empty[i], kPromptThreads / 32);  // every warp
    }
    *abort_flag = 0u;
    fence_mbarrier_init();
  }
  if (warp == kMma) {
    tmem_alloc(tmem_ptr, C::TM_COLS);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  griddep_launch_dependents();
  griddep_wait();

  // The it-th item of this CTA, copied from the scheduler's slots.
  auto next_item = [&](int32_t it, PromptItem& item) {
    const int slot = it % kItemSlots;
    if (!mbar_wait(&i_full[slot], static_cast<uint32_t>(it / kItemSlots) & 1u, abort_flag, to))
      return false;
    item = items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&i_empty[slot]);
    return item.len > 0;
  };
  // Row tile s of an item: tokens [t0 + s TQ, end), K/V tiles.
  auto end_of = [&](const PromptItem& item, int s) {
    return min(item.len, item.t0 + (s + 1) * p.tq);
  };
  auto tiles_of = [&](const PromptItem& item, int s) {
    return item.t0 + s * p.tq < item.len ? (end_of(item, s) + kKeys - 1) / kKeys : 0;
  };

  if (warp >= kLoadQK) {
    reg_dec<56>();
    if (warp == kLoadQK) {
      // ---- loads of Q and K
      const uint32_t q_bytes = static_cast<uint32_t>(C::QH * 128 * p.group * p.tq);
      PromptItem item;
      uint32_t nk = 0, nq[2] = {0, 0};
      bool ok = true;
      for (int32_t it = 0; ok && next_item(it, item); ++it) {
        const int32_t n = max(tiles_of(item, 0), tiles_of(item, 1));
        auto load_q = [&](int s) {
          if (tiles_of(item, s) == 0) return;
          ok = ok && mbar_wait(&q_empty[s], (nq[s] & 1u) ^ 1u, abort_flag, to);
          ++nq[s];
          if (ok && lane == 0) {
            mbar_arrive_expect_tx(&q_full[s], q_bytes);
            for (int h = 0; h < C::QH; ++h)
              tma_load_4d(smem + s * C::Q_BYTES + h * C::QHALF, &tmap_q, &q_full[s], h * 64, 0,
                          item.kvh, item.first + item.t0 + s * p.tq);
          }
        };
        auto load_k = [&](int32_t j) {
          const uint32_t ks = nk % C::NK;
          ok = ok && mbar_wait(&k_empty[ks], ((nk / C::NK) & 1u) ^ 1u, abort_flag, to);
          ++nk;
          if (ok && lane == 0) {
            mbar_arrive_expect_tx(&k_full[ks], C::K_BYTES);
            for (int h = 0; h < C::QH; ++h)
              tma_load_3d(smem + C::OFF_K + ks * C::K_BYTES + h * C::HALF, &tmap_k, &k_full[ks],
                          h * 64, item.kvh, item.first + j * kKeys);
          }
        };
        // Q waits for the last item's scores; L2 can have it already.
        if (it > 0 && lane < 2 * C::QH) {
          const int s = lane / C::QH;
          if (tiles_of(item, s) > 0)
            tma_prefetch_4d(&tmap_q, (lane % C::QH) * 64, 0, item.kvh,
                            item.first + item.t0 + s * p.tq);
        }
        __syncwarp();
        load_q(0);
        load_k(0);
        load_q(1);
        for (int32_t j = 1; j < n && ok; ++j) load_k(j);
      }
      if (*abort_flag) __nanosleep(20000);  // loads already issued may still be landing
    } else if (warp == kLoadV) {
      // ---- items and loads of V.  The first item is the CTA's own number; then
      // it takes those of CTAs that have not been launched yet, each a few tiles
      // before the one before ends: earlier, and an item would wait here while
      // another SM is idle; later, and this SM waits for its first tiles.
      bool ok = true, done = false;
      ItemFinder finder;
      finder.start(p);
      // Blocks of all sequences, for one head.  Items are fewer than 2^31: their
      // numbers are those of CTAs.
      const int32_t blocks = finder.count(p, 0);
      const int64_t items_of_call = static_cast<int64_t>(blocks) * p.hkv;
      const int32_t per_group = static_cast<int32_t>(
          min(static_cast<int64_t>(blocks) * p.heads_at_once, static_cast<int64_t>(0x7fffffff)));
      int32_t last_group = -1;
      uint32_t answers = 0;
      auto ask = [&]() {
        fence_proxy_async_smem();  // the last answer has been read
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_expect_tx(answer_full, 16);
          take_cta(answer, answer_full);
        }
      };
      auto hear = [&](int32_t& index) {
        ok = ok && mbar_wait(answer_full, answers++ & 1u, abort_flag, to);
        uint32_t cta = 0;
        const bool got = ok && taken_cta(answer, cta);
        index = static_cast<int32_t>(cta);
        return got;
      };
      // The item of a number, if it has one: the grid is an upper bound.
      auto item_of = [&](int32_t index, PromptItem& item) {
        if (index >= items_of_call) return false;
        const int32_t group = index / per_group;
        const int32_t head0 = group * p.heads_at_once;
        const int32_t heads = min(p.heads_at_once, p.hkv - head0);
        if (group != last_group) finder.below = finder.most(p);
        last_group = group;
        index -= group * per_group;
        const int32_t block = index / heads;
        item.kvh = head0 + index - block * heads;
        return finder.find(p, block, item);
      };
      auto publish = [&](int32_t it) {
        if (done || !ok) return;
        PromptItem item;
        done = !next_number(it == 0, static_cast<int32_t>(blockIdx.x), ask, hear,
                            [&](int32_t index) { return item_of(index, item); });
        if (!ok) return;
        if (done) item.len = 0;  // the end
        const int slot = it % kItemSlots;
        ok = ok && mbar_wait(&i_empty[slot], (static_cast<uint32_t>(it / kItemSlots) & 1u) ^ 1u,
                             abort_flag, to);
        if (ok && lane == 0) {
          items[slot] = item;
          mbar_arrive(&i_full[slot]);
        }
        __syncwarp();
      };
      PromptItem item;
      uint32_t nv = 0;
      publish(0);
      for (int32_t it = 0; ok && next_item(it, item); ++it) {
        const int32_t n = max(tiles_of(item, 0), tiles_of(item, 1));
        for (int32_t j = 0; j < n && ok; ++j, ++nv) {
          const uint32_t vs = nv % C::NV;
          ok = mbar_wait(&v_empty[vs], ((nv / C::NV) & 1u) ^ 1u, abort_flag, to);
          if (ok && lane == 0) {
            mbar_arrive_expect_tx(&v_full[vs], C::V_BYTES);
            for (int h = 0; h < C::VH; ++h)
              tma_load_3d(smem + C::OFF_V + vs * C::V_BYTES + h * C::HALF, &tmap_v, &v_full[vs],
                          h * 64, item.kvh, item.first + j * kKeys);
          }
          if (j == max(0, n - kAhead)) publish(it + 1);
        }
      }
      if (*abort_flag) __nanosleep(20000);  // loads already issued may still be landing
    } else {
      // ---- MMAs of row tile s: the whole warp runs the loop, one lane issues.
      // What lies between a P and the next S is on the critical path, and waiting
      // for a barrier costs two MMAs' time even if it is complete: one warp for
      // both row tiles left the tensor core idle a third of the time.  The warps
      // take turns, a PV and the following S at a time: left alone they fall
      // into step, both softmaxes together, then both products (18% slower).
      // A K/V tile is released by both warps; one whose row tile does not reach
      // it waits for it all the same, to count in the right phase.
      const int s = warp - kMma;
      const uint32_t base = smem_addr(smem);
      constexpr uint32_t kFmt = Elem16<T>::kUmmaFormat;
      constexpr uint32_t kSteps = kKeys / 16;
      constexpr uint32_t kIdescPV = make_idesc_f16(kFmt, kRows, DV) | (1u << 16);  // B along keys
      const uint32_t idesc_qk = make_idesc_f16(kFmt, kRows, 0) | (p.negate << 13);
      const uint64_t qd = make_smem_desc_k_sw128(base + s * C::Q_BYTES);
      const uint64_t kd0 = make_smem_desc_k_sw128(base + C::OFF_K);
      const uint64_t vd0 = make_smem_desc_mn_sw128(base + C::OFF_V, C::HALF);
      const uint32_t tm_s = tmem + C::TM_S + s * 128, tm_o = tmem + C::TM_O + s * DV;
      uint32_t ks = 0, kp = 0, vs = 0, vp = 0, qp = 0, pp = 0;  // ring slots and parities
      uint32_t mp = 0, op = 1;
      bool ok = true;
      // MMA steps (16 keys) of the row tile's last K/V tile.
      auto last_steps = [&](const PromptItem& x, int32_t nt) {
        return static_cast<uint32_t>(end_of(x, s) - (nt - 1) * kKeys + 15) / 16u;
      };
      // The operands of an item's K tile j have arrived.
      auto wait_qk = [&](int32_t j, int32_t nt) {
        if (j == 0 && nt > 0) {
          ok = ok && mbar_wait(&q_full[s], qp, abort_flag, to);
          qp ^= 1u;
        }
        ok = ok && mbar_wait(&k_full[ks], kp, abort_flag, to);
      };
      // By one lane: S of that tile, if the row tile has it.
      auto issue_qk = [&](int32_t j, int32_t nt, uint32_t ragged) {
        if (j < nt) {
          const bool last = j + 1 == nt;
          const uint32_t idesc = idesc_qk | ((last ? ragged : kSteps) << 18);  // N = 16 a step
          const uint64_t kd = kd0 + ks * (C::K_BYTES >> 4);
#pragma unroll
          for (int i = 0; i < DQK / 16; ++i) {
            umma_f16_ss(tm_s, qd + (((i / 4) * C::QHALF + (i % 4) * 32) >> 4),
                        kd + (((i / 4) * C::HALF + (i % 4) * 32) >> 4), idesc, i > 0);
          }
          umma_commit(&s_full[s]);
          umma_commit(&k_empty[ks]);
          if (last) umma_commit(&q_empty[s]);
        } else {
          mbar_arrive(&k_empty[ks]);
        }
      };
      // By one lane: steps [from, upto) of O += P V.
      auto pv_steps = [&](auto from, auto upto, uint32_t steps, uint64_t vd, bool fresh) {
        if (steps == kSteps) {
#pragma unroll
          for (int i = decltype(from)::value; i < decltype(upto)::value; ++i)
            umma_f16_ts(tm_o, tm_s + i * 8, vd + ((i * 2048) >> 4), kIdescPV, !fresh || i > 0);
        } else {
#pragma unroll 1
          for (int i = decltype(from)::value;
               i < min(decltype(upto)::value, static_cast<int>(steps)); ++i)
            umma_f16_ts(tm_o, tm_s + i * 8, vd + ((i * 2048) >> 4), kIdescPV, !fresh || i > 0);
        }
      };
      constexpr std::integral_constant<int, 0> kFirst{};
      constexpr std::integral_constant<int, C::MOST / 16> kRest{};
      constexpr std::integral_constant<int, kKeys / 16> kEnd{};
      auto next_k = [&]() {
        if (++ks == C::NK) {
          ks = 0;
          kp ^= 1u;
        }
      };
      // The turn, and most of P with it: one wait for both.  Where there is no P
      // to wait for, this warp stands in for the softmax warps.
      auto take_turn = [&](bool with_p) {
        if (!with_p && lane < 4) mbar_arrive(&p_most[s]);
        ok = ok && mbar_wait(&p_most[s], mp, abort_flag, to);
        mp ^= 1u;
      };
      if (s == 0 && lane == 0) mbar_arrive(&p_most[0]);  // row tile 0 begins
      PromptItem item, next;
      bool some = next_item(0, item);
      int32_t nt = 0, other = 0;
      uint32_t ragged = 0;
      if (some) {
        nt = tiles_of(item, s);
        other = tiles_of(item, s ^ 1);
        ragged = last_steps(item, nt);
        wait_qk(0, nt);
        take_turn(false);
        if (ok && elect_one()) {
          issue_qk(0, nt, ragged);
          mbar_arrive(&p_most[s ^ 1]);
        }
        __syncwarp();
        next_k();
      }
      for (int32_t it = 0; some && ok; ++it) {
        const int32_t n = max(nt, other);
        bool more = false;
        int32_t next_nt = 0, next_other = 0;
        uint32_t next_ragged = 0;
        for (int32_t j = 0; j < n && ok; ++j) {
          // Everything else that PV(j) and what follows it need, before P.
          bool follows = true;
          if (j + 1 < n) {
            wait_qk(j + 1, nt);
          } else {
            follows = more = next_item(it + 1, next);
            if (more) {
              next_nt = tiles_of(next, s);
              next_other = tiles_of(next, s ^ 1);
              next_ragged = last_steps(next, next_nt);
              wait_qk(0, next_nt);
            }
          }
          ok = ok && mbar_wait(&v_full[vs], vp, abort_flag, to);
          if (j == 0 && nt > 0) {  // the last item's output is out of TMEM
            ok = ok && mbar_wait(&o_empty[s], op, abort_flag, to);
            op ^= 1u;
          }
          if (!ok) break;
          const bool here = j < nt, last = j + 1 == nt;
          const uint32_t steps = last ? ragged : kSteps;
          const uint64_t vd = vd0 + vs * (C::V_BYTES >> 4);
          if (here) {
            const int32_t left = item.len - j * kKeys;
            if (left < kKeys && (left & 15)) {
              // The last MMA step reaches past the sequence: what lies there has
              // weight zero, but zero times a NaN or infinity is not zero.
              // (Both MMA warps may write these zeros.)
              const int rows = 16 - (left & 15);
              for (int i = lane; i < rows * 8 * C::VH; i += 32) {
                const int r = left + i / (8 * C::VH), c = i % (8 * C::VH);
                st_shared_v4(base + C::OFF_V + vs * C::V_BYTES + (c / 8) * C::HALF + r * 128 +
                                 (c % 8) * 16,
                             0, 0, 0, 0);
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
          }
          take_turn(here);
          if (!ok) break;
          if (here) {
            tc_fence_after();
            if (elect_one()) pv_steps(kFirst, kRest, steps, vd, j == 0);
            __syncwarp();
            ok = mbar_wait(&p_ready[s], pp, abort_flag, to);
            pp ^= 1u;
            if (!ok) break;
            tc_fence_after();
          }
          if (elect_one()) {
            if (here) {
              pv_steps(kRest, kEnd, steps, vd, false);
              if (last) umma_commit(&o_full[s]);
            }
            if (follows) issue_qk(j + 1 < n ? j + 1 : 0, j + 1 < n ? nt : next_nt,
                                  j + 1 < n ? ragged : next_ragged);
            mbar_arrive(&p_most[s ^ 1]);
            if (here)
              umma_commit(&v_empty[vs]);
            else
              mbar_arrive(&v_empty[vs]);
          }
          __syncwarp();
          if (follows) next_k();
          if (++vs == C::NV) {
            vs = 0;
            vp ^= 1u;
          }
        }
        item = next;
        some = more;
        nt = next_nt;
        other = next_other;
        ragged = next_ragged;
      }
    }
  } else if (warp >= kOut) {
    reg_dec<88>();
    // ---- output: O over the row's sum, while the softmax warps go on with the
    // next item
    const int row = (warp & 3) * 32 + lane;
    const int row_tok = row / p.group, row_head = row - row_tok * p.group;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int warp_tok0 = (warp & 3) * 32 / p.group;  // token of the warp's first row
    const uint32_t stage = smem_addr(smem + C::OFF_OUT) + (warp & 3) * (C::NOUT * 2048);
    uint32_t no0 = 0, no1 = 0;  // items so far, of each row tile
    bool ok = true;
    PromptItem item;
    for (int32_t it = 0; ok && next_item(it, item); ++it) {
#pragma unroll 1
      for (int s = 0; s < 2; ++s) {
        if (tiles_of(item, s) == 0) continue;
        const uint32_t done = s ? no1 : no0;
        const int32_t tok = item.t0 + s * p.tq + row_tok;
        const uint32_t tm_o = tmem + lanes + C::TM_O + s * DV;
        const uint32_t slot = done & 1u;
        ok = ok && mbar_wait(&l_full[slot * 2 + s], (done >> 1) & 1u, abort_flag, to) &&
             mbar_wait(&o_full[s], slot, abort_flag, to);
        if (s) ++no1; else ++no0;
        if (!ok) break;
        tc_fence_after();
        const float inv =
            1.f / reinterpret_cast<float*>(smem + C::OFF_L)[slot * 256 + s * 128 + row];
        const int head = item.kvh * p.group + row_head;
        const bool live = row_tok < p.tq && tok < item.len;
        // A warp whose rows are whole tokens, all of them there, leaves the
        // store to TMA; else the rows go one by one.
        const int32_t tok0 = item.t0 + s * p.tq + warp_tok0;
        const bool bulk = 32 % p.group == 0 && tok0 + 32 / p.group <= item.len;
        // Offset of the row in the output, -1: no such row.
        const int64_t at = live ? static_cast<int64_t>(item.first + tok) * p.out_token +
                                      static_cast<int64_t>(head) * p.out_head
                                : -1;
        float2 odd = make_float2(0.f, 0.f);  // not zero if a value is not finite
        // TMEM first, so that the next item's products can begin.
        uint32_t w[DV / 2];
#pragma unroll
        for (int d = 0; d < DV / 32; ++d) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tm_o + d * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 f = mul2(make_float2(__uint_as_float(o[2 * i]),
                                              __uint_as_float(o[2 * i + 1])),
                                  make_float2(inv, inv));
            odd = fma2(f, make_float2(0.f, 0.f), odd);
            w[d * 16 + i] = float2_to_pair<T>(f.x, f.y);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[s]);
#pragma unroll
        for (int d0 = 0; d0 < DV / 32; d0 += C::NOUT) {
          if (lane == 0) bulk_wait_group_read<0>();  // the last stores have read the staging
          __syncwarp();
#pragma unroll
          for (int d = d0; d < d0 + C::NOUT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)  // rows of 64 bytes, 64-byte swizzle
              st_shared_v4(stage + (d - d0) * 2048 + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4),
                           w[d * 16 + i * 4], w[d * 16 + i * 4 + 1], w[d * 16 + i * 4 + 2],
                           w[d * 16 + i * 4 + 3]);
          if (bulk) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
#pragma unroll
              for (int d = d0; d < d0 + C::NOUT; ++d)
                tma_store_4d(&tmap_o, stage + (d - d0) * 2048, d * 32, 0, item.kvh,
                             item.first + tok0);
              bulk_commit_group();
            }
          } else {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // 8 rows, 64 contiguous bytes of each piece
              const int r = i * 8 + (lane >> 2), c = lane & 3;
              const int64_t to_row = __shfl_sync(0xffffffffu, at, r);
              if (to_row >= 0)
#pragma unroll
                for (int d = d0; d < d0 + C::NOUT; ++d)
                  *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + to_row + d * 32 + c * 8) =
                      ld_shared_v4(stage + (d - d0) * 2048 + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
            }
            __syncwarp();
          }
        }
        // A sum that is not finite is that of the row's own scores: NaN it stays.
        const uint32_t again =
            __ballot_sync(0xffffffffu, live && !(odd.x + odd.y == 0.f) && isfinite(inv));
        if (again) {  // these rows are written once more, after the stores above
          if (lane == 0) bulk_wait_group_all();
          __syncwarp();
          // Keys that the rows' MMAs covered, up to a whole step past their tile.
          const int32_t covered = min(item.len, (end_of(item, s) + 15) / 16 * 16);
          redo_rows<T, DQK, DV>(p, again, item.first, tok0, tok, item.kvh, head, covered,
                                abort_flag);
        }
      }
    }
    if (lane == 0) bulk_wait_group_read<0>();  // the staging is read before the CTA ends
  } else {
    reg_inc<184>();
    // ---- softmax: one row a thread
    const int s = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int row_tok = row / p.group;
    // Tokens of the warp's first and last row.
    const int warp_tok0 = (warp & 3) * 32 / p.group, warp_tok1 = ((warp & 3) * 32 + 31) / p.group;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tm_s = tmem + lanes + C::TM_S + s * 128;
    const uint32_t tm_o = tmem + lanes + C::TM_O + s * DV;
    uint32_t ns = 0, no = 0;  // tiles and items so far
    bool ok = true;
    PromptItem item;
    for (int32_t it = 0; ok && next_item(it, item); ++it) {
      const int32_t nt = tiles_of(item, s);
      if (nt == 0) continue;
      const int32_t t0 = item.t0 + s * p.tq;
      const int32_t tok = t0 + row_tok;  // position in the sequence
      float m_used = 0.f, l = 0.f;
      for (int32_t j = 0; j < nt; ++j) {
        ok = mbar_wait(&s_full[s], ns++ & 1u, abort_flag, to);
        if (!ok) break;
        tc_fence_after();
        float x[kKeys];
        tmem_ld_row(tm_s, x);
        tmem_ld_wait();
        float2 sum = make_float2(0.f, 0.f);
        // exp2 of 32 scores, their P and their sum.
        auto piece = [&](const float* v, uint32_t (&w)[16]) {
          const float2 scale2 = make_float2(p.qscale, p.qscale);
          // fp16: P is kept 2^7 higher (it stays below 2^15), so that fewer small
          // ones fall below the type's normal range; the sums carry the same factor.
          constexpr float kUp = Elem16<T>::kUmmaFormat == 0u ? 15.f - kLag : 0.f;
          const float shift = fmaf(-m_used, p.qscale, kUp);
          const float2 shift2 = make_float2(shift, shift);
          float2 part[2];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 y = fma2(make_float2(v[2 * i], v[2 * i + 1]), scale2, shift2);
            y.x = prompt_exp2(y.x);
            y.y = prompt_exp2(y.y);
            w[i] = float2_to_pair<T>(y.x, y.y);
            part[i & 1] = i < 2 ? y : add2(part[i & 1], y);
          }
          sum = add2(sum, add2(part[0], part[1]));
        };
        auto store = [&](int h, const uint32_t (&w)[16]) {
          tmem_st_32x32b_x16(tm_s + h * 16, w);
          if (h == C::MOST / 32 - 1 || h == kKeys / 32 - 1) {
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(h == kKeys / 32 - 1 ? &p_ready[s] : &p_most[s]);
          }
        };
        // A new maximum for the rows that need one: what was summed so far is
        // brought to it.  The others keep theirs (their factor is one): a row's
        // bits must not depend on what lies in the rows beside it.
        auto move_max = [&](float m_new) {
          // PV(j - 1) is complete (see the order of issue) and PV(j) waits for
          // this P, so O is this warp's to change.
          const float c = m_new == m_used ? 1.f : prompt_exp2((m_used - m_new) * p.qscale);
          m_used = m_new;
          l *= c;
#pragma unroll
          for (int b = 0; b < DV; b += 16) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(tm_o + b, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * c);
            tmem_st_32x32b_x16(tm_o + b, o);
          }
        };
        const int32_t least = t0 + warp_tok0 + 1 - j * kKeys;  // keys that every row sees
        const int32_t most = t0 + warp_tok1 + 1 - j * kKeys;   // and that any row does
        if (least < kKeys) {
          const int32_t seen = tok + 1 - j * kKeys;  // keys of this tile that the row sees
#pragma unroll
          for (int h = 0; h < kKeys / 32; ++h)
            if (least < h * 32 + 32) {
#pragma unroll
              for (int i = h * 32; i < h * 32 + 32; ++i)
                if (i >= seen) x[i] = -INFINITY;
            }
        }
        auto max_of = [&](int h, float m) {
          float m2 = fmaxf(x[h * 32], x[h * 32 + 1]);
#pragma unroll
          for (int i = h * 32 + 2; i < h * 32 + 30; i += 4) {
            m = max3(m, x[i], x[i + 1]);
            m2 = max3(m2, x[i + 2], x[i + 3]);
          }
          return max3(m, m2, fmaxf(x[h * 32 + 30], x[h * 32 + 31]));
        };
        // The first piece goes ahead with the maximum so far (an item's first
        // tile: with the piece's own), while the tile's is found; rarely, it has
        // to be done again.
        float m_tile = max_of(0, kFloor);
        if (j == 0) m_used = m_tile;
        uint32_t w[16];
        float less = 0.f;  // what was taken from the scores beforehand
#pragma unroll 1
        for (;;) {
          piece(x, w);
#pragma unroll
          for (int h = 1; h < kKeys / 32; ++h) m_tile = max_of(h, m_tile);
          // -m * scale is rounded, which moves a row's exponents.  Beyond kFar that
          // would tell in the weights, and from 2^24 on be a power of two or more:
          // there the difference is taken first, once the maximum is known.
          // A row is in order after one time through the rest: its maximum is then at
          // most kLag behind, and near zero.
          const auto is_far = [](float m) { return fabsf(m) * (kLag / kFar); };
          const float rise = m_tile - m_used;
          if (!__any_sync(0xffffffffu, fmaxf(rise, is_far(m_used)) * p.qscale > kLag)) break;
          const bool grow = rise * p.qscale > kLag;
          const float m_new = grow ? m_tile : m_used;
          if (j > 0 && __any_sync(0xffffffffu, grow))
            move_max(m_new);
          else
            m_used = m_new;
          if (is_far(m_used) * p.qscale > kLag) {
            less = m_used;
            m_tile -= less;
            m_used = 0.f;
#pragma unroll
            for (int i = 0; i < kKeys; ++i) x[i] -= less;
          }
          sum = make_float2(0.f, 0.f);
        }
        store(0, w);
#pragma unroll
        for (int h = 1; h < kKeys / 32; ++h) {
          // Only the last piece is skipped where no row of the warp sees its keys:
          // branches between the others keep them from overlapping (3% at 8192
          // tokens).
          if (h < kKeys / 32 - 1 || h * 32 < most) {
            piece(x + h * 32, w);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = 0u;
          }
          store(h, w);
        }
        l += sum.x + sum.y;
        m_used += less;
      }
      // The sums go to the output warps, by two slots (and barriers) in turn: the
      // first product of the next item waits for the output of this one, so the
      // item after next cannot be here before.
      if (!ok) break;
      reinterpret_cast<float*>(smem + C::OFF_L)[(no & 1u) * 256 + s * 128 + row] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_full[(no & 1u) * 2 + s]);
      ++no;
    }
  }
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TM_COLS);
  }
}

// ------------------------------------------------------------------ host side

template <typename T, int DQK, int DV>
static int launch_prompt(const PromptProblem& g, cudaStream_t stream) {
  using C = PromptCfg<DQK, DV>;
  auto kern = prompt_attention_kernel<T, DQK, DV>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_error("cudaGetDevice");
  static bool ready[kMaxDevices] = {};
  if (dev >= kMaxDevices || !ready[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    if (e != cudaSuccess) return set_cuda_error("cudaFuncSetAttribute(prompt attention)", e);
    if (dev < kMaxDevices) ready[dev] = true;
  }
  const int64_t G = g.Hq / g.Hkv, tq = kRows / G;
  const CUtensorMapDataType dt = Elem16<T>::kTmaType;
  CUtensorMap tq_map, tk, tv, to;
  {  // (d, head of the group, KV head, token)
    const uint64_t dims[4] = {static_cast<uint64_t>(DQK), static_cast<uint64_t>(G),
                              static_cast<uint64_t>(g.Hkv), static_cast<uint64_t>(g.tokens)};
    const uint64_t strides[3] = {static_cast<uint64_t>(g.q_head_stride) * 2,
                                 static_cast<uint64_t>(G * g.q_head_stride) * 2,
                                 static_cast<uint64_t>(g.q_token_stride) * 2};
    const uint32_t box[4] = {64, static_cast<uint32_t>(G), 1, static_cast<uint32_t>(tq)};
    const int rc = encode_tmap_4d(&tq_map, dt, g.q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  {  // the same view of the output; used where a warp's 32 rows are whole tokens
    const uint64_t dims[4] = {static_cast<uint64_t>(DV), static_cast<uint64_t>(G),
                              static_cast<uint64_t>(g.Hkv), static_cast<uint64_t>(g.tokens)};
    const uint64_t strides[3] = {static_cast<uint64_t>(g.out_head_stride) * 2,
                                 static_cast<uint64_t>(G * g.out_head_stride) * 2,
                                 static_cast<uint64_t>(g.out_token_stride) * 2};
    const uint32_t box[4] = {32, static_cast<uint32_t>(32 % G == 0 ? G : 1), 1,
                             static_cast<uint32_t>(32 % G == 0 ? 32 / G : 1)};
    const int rc = encode_tmap_4d(&to, dt, g.out, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc) return rc;
  }
  const uint32_t box[3] = {64, 1, C::KEYS};
  {
    const uint64_t dims[3] = {static_cast<uint64_t>(DQK), static_cast<uint64_t>(g.Hkv),
                              static_cast<uint64_t>(g.tokens)};
    const uint64_t strides[2] = {static_cast<uint64_t>(g.k_head_stride) * 2,
                                 static_cast<uint64_t>(g.k_token_stride) * 2};
    const int rc = encode_tmap_3d(&tk, dt, g.k, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  {
    const uint64_t dims[3] = {static_cast<uint64_t>(DV), static_cast<uint64_t>(g.Hkv),
                              static_cast<uint64_t>(g.tokens)};
    const uint64_t strides[2] = {static_cast<uint64_t>(g.v_head_stride) * 2,
                                 static_cast<uint64_t>(g.v_token_stride) * 2};
    const int rc = encode_tmap_3d(&tv, dt, g.v, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  PromptParams p;
  p.q = g.q;
  p.k = g.k;
  p.v = g.v;
  p.q_token = g.q_token_stride;
  p.q_head = g.q_head_stride;
  p.k_token = g.k_token_stride;
  p.k_head = g.k_head_stride;
  p.v_token = g.v_token_stride;
  p.v_head = g.v_head_stride;
  p.out = g.out;
  p.out_token = g.out_token_stride;
  p.out_head = g.out_head_stride;
  p.cu = g.cu_seqlens;
  p.batch = static_cast<int32_t>(g.batch);
  p.tokens = static_cast<int32_t>(g.tokens);
  p.max_seqlen = static_cast<int32_t>(g.max_seqlen);
  p.group = static_cast<int32_t>(G);
  p.hkv = static_cast<int32_t>(g.Hkv);
  p.tq = static_cast<int32_t>(tq);
  // All blocks of some KV heads come before those of the next, so that the keys
  // and values that the blocks share stay in L2 (a third of it).
  const int64_t head_bytes = g.tokens * (DQK + DV) * 2;
  int64_t at_once = (int64_t(40) << 20) / head_bytes;
  if (at_once < 1) at_once = 1;
  const int64_t groups = (g.Hkv + at_once - 1) / at_once;
  p.heads_at_once = static_cast<int32_t>((g.Hkv + groups - 1) / groups);
  p.negate = g.scale < 0.f ? 1u : 0u;
  // A scale of zero (every key the same weight) still has to send the masked
  // scores, -inf, to -inf: any factor far below the scores' rounding will do.
  p.qscale = fabsf(g.scale) * 1.4426950408889634f;
  if (p.qscale < 1e-30f) p.qscale = 1e-30f;  // a NaN stays
  // The output warps may redo 64 rows (redo_rows) between two reads of TMEM, for
  // which the others wait: 20 ns a row and key with heads of 128, 90 with 64 heads of
  // 192 / 128 out of DRAM.  1000 are allowed beyond the usual limit.
  p.timeout_ns = wait_timeout_ns() + static_cast<uint64_t>(p.max_seqlen) * 64 * 1000;
  // No more items than the whole blocks of all tokens and one ragged one a
  // sequence, nor than every sequence at its longest.
  const int64_t per = 2 * tq;
  int64_t items = g.tokens / per + g.batch;
  const int64_t longest = g.batch * ((g.max_seqlen + per - 1) / per);
  if (longest < items) items = longest;
  cudaLaunchConfig_t cfg = {};
  if (items * g.Hkv > 0x7fffffffLL)
    return set_error(FRN_ERR_UNSUPPORTED, "prompt attention: too many work items");
  cfg.gridDim = dim3(static_cast<unsigned>(items * g.Hkv));
  cfg.blockDim = dim3(kPromptThreads);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tq_map, tk, tv, to, p);
  if (e != cudaSuccess) return set_cuda_error("launch prompt_attention", e);
  return 0;
}

template <typename T>
static int launch_prompt_d(const PromptProblem& g, cudaStream_t s) {
  if (g.Dqk == 192) return launch_prompt<T, 192, 128>(g, s);
  if (g.Dqk == 128) return launch_prompt<T, 128, 128>(g, s);
  return launch_prompt<T, 64, 64>(g, s);
}

cudaError_t prompt_device_error(uint32_t* flags, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(flags, g_frn_device_error, sizeof(uint32_t));
  const uint32_t zero = 0;
  if (e == cudaSuccess && clear && *flags)
    e = cudaMemcpyToSymbol(g_frn_device_error, &zero, sizeof(uint32_t));
  return e;
}

int run_prompt_attention(const PromptProblem& g, cudaStream_t s) {
  return g.dtype == FRN_DTYPE_BF16 ? launch_prompt_d<__nv_bfloat16>(g, s)
                                   : launch_prompt_d<__half>(g, s);
}

}  // namespace frn
