// frn_paged_decode.cu -- single-token (decode) grouped-query attention over a
// paged key-value cache.
//
//   out[b, h, :] = sum_t p[t] V[b, t, h / G, :],
//   p = softmax over t < seq_lens[b] of scale * q[b, h, :] . K[b, t, h / G, :]
//
// where token t of sequence b lives in slot t % page_size of page
// page_table[b, t / page_size].  The K/V stream is the cost: 2 * sum(len) *
// Hkv * D elements, each read once for all G query heads of its KV head.
//
// Split.  The lengths live on the device and differ, so the work is cut there:
// the 64-token tiles of all (sequence, KV head) items, laid end to end, are
// dealt to the CTAs in equal contiguous shares, whatever the lengths.  A CTA
// walks its share item by item; an item that lies within one share is written
// directly, of the others every share leaves (max, sum, acc) in the workspace
// (at most two parts a CTA: an item can be cut at its share's start and at
// its end), and a second, dependent launch joins the parts in share order.  No
// atomics: the result does not depend on the order in which CTAs finish.
//
// Streams.  The four warps of a CTA take 16 tokens of every tile each and
// share nothing until an item ends: a warp copies its own tokens with 16-byte
// cp.async into its own ring, several tiles ahead and across item borders, so
// no block barrier and no page boundary interrupts the stream.  Tokens past
// the length are never read (their slots are zero-filled and their scores are
// -inf), so whatever lies in unused slots or pages has no effect.
//
// Arithmetic.  bf16 / fp16: the query heads of a group are the rows of 16x8x16
// MMAs (S = Q K^T, O += P V; up to 16 heads), online softmax in base 2 on the
// fragments, statistics and accumulators in fp32; P is rounded to the input
// type for the second product, its row sums are not.  fp32: CUDA cores, one
// token a lane for the scores, head dims across lanes for the output.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

#include "frn_internal.h"
#include "frn_ptx.cuh"

namespace frn {

constexpr int kPagedWarps = 4;
constexpr int kPagedThreads = 32 * kPagedWarps;
constexpr int kWarpTokens = 16;                         // a warp's tokens of a tile
constexpr int kTileTokens = kPagedWarps * kWarpTokens;  // 64

struct PagedDecodeParams {
  PagedView kv;
  const void* q;
  int64_t q_batch, q_head;      // element strides
  void* out;
  int64_t out_batch, out_head;  // element strides
  const int32_t* seq_lens;
  float* ws;       // [2 * CTAs][G][D] accumulators, then [2 * CTAs][G][2] (max, sum)
  int32_t* joins;  // [batch * Hkv][2] first part's slot (-1: nothing to join), last CTA
  int32_t batch, hkv, group, ctas;
  float qscale;    // scale * log2(e): the softmax runs in base 2
};

template <typename T, int D, int GMAX>
struct PagedCfg {
  static constexpr int ROW_BYTES = D * static_cast<int>(sizeof(T));
  static constexpr int HALF_BYTES = kWarpTokens * ROW_BYTES;  // a warp's K (or V) of a tile
  static constexpr int STAGE_BYTES = 2 * HALF_BYTES;
  // 24 KB of ring a warp, two CTAs an SM; the 512-byte rows of fp32 at D = 128
  // take 48 KB and an SM each.
  static constexpr int CTAS_PER_SM = HALF_BYTES > 4096 ? 1 : 2;
  static constexpr int STAGES = (CTAS_PER_SM == 1 ? 49152 : 24576) / STAGE_BYTES;
  static constexpr int RING_BYTES = kPagedWarps * STAGES * STAGE_BYTES;
  // Join of the four warps: 8 heads at a time, [warp][8][D] acc, [warp][8] max and sum.
  static constexpr int JOIN_FLOATS = kPagedWarps * 8 * (D + 2);
  static constexpr int Q_FLOATS = sizeof(T) == 4 ? GMAX * D : 0;  // fp32: the queries
  static constexpr int SMEM_BYTES = RING_BYTES + (JOIN_FLOATS + Q_FLOATS) * 4;
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (Elem16<T>::kUmmaFormat == 1u)
      asm volatile(
          "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
          "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
      asm volatile(
          "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
          "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

template <bool TRANS>
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// A place in the sequence of tiles: tile `tile` of the item (b, head).
struct TileAt {
  int32_t b, head, tile, tiles, len;
};

// Length of sequence b as the kernel uses it: not negative, and within the
// sequence's row of the page table.
__device__ __forceinline__ int32_t length_of(const PagedDecodeParams& p, int b) {
  const int64_t most = p.kv.max_pages * static_cast<int64_t>(p.kv.page_size);  // at most 2^31 - 1, checked by the host
  const int32_t n = p.seq_lens[b];
  if (n < 0 || n > most) {
    atomicOr(&g_frn_device_error, kDevErrBadPage);
    return n < 0 ? 0 : static_cast<int32_t>(most);
  }
  return n;
}

__device__ __forceinline__ int32_t tiles_of(int32_t len) {
  return static_cast<int32_t>((static_cast<int64_t>(len) + kTileTokens - 1) / kTileTokens);
}

__device__ __forceinline__ void advance(const PagedDecodeParams& p, TileAt& at) {
  if (++at.tile < at.tiles) return;
  at.tile = 0;
  if (++at.head < p.hkv) return;
  at.head = 0;
  do {
    if (++at.b >= p.batch) return;  // past the last tile: not used any more
    at.len = length_of(p, at.b);
    at.tiles = tiles_of(at.len);
  } while (at.tiles == 0);
}

// Byte offset of 16-byte piece c of row r; rows are ROW_BYTES long.  The
// permutation puts the eight rows of an ldmatrix (or of a quarter-warp's
// 16-byte loads) on distinct banks.
template <int ROW_BYTES>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  return static_cast<uint32_t>(r * ROW_BYTES + ((c ^ (r & 7)) << 4));
}

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Tiles before sequence b, times Hkv, for every b at once: thread i sums its
// run of sequences, a block scan does the rest.  Returns the total; *mine is
// the sum of the runs before this thread's.
__device__ __forceinline__ int64_t scan_tiles(const PagedDecodeParams& p, int64_t* sm_warp,
                                              int64_t* mine, int64_t* own) {
  const int per = (p.batch + kPagedThreads - 1) / kPagedThreads;
  const int b0 = static_cast<int>(threadIdx.x) * per;
  int64_t sum = 0;
  for (int b = b0; b < min(p.batch, b0 + per); ++b) sum += tiles_of(length_of(p, b));
  sum *= p.hkv;
  const int lane = static_cast<int>(threadIdx.x & 31), warp = static_cast<int>(threadIdx.x >> 5);
  int64_t inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) sm_warp[warp] = inc;
  __syncthreads();
  int64_t before = inc - sum, total = 0;
#pragma unroll
  for (int w = 0; w < kPagedWarps; ++w) {
    if (w < warp) before += sm_warp[w];
    total += sm_warp[w];
  }
  *mine = before;
  *own = sum;
  return total;
}

template <typename T, int D, int GMAX>
__global__ void __launch_bounds__(kPagedThreads, 2)
    paged_decode_kernel(const PagedDecodeParams p) {
  using C = PagedCfg<T, D, GMAX>;
  constexpr bool MMA = sizeof(T) == 2;
  constexpr int NR = MMA ? (GMAX + 7) / 8 : 1;  // 8-row halves of the MMA in use
  constexpr int NKC = D / 16, NDT = D / 8;
  constexpr int E = D / 32;                     // fp32: output dims of a lane
  constexpr int CHUNKS = C::ROW_BYTES / 16;     // 16-byte pieces of a row
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t sm_warp[kPagedWarps];
  __shared__ TileAt sm_first;

  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  const int G = p.group;
  griddep_launch_dependents();
  griddep_wait();

  // ---- this CTA's share [u0, u1) of the tiles, and where it starts
  int64_t before, own;
  const int64_t total = scan_tiles(p, sm_warp, &before, &own);
  const int64_t share = (total + p.ctas - 1) / p.ctas;
  const int64_t u0 = share * blockIdx.x, u1 = min(total, u0 + share);
  if (u0 >= u1) return;
  if (before <= u0 && u0 < before + own) {  // one thread's run holds tile u0
    const int per = (p.batch + kPagedThreads - 1) / kPagedThreads;
    int b = static_cast<int>(threadIdx.x) * per;
    int64_t at = before;
    TileAt f;
    for (;; ++b) {
      f.len = length_of(p, b);
      f.tiles = tiles_of(f.len);
      const int64_t n = static_cast<int64_t>(f.tiles) * p.hkv;
      if (u0 < at + n) break;
      at += n;
    }
    f.b = b;
    f.head = static_cast<int32_t>((u0 - at) / f.tiles);
    f.tile = static_cast<int32_t>((u0 - at) % f.tiles);
    sm_first = f;
  }
  __syncthreads();
  TileAt now = sm_first, ahead = now;
  const int64_t ntiles = u1 - u0;

  uint8_t* ring = smem + warp * (C::STAGES * C::STAGE_BYTES);
  const uint32_t ring_a = smem_addr(ring);
  float* sm_acc = reinterpret_cast<float*>(smem + C::RING_BYTES);  // [4][8][D]
  float* sm_m = sm_acc + kPagedWarps * 8 * D;                      // [4][8]
  float* sm_l = sm_m + kPagedWarps * 8;                            // [4][8]
  float* sm_q = sm_acc + C::JOIN_FLOATS;                           // fp32: [G][D]

  // ---- loads: lane r < 16 looks up the page of the warp's token r one tile
  // before that tile's copies are issued.
  int32_t page = -1, slot = 0;
  auto look_up = [&]() {
    const int32_t t = ahead.tile * kTileTokens + warp * kWarpTokens + (lane & 15);
    page = -1;
    if (t < ahead.len) {
      const int32_t n = t / p.kv.page_size;
      slot = t - n * p.kv.page_size;
      page = p.kv.page_table[ahead.b * p.kv.table_stride + n];
      if (page < 0 || page >= p.kv.num_pages) {
        page = -1;  // reads as zeros
        atomicOr(&g_frn_device_error, kDevErrBadPage);
      }
    }
  };
  auto issue = [&](int stage) {
    const uint32_t kdst = ring_a + stage * C::STAGE_BYTES, vdst = kdst + C::HALF_BYTES;
    constexpr int ROWS = 32 / CHUNKS > 0 ? 32 / CHUNKS : 1;  // rows of one pass of the warp
    const T* kb = static_cast<const T*>(p.kv.k) + ahead.head * p.kv.k_head_stride;
    const T* vb = static_cast<const T*>(p.kv.v) + ahead.head * p.kv.v_head_stride;
    const int c = lane % CHUNKS;
#pragma unroll
    for (int i = 0; i < kWarpTokens / ROWS; ++i) {
      const int r = i * ROWS + lane / CHUNKS;
      const int32_t pg = __shfl_sync(0xffffffffu, page, r);
      const int64_t sl = __shfl_sync(0xffffffffu, slot, r);
      const uint32_t bytes = pg >= 0 ? 16u : 0u;
      const int64_t pp = pg >= 0 ? pg : 0;
      const T* ks = kb + pp * p.kv.k_page_stride + sl * p.kv.k_token_stride + c * (16 / sizeof(T));
      const T* vs = vb + pp * p.kv.v_page_stride + sl * p.kv.v_token_stride + c * (16 / sizeof(T));
      cp_async_16(kdst + swz<C::ROW_BYTES>(r, c), ks, bytes);
      cp_async_16(vdst + swz<C::ROW_BYTES>(r, c), vs, bytes);
    }
  };
  int64_t issued = 0;
  look_up();
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) {
    if (issued < ntiles) {
      issue(s);
      ++issued;
      if (issued < ntiles) {
        advance(p, ahead);
        look_up();
      }
    }
    cp_async_commit();
  }

  // ---- per item: queries, running statistics, accumulators
  const int g = lane >> 2, tq = lane & 3;
  uint32_t qa[MMA ? NKC : 1][4];
  float o[MMA ? NDT : 1][4];
  float m_run[MMA ? NR : GMAX], l_run[MMA ? NR : GMAX];
  float accf[MMA ? 1 : GMAX][E];
  const int mi = lane >> 3, mr = lane & 7;
  bool fresh = true;
  bool first_segment = true;
  int stage = 0;

  for (int64_t u = 0; u < ntiles; ++u) {
    // Keep the ring full: the slot freed by the previous tile takes a new one.
    if (issued < ntiles) {
      int s = stage + C::STAGES - 1;
      if (s >= C::STAGES) s -= C::STAGES;
      issue(s);
      ++issued;
      if (issued < ntiles) {
        advance(p, ahead);
        look_up();
      }
    }
    cp_async_commit();

    if (fresh) {
      fresh = false;
      const T* qp = static_cast<const T*>(p.q) + now.b * p.q_batch +
                    static_cast<int64_t>(now.head) * G * p.q_head;
      if constexpr (MMA) {
#pragma unroll
        for (int kc = 0; kc < NKC; ++kc)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = g + (e & 1) * 8, d = kc * 16 + (e >> 1) * 8 + 2 * tq;
            qa[kc][e] = (e & 1) < NR && row < G
                            ? *reinterpret_cast<const uint32_t*>(qp + row * p.q_head + d)
                            : 0u;
          }
#pragma unroll
        for (int j = 0; j < NDT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          m_run[r] = -FLT_MAX;
          l_run[r] = 0.f;
        }
      } else {
        __syncthreads();  // every warp is done with the last item's queries
        for (int i = static_cast<int>(threadIdx.x); i < G * D; i += kPagedThreads)
          sm_q[i] = static_cast<float>(qp[(i / D) * p.q_head + i % D]);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < GMAX; ++r) {
          m_run[r] = -FLT_MAX;
          l_run[r] = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) accf[r][e] = 0.f;
        }
      }
    }

    cp_async_wait<C::STAGES - 1>();
    __syncwarp();
    const uint32_t kb = ring_a + stage * C::STAGE_BYTES, vb = kb + C::HALF_BYTES;
    const int32_t t0 = now.tile * kTileTokens + warp * kWarpTokens;  // the warp's first token
    if constexpr (MMA) {
      // S = Q . K^T of this warp's 16 tokens: two 8-token tiles.
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int kc = 0; kc < NKC; ++kc) {
        uint32_t kf[4];  // matrices (tokens 0-7 | 8-15) x (low | high 8 of the 16 dims)
        ldsm4<false>(kb + swz<C::ROW_BYTES>(((mi >> 1) << 3) + mr, kc * 2 + (mi & 1)), kf);
        mma_16816<T>(sc[0], qa[kc], kf[0], kf[1]);
        mma_16816<T>(sc[1], qa[kc], kf[2], kf[3]);
      }
      uint32_t pa[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float x[4];  // columns: tokens 2tq, 2tq + 1 of each tile
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int32_t t = t0 + (e >> 1) * 8 + 2 * tq + (e & 1);
          x[e] = t < now.len ? sc[e >> 1][r * 2 + (e & 1)] * p.qscale : -INFINITY;
        }
        float bm = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
        const float m_new = fmaxf(m_run[r], bm);
        const float corr = exp2_approx(m_run[r] - m_new);
        m_run[r] = m_new;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = exp2_approx(x[e] - m_new);
        l_run[r] = l_run[r] * corr + (x[0] + x[1]) + (x[2] + x[3]);
#pragma unroll
        for (int j = 0; j < NDT; ++j) {
          o[j][r * 2] *= corr;
          o[j][r * 2 + 1] *= corr;
        }
        pa[r] = float2_to_pair<T>(x[0], x[1]);
        pa[2 + r] = float2_to_pair<T>(x[2], x[3]);
      }
      // O += P . V: V transposed by the load, 16 dims (two tiles) a step.
#pragma unroll
      for (int j = 0; j < NDT; j += 2) {
        uint32_t vf[4];
        ldsm4<true>(vb + swz<C::ROW_BYTES>(((mi & 1) << 3) + mr, j + (mi >> 1)), vf);
        mma_16816<T>(o[j], pa, vf[0], vf[1]);
        mma_16816<T>(o[j + 1], pa, vf[2], vf[3]);
      }
    } else {
      // Scores: lanes r and r + 16 hold token r, one half of the dims each.
      // Four chains a dot product keep its rounding error (which the exponential
      // turns into a relative one) at that of 8- or 16-term sums.
      const int tok = lane & 15, half = lane >> 4;
      const bool live = t0 + tok < now.len;
      float4 kf[CHUNKS / 2];
#pragma unroll
      for (int c = 0; c < CHUNKS / 2; ++c)
        kf[c] = ld_shared_v4f(kb + swz<C::ROW_BYTES>(tok, half * (CHUNKS / 2) + c));
      float s[GMAX];
#pragma unroll
      for (int r = 0; r < GMAX; ++r) {
        if (r >= G) continue;
        const float4* qf = reinterpret_cast<const float4*>(sm_q + r * D) + half * (CHUNKS / 2);
        float4 d = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < CHUNKS / 2; ++c) {
          d.x = fmaf(qf[c].x, kf[c].x, d.x);
          d.y = fmaf(qf[c].y, kf[c].y, d.y);
          d.z = fmaf(qf[c].z, kf[c].z, d.z);
          d.w = fmaf(qf[c].w, kf[c].w, d.w);
        }
        float x = (d.x + d.y) + (d.z + d.w);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        float bm = live ? x * p.qscale : -FLT_MAX;
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, w));
        const float m_new = fmaxf(m_run[r], bm);
        const float corr = exp2f(m_run[r] - m_new);
        m_run[r] = m_new;
        s[r] = live ? exp2f(fmaf(x, p.qscale, -m_new)) : 0.f;
        l_run[r] = l_run[r] * corr + (half == 0 ? s[r] : 0.f);  // one of the two copies counts
#pragma unroll
        for (int e = 0; e < E; ++e) accf[r][e] *= corr;
      }
#pragma unroll 4
      for (int t = 0; t < kWarpTokens; ++t) {
        float vf[E];
        const uint32_t a = vb + swz<C::ROW_BYTES>(t, (lane * E) / 4) + ((lane * E) % 4) * 4;
        if constexpr (E == 4) {
          const float4 v4 = ld_shared_v4f(a);
          vf[0] = v4.x; vf[1] = v4.y; vf[2] = v4.z; vf[3] = v4.w;
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) vf[e] = ld_shared_f32(a + e * 4);
        }
#pragma unroll
        for (int r = 0; r < GMAX; ++r) {
          if (r >= G) continue;
          const float pt = __shfl_sync(0xffffffffu, s[r], t);
#pragma unroll
          for (int e = 0; e < E; ++e) accf[r][e] = fmaf(pt, vf[e], accf[r][e]);
        }
      }
    }
    __syncwarp();  // the slot is refilled at the top of the next tile
    if (++stage == C::STAGES) stage = 0;

    // ---- the item, or this share's part of it, ends here
    if (now.tile + 1 == now.tiles || u + 1 == ntiles) {
      const int64_t item = static_cast<int64_t>(now.b) * p.hkv + now.head;
      // Tiles of the item before this share, and whether it goes on after it.
      const int64_t seg_tiles = min(static_cast<int64_t>(now.tile) + 1, u + 1);
      const bool starts = seg_tiles == now.tile + 1, ends = now.tile + 1 == now.tiles;
      const int part = 2 * static_cast<int>(blockIdx.x) + (first_segment ? 0 : 1);
      if (starts && threadIdx.x == 0) {
        p.joins[item * 2] = ends ? -1 : part;
        p.joins[item * 2 + 1] =
            static_cast<int32_t>((u0 + u - now.tile + now.tiles - 1) / share);
      }
#pragma unroll
      for (int h8 = 0; h8 < (GMAX + 7) / 8; ++h8) {  // 8 heads at a time
        const int heads = min(8, G - h8 * 8);
        if (heads <= 0) break;
        __syncthreads();  // the join buffers are free
        if constexpr (MMA) {
          float l = l_run[h8];
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          if (g < heads) {
#pragma unroll
            for (int j = 0; j < NDT; ++j)
              *reinterpret_cast<float2*>(sm_acc + (warp * 8 + g) * D + j * 8 + 2 * tq) =
                  make_float2(o[j][h8 * 2], o[j][h8 * 2 + 1]);
            if (tq == 0) {
              sm_m[warp * 8 + g] = m_run[h8];
              sm_l[warp * 8 + g] = l;
            }
          }
        } else {
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int row = h8 * 8 + r;
            if (r >= heads) continue;
            float l = l_run[row];
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
#pragma unroll
            for (int e = 0; e < E; ++e) sm_acc[(warp * 8 + r) * D + lane * E + e] = accf[row][e];
            if (lane == 0) {
              sm_m[warp * 8 + r] = m_run[row];
              sm_l[warp * 8 + r] = l;
            }
          }
        }
        __syncthreads();
        for (int i = static_cast<int>(threadIdx.x); i < heads * D; i += kPagedThreads) {
          const int r = i / D, d = i % D, row = h8 * 8 + r;
          float mx = -FLT_MAX;
#pragma unroll
          for (int w = 0; w < kPagedWarps; ++w) mx = fmaxf(mx, sm_m[w * 8 + r]);
          float num = 0.f, den = 0.f;
#pragma unroll
          for (int w = 0; w < kPagedWarps; ++w) {
            const float f = exp2f(sm_m[w * 8 + r] - mx);
            num = fmaf(sm_acc[(w * 8 + r) * D + d], f, num);
            den = fmaf(sm_l[w * 8 + r], f, den);
          }
          if (starts && ends) {
            T* op = static_cast<T*>(p.out) + now.b * p.out_batch +
                    (static_cast<int64_t>(now.head) * G + row) * p.out_head;
            op[d] = from_float<T>(num / den);
          } else {
            p.ws[(static_cast<int64_t>(part) * G + row) * D + d] = num;
            if (d == 0) {
              float* ml = p.ws + static_cast<int64_t>(2 * p.ctas) * G * D +
                          (static_cast<int64_t>(part) * G + row) * 2;
              ml[0] = mx;
              ml[1] = den;
            }
          }
        }
      }
      fresh = true;
      first_segment = false;
    }
    if (u + 1 < ntiles) advance(p, now);
  }
}

// Joins the parts of every item that was cut, in share order, and writes the
// zeros of empty sequences.  One CTA per (KV head, sequence), a thread per
// (head, dim).
template <typename T>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedDecodeParams p, int D) {
  griddep_launch_dependents();
  griddep_wait();
  const int head = blockIdx.x, b = blockIdx.y;
  const int64_t item = static_cast<int64_t>(b) * p.hkv + head;
  T* op = static_cast<T*>(p.out) + b * p.out_batch + static_cast<int64_t>(head) * p.group * p.out_head;
  if (p.seq_lens[b] <= 0) {
    for (int i = static_cast<int>(threadIdx.x); i < p.group * D; i += blockDim.x)
      op[(i / D) * p.out_head + i % D] = from_float<T>(0.f);
    return;
  }
  const int first = p.joins[item * 2];
  if (first < 0) return;
  const int last = p.joins[item * 2 + 1];  // CTA of the last part; its slot is the CTA's first
  const int c0 = first / 2, n = last - c0 + 1;
  const float* ml = p.ws + static_cast<int64_t>(2 * p.ctas) * p.group * D;
  for (int i = static_cast<int>(threadIdx.x); i < p.group * D; i += blockDim.x) {
    const int row = i / D, d = i % D;
    float mx = -FLT_MAX;
    for (int s = 0; s < n; ++s) {
      const int64_t part = s == 0 ? first : 2 * (c0 + s);
      mx = fmaxf(mx, ml[(part * p.group + row) * 2]);
    }
    float num = 0.f, den = 0.f;
    for (int s = 0; s < n; ++s) {
      const int64_t part = s == 0 ? first : 2 * (c0 + s);
      const float f = exp2f(ml[(part * p.group + row) * 2] - mx);
      num = fmaf(p.ws[(part * p.group + row) * D + d], f, num);
      den = fmaf(ml[(part * p.group + row) * 2 + 1], f, den);
    }
    op[row * p.out_head + d] = from_float<T>(num / den);
  }
}

// ------------------------------------------------------------------ host side

// Every CTA resident (PagedCfg::CTAS_PER_SM of them on an SM), and no more of
// them than there can be tiles.
static int paged_ctas(int dtype, int64_t batch, int64_t hkv, int64_t d, int64_t capacity, int sms) {
  const int64_t resident = (dtype == FRN_DTYPE_F32 && d == 128 ? 1 : 2) * static_cast<int64_t>(sms);
  const int64_t most = batch * hkv * ((capacity + kTileTokens - 1) / kTileTokens);
  return static_cast<int>(most < resident ? (most > 0 ? most : 1) : resident);
}

size_t paged_decode_workspace(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d,
                              int64_t capacity, int sms) {
  const int64_t c = paged_ctas(dtype, batch, hkv, d, capacity, sms);
  const int64_t floats = 2 * c * (hq / hkv) * (d + 2);
  return static_cast<size_t>((floats + 2 * batch * hkv) * 4);
}

template <typename T, int D, int GMAX>
static int launch_paged(const PagedDecodeProblem& g, PagedDecodeParams& p, cudaStream_t stream) {
  using C = PagedCfg<T, D, GMAX>;
  auto kern = paged_decode_kernel<T, D, GMAX>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_error("cudaGetDevice");
  static bool ready[kMaxDevices] = {};
  if (dev >= kMaxDevices || !ready[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    if (e != cudaSuccess) return set_cuda_error("cudaFuncSetAttribute(paged decode)", e);
    if (dev < kMaxDevices) ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.ctas));
  cfg.blockDim = dim3(kPagedThreads);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return set_cuda_error("launch paged_decode", e);
  cfg.gridDim = dim3(static_cast<unsigned>(g.kv.num_kv_heads), static_cast<unsigned>(g.batch));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, paged_join_kernel<T>, p, D);
  if (e != cudaSuccess) return set_cuda_error("launch paged_join", e);
  return 0;
}

template <typename T, int D>
static int launch_paged_g(const PagedDecodeProblem& g, PagedDecodeParams& p, cudaStream_t s) {
  return p.group <= 8 ? launch_paged<T, D, 8>(g, p, s) : launch_paged<T, D, 16>(g, p, s);
}

template <typename T>
static int launch_paged_d(const PagedDecodeProblem& g, PagedDecodeParams& p, cudaStream_t s) {
  return g.kv.head_dim == 128 ? launch_paged_g<T, 128>(g, p, s) : launch_paged_g<T, 64>(g, p, s);
}

int run_paged_decode(const PagedDecodeProblem& g, cudaStream_t stream) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_error("cudaGetDevice");
  PagedDecodeParams p;
  p.kv = g.kv;
  p.q = g.q;
  p.q_batch = g.q_batch_stride;
  p.q_head = g.q_head_stride;
  p.out = g.out;
  p.out_batch = g.out_batch_stride;
  p.out_head = g.out_head_stride;
  p.seq_lens = g.seq_lens;
  p.batch = static_cast<int32_t>(g.batch);
  p.hkv = static_cast<int32_t>(g.kv.num_kv_heads);
  p.group = static_cast<int32_t>(g.num_q_heads / g.kv.num_kv_heads);
  p.ctas = paged_ctas(g.dtype, g.batch, g.kv.num_kv_heads, g.kv.head_dim,
                      g.kv.max_pages * g.kv.page_size, sm_count(dev));
  p.ws = static_cast<float*>(g.workspace);
  p.joins = reinterpret_cast<int32_t*>(
      p.ws + static_cast<int64_t>(2 * p.ctas) * p.group * (g.kv.head_dim + 2));
  p.qscale = g.scale * 1.4426950408889634f;  // log2(e): the softmax runs in base 2
  switch (g.dtype) {
    case FRN_DTYPE_BF16: return launch_paged_d<__nv_bfloat16>(g, p, stream);
    case FRN_DTYPE_F16: return launch_paged_d<__half>(g, p, stream);
    default: return launch_paged_d<float>(g, p, stream);
  }
}

}  // namespace frn
