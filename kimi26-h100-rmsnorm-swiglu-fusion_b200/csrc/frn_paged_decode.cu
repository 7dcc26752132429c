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
// the 16-token tiles of all (sequence, KV head) items, laid end to end, are
// dealt to the warps in equal contiguous shares, whatever the lengths (an item
// counts as at least `least` tiles, which pays for its queries and its end, and
// keeps tiny items from sharing a warp while others idle).  A warp
// walks its share item by item; an item that lies within one share is written
// directly, of the others every share leaves (max, sum, acc) in the workspace
// (at most two parts a warp: an item can be cut at its share's start and at
// its end), and a second, dependent launch joins the parts in share order.  No
// atomics: the result does not depend on the order in which warps finish.
// Shares are a warp's, not a CTA's: with four warps on every tile the warps had to
// be joined at each item's end, and a batch of 64 sequences of 1 to 8192 tokens took
// 96.8 us instead of 91.7, one of 1000 16.1 instead of 14.1 (both without the later
// steps).
//
// Streams.  A warp copies its tiles with 16-byte cp.async into its own ring,
// several tiles ahead and across item borders: no block barrier and no page
// boundary interrupts the stream.  Tokens past the length are never read
// (their slots are zero-filled and their scores are -inf), so whatever lies in
// unused slots or pages has no effect.
//
// What bounds it: HBM.  8 sequences of 100 to 131 thousand tokens (3.8 GB) take
// 596 to 635 us, 6.0 to 6.4 TB/s or 92 to 98% of a plain copy's rate; 64 sequences
// of 1 to 8192 tokens (352 MB) 67 to 71 us, about 10 of them the start of the
// streams and the join; one sequence of 1000 tokens 8.5 us, of which a one-token
// call's chain of dependent loads and two launches is 5.7.  Two CTAs an SM with
// three tiles in flight a warp: one CTA with seven is 6 to 20% slower, three with
// two up to 12%.
//
// Arithmetic.  bf16 / fp16: the query heads of a group are the rows of 16x8x16
// MMAs (S = Q K^T, O += P V; up to 16 heads), online softmax in base 2 on the
// fragments, statistics and accumulators in fp32; P is rounded to the input
// type for the second product, its row sums are not (a second product with what
// the rounding leaves would take the error from 1.4 times the output's own
// rounding to that, and costs 2 to 4% of the time).  fp32: CUDA cores, one
// token a lane for the scores, head dims across lanes for the output.  Four heads'
// scores are taken together, so that their shuffles and exponentials overlap: 8
// sequences of 8192 tokens, 32 / 8 heads of 128, took 132 us instead of 158, and
// another twentieth less with eight tokens of the second product unrolled instead of
// four.  They take 132 us (4.1 TB/s) with the scores' differences taken before they
// are scaled, 130.5 on the same card without; with rings of 16 KB tiles an SM holds
// four warps, which leave the latencies of shared memory uncovered.  Eight heads
// together were 15% slower there and 2% faster with eight heads of 64.
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
constexpr int kTileTokens = 16;

// CTAs of an SM: as many as leave every warp a ring of at least 14 KB, fp32 with
// head dim 128 (16 KB a tile) 48 KB.
constexpr int paged_ctas_per_sm(bool fp32, int d) {
  return fp32 ? (d == 128 ? 1 : 2) : (d == 128 ? 2 : 4);
}

struct PagedDecodeParams {
  PagedView kv;
  const void* q;
  int64_t q_batch, q_head;      // element strides
  void* out;
  int64_t out_batch, out_head;  // element strides
  const int32_t* seq_lens;
  float* ws;       // [2 * warps][G][D] accumulators, then [2 * warps][G][2] (max, sum)
  int32_t* joins;  // [batch * Hkv][2] first part (-1: nothing to join), last warp
  int32_t batch, hkv, group, warps;
  int32_t least, least_share;  // tiles that an item counts as, and that a share has, at least
  int32_t join_rows;  // query heads of a CTA of the join: 1 or 4
  // scale * log2(e): the softmax runs in base 2.  16-bit: maxima (the parts' too) are
  // those of the scaled scores, unit is 1.  fp32: of the unscaled ones, of a negated
  // query where the scale is negative; qscale and unit are |scale| * log2(e).
  float qscale, unit;
  float qsign;
};

template <typename T, int D, int GMAX>
struct PagedCfg {
  static constexpr int ROW_BYTES = D * static_cast<int>(sizeof(T));
  static constexpr int HALF_BYTES = kTileTokens * ROW_BYTES;  // K (or V) of a tile
  static constexpr int STAGE_BYTES = 2 * HALF_BYTES;
  static constexpr int CTAS_PER_SM = paged_ctas_per_sm(sizeof(T) == 4, D);
  static constexpr int Q_BYTES = sizeof(T) == 4 ? GMAX * D * 4 : 0;  // fp32: the item's queries
  static constexpr int STAGES = (224 * 1024 / CTAS_PER_SM / kPagedWarps - Q_BYTES) / STAGE_BYTES;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int WARP_BYTES = RING_BYTES + Q_BYTES;
  static constexpr int SMEM_BYTES = kPagedWarps * WARP_BYTES;
  static_assert(STAGES >= 2, "one tile in flight while one is used");
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

// Two fp32 multiply-adds an instruction.
__device__ __forceinline__ float2 fma_f32x2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// A place in the sequence of tiles: tile `tile` of the item (b, head), at
// position u of all.
struct TileAt {
  int32_t b, head, tile, tiles, len;
  int64_t u;
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

// Positions that an item of a sequence takes up.
__device__ __forceinline__ int32_t places_of(const PagedDecodeParams& p, int32_t tiles) {
  return tiles > 0 ? max(tiles, p.least) : 0;
}

// The next tile; past the last one u is the total.
__device__ __forceinline__ void advance(const PagedDecodeParams& p, TileAt& at) {
  ++at.u;
  if (++at.tile < at.tiles) return;
  at.u += places_of(p, at.tiles) - at.tiles;
  at.tile = 0;
  if (++at.head < p.hkv) return;
  at.head = 0;
  do {
    if (++at.b >= p.batch) return;
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

// Positions before sequence b, for every b at once: thread i sums its
// run of sequences, a block scan does the rest.  Returns the total; *mine is
// the sum of the runs before this thread's.
__device__ __forceinline__ int64_t scan_tiles(const PagedDecodeParams& p, int64_t* sm_warp,
                                              int64_t* mine, int64_t* own) {
  const int per = (p.batch + kPagedThreads - 1) / kPagedThreads;
  const int b0 = static_cast<int>(threadIdx.x) * per;
  int64_t sum = 0;
  for (int b = b0; b < min(p.batch, b0 + per); ++b) sum += places_of(p, tiles_of(length_of(p, b)));
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

// UNI: pages hold whole tiles, so a tile's rows are `token_stride` apart.
template <typename T, int D, int GMAX, bool UNI>
__global__ void __launch_bounds__(kPagedThreads, paged_ctas_per_sm(sizeof(T) == 4, D))
    paged_decode_kernel(const PagedDecodeParams p) {
  using C = PagedCfg<T, D, GMAX>;
  constexpr bool MMA = sizeof(T) == 2;
  constexpr int NR = MMA ? (GMAX + 7) / 8 : 1;  // 8-row halves of the MMA in use
  constexpr int NKC = D / 16, NDT = D / 8;
  constexpr int E = D / 32;                     // fp32: output dims of a lane
  constexpr int HB = GMAX > 4 ? 4 : 1;          // fp32: heads whose scores are taken together
  constexpr int CHUNKS = C::ROW_BYTES / 16;     // 16-byte pieces of a row
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t sm_warp[kPagedWarps];
  __shared__ TileAt sm_first[kPagedWarps];

  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  const int G = p.group;
  griddep_launch_dependents();
  griddep_wait();

  // ---- the warps' shares of the tiles, and where they start
  int64_t before, own;
  const int64_t total = scan_tiles(p, sm_warp, &before, &own);
  const int64_t share = max((total + p.warps - 1) / p.warps, static_cast<int64_t>(p.least_share));
  const int me = static_cast<int>(blockIdx.x) * kPagedWarps + warp;  // this warp's number
  if (own > 0) {
    // The shares of this CTA that start within this thread's run of sequences.
    const int per = (p.batch + kPagedThreads - 1) / kPagedThreads;
    for (int w = 0; w < kPagedWarps; ++w) {
      const int64_t u = share * (static_cast<int64_t>(blockIdx.x) * kPagedWarps + w);
      if (u < before || u >= before + own) continue;
      int b = static_cast<int>(threadIdx.x) * per;
      int64_t at = before;
      TileAt f;
      for (;; ++b) {
        f.len = length_of(p, b);
        f.tiles = tiles_of(f.len);
        const int64_t n = static_cast<int64_t>(places_of(p, f.tiles)) * p.hkv;
        if (u < at + n) break;
        at += n;
      }
      const int32_t places = places_of(p, f.tiles);
      f.b = b;
      f.head = static_cast<int32_t>((u - at) / places);
      f.tile = static_cast<int32_t>((u - at) % places);
      f.u = u;
      if (f.tile >= f.tiles) {  // past the item's tiles: the next item
        f.u -= f.tile - (f.tiles - 1);
        f.tile = f.tiles - 1;
        advance(p, f);
      }
      sm_first[w] = f;
    }
  }
  __syncthreads();
  const int64_t u0 = share * me, u1 = min(total, u0 + share);
  if (u0 >= u1) return;
  TileAt now = sm_first[warp], ahead = now;
  if (now.u >= u1) return;

  uint8_t* ring = smem + warp * C::WARP_BYTES;
  const uint32_t ring_a = smem_addr(ring);
  float* sm_q = reinterpret_cast<float*>(ring + C::RING_BYTES);  // fp32: [GMAX][D]

  // ---- loads: the page of a tile (or of each of its tokens, one a lane) is
  // looked up one tile before the tile's copies are issued.
  constexpr int ROWS = 32 / CHUNKS > 0 ? 32 / CHUNKS : 1;  // rows of one pass of the warp
  const int my_row = lane / CHUNKS, my_col = lane % CHUNKS;
  int32_t page = -1, slot = 0;
  auto look_up = [&]() {
    const int32_t t = ahead.tile * kTileTokens + (UNI ? 0 : (lane & 15));
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
    const T* kb = static_cast<const T*>(p.kv.k) + ahead.head * p.kv.k_head_stride +
                  my_col * (16 / sizeof(T));
    const T* vb = static_cast<const T*>(p.kv.v) + ahead.head * p.kv.v_head_stride +
                  my_col * (16 / sizeof(T));
    const int64_t kt = p.kv.k_token_stride, vt = p.kv.v_token_stride;
    const int32_t left = ahead.len - ahead.tile * kTileTokens;
    if constexpr (UNI) {
      const int64_t pp = page >= 0 ? page : 0;
      const int32_t rows = page >= 0 ? left : 0;
      kb += pp * p.kv.k_page_stride + (slot + my_row) * kt;
      vb += pp * p.kv.v_page_stride + (slot + my_row) * vt;
#pragma unroll
      for (int i = 0; i < kTileTokens / ROWS; ++i) {
        const int r = i * ROWS + my_row;
        const uint32_t bytes = r < rows ? 16u : 0u;
        cp_async_16(kdst + swz<C::ROW_BYTES>(r, my_col), kb, bytes);
        cp_async_16(vdst + swz<C::ROW_BYTES>(r, my_col), vb, bytes);
        if (r + ROWS < rows) {  // a row that is not read keeps an address that is
          kb += ROWS * kt;
          vb += ROWS * vt;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kTileTokens / ROWS; ++i) {
        const int r = i * ROWS + my_row;
        const int32_t pg = __shfl_sync(0xffffffffu, page, r);
        const int64_t sl = __shfl_sync(0xffffffffu, slot, r);
        const uint32_t bytes = pg >= 0 ? 16u : 0u;
        const int64_t pp = pg >= 0 ? pg : 0;
        cp_async_16(kdst + swz<C::ROW_BYTES>(r, my_col),
                    kb + pp * p.kv.k_page_stride + (pg >= 0 ? sl * kt : 0), bytes);
        cp_async_16(vdst + swz<C::ROW_BYTES>(r, my_col),
                    vb + pp * p.kv.v_page_stride + (pg >= 0 ? sl * vt : 0), bytes);
      }
    }
  };
  auto issue_next = [&](int stage) {
    if (ahead.u < u1) {
      issue(stage);
      advance(p, ahead);
      if (ahead.u < u1) look_up();
    }
    cp_async_commit();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) issue_next(s);

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

  while (now.u < u1) {
    // Keep the ring full: the slot freed by the previous tile takes a new one.
    issue_next(stage == 0 ? C::STAGES - 1 : stage - 1);

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
        __syncwarp();  // every lane is done with the last item's queries
        float qv[GMAX][E];
#pragma unroll
        for (int r = 0; r < GMAX; ++r)
#pragma unroll
          for (int e = 0; e < E; ++e)
            qv[r][e] =
                r < G ? static_cast<float>(qp[r * p.q_head + e * 32 + lane]) * p.qsign : 0.f;
#pragma unroll
        for (int r = 0; r < GMAX; ++r)
#pragma unroll
          for (int e = 0; e < E; ++e) sm_q[r * D + e * 32 + lane] = qv[r][e];
        __syncwarp();
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
    const int32_t left = now.len - now.tile * kTileTokens;  // tokens from the tile's first on
    if constexpr (MMA) {
      // S = Q . K^T of the 16 tokens: two 8-token tiles.
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
          const int32_t t = (e >> 1) * 8 + 2 * tq + (e & 1);
          x[e] = t < left ? sc[e >> 1][r * 2 + (e & 1)] * p.qscale : -INFINITY;
        }
        float bm = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
        const float m_new = fmaxf(m_run[r], bm);
        if (__any_sync(0xffffffffu, m_new != m_run[r])) {
          const float corr = exp2_approx(m_run[r] - m_new);
          m_run[r] = m_new;
          l_run[r] *= corr;
#pragma unroll
          for (int j = 0; j < NDT; ++j) {
            o[j][r * 2] *= corr;
            o[j][r * 2 + 1] *= corr;
          }
        }
        // fp16: P is kept 2^15 higher, so that fewer small ones fall below the
        // type's normal range; sums and parts carry the same factor.
        // The difference comes first, so that the largest P is 2^15 whatever the
        // size of the scores: 15 - m alone would be rounded, by more than one from
        // 2^24 on, and P leave the type's range.
        constexpr float kUp = Elem16<T>::kUmmaFormat == 0u ? 15.f : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = exp2_approx((x[e] - m_new) + kUp);
        l_run[r] += (x[0] + x[1]) + (x[2] + x[3]);
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
      const bool live = tok < left;
      float4 kf[CHUNKS / 2];
#pragma unroll
      for (int c = 0; c < CHUNKS / 2; ++c)
        kf[c] = ld_shared_v4f(kb + swz<C::ROW_BYTES>(tok, half * (CHUNKS / 2) + c));
      __syncwarp();  // K is read: its place takes the probabilities, [token][head]
      float s[GMAX];
#pragma unroll
      for (int r4 = 0; r4 < GMAX; r4 += HB) {
        if (r4 >= G) {
#pragma unroll
          for (int r = 0; r < HB; ++r) s[r4 + r] = 0.f;
          continue;
        }
        float x[HB], bm[HB];
#pragma unroll
        for (int r = 0; r < HB; ++r) {
          const float4* qf =
              reinterpret_cast<const float4*>(sm_q + (r4 + r) * D) + half * (CHUNKS / 2);
          float2 d0 = make_float2(0.f, 0.f), d1 = d0;
#pragma unroll
          for (int c = 0; c < CHUNKS / 2; ++c) {
            const float4 q4 = qf[c];
            d0 = fma_f32x2(make_float2(q4.x, q4.y), make_float2(kf[c].x, kf[c].y), d0);
            d1 = fma_f32x2(make_float2(q4.z, q4.w), make_float2(kf[c].z, kf[c].w), d1);
          }
          x[r] = (d0.x + d0.y) + (d1.x + d1.y);
        }
#pragma unroll
        for (int r = 0; r < HB; ++r) x[r] += __shfl_xor_sync(0xffffffffu, x[r], 16);
#pragma unroll
        for (int r = 0; r < HB; ++r) bm[r] = live ? x[r] : -FLT_MAX;
#pragma unroll
        for (int w = 8; w > 0; w >>= 1)
#pragma unroll
          for (int r = 0; r < HB; ++r)
            bm[r] = fmaxf(bm[r], __shfl_xor_sync(0xffffffffu, bm[r], w));
        // The maxima are the same in every lane.
        bool grows = false;
#pragma unroll
        for (int r = 0; r < HB; ++r) grows |= bm[r] > m_run[r4 + r];
        if (grows) {
#pragma unroll
          for (int r = 0; r < HB; ++r) {
            const float m_new = fmaxf(m_run[r4 + r], bm[r]);
            const float corr = m_run[r4 + r] == -FLT_MAX
                                   ? 0.f
                                   : exp2f((m_run[r4 + r] - m_new) * p.qscale);
            m_run[r4 + r] = m_new;
            l_run[r4 + r] *= corr;
#pragma unroll
            for (int e = 0; e < E; ++e) accf[r4 + r][e] *= corr;
          }
        }
#pragma unroll
        for (int r = 0; r < HB; ++r) {
          // The difference is taken before it is scaled: that of large scores (2^24 and
          // more) is exact, and zero for the largest, where a rounding of the scaled
          // ones would be worth a power of two.
          s[r4 + r] = live ? exp2f((x[r] - m_run[r4 + r]) * p.qscale) : 0.f;
          l_run[r4 + r] += half == 0 ? s[r4 + r] : 0.f;  // one of the two copies counts
        }
      }
      if (half == 0) {
#pragma unroll
        for (int r = 0; r < GMAX; r += 4)
          st_shared_v4(kb + (tok * GMAX + r) * 4, __float_as_uint(s[r]), __float_as_uint(s[r + 1]),
                       __float_as_uint(s[r + 2]), __float_as_uint(s[r + 3]));
      }
      __syncwarp();
#pragma unroll 8
      for (int t = 0; t < kTileTokens; ++t) {
        float2 vf[E / 2];
        const uint32_t a = vb + swz<C::ROW_BYTES>(t, (lane * E) / 4) + ((lane * E) % 4) * 4;
        if constexpr (E == 4) {
          const float4 v4 = ld_shared_v4f(a);
          vf[0] = make_float2(v4.x, v4.y);
          vf[1] = make_float2(v4.z, v4.w);
        } else {
          vf[0] = make_float2(ld_shared_f32(a), ld_shared_f32(a + 4));
        }
#pragma unroll
        for (int r4 = 0; r4 < GMAX; r4 += 4) {
          if (r4 >= G) continue;
          const float4 p4 = ld_shared_v4f(kb + (t * GMAX + r4) * 4);
          const float pt[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < E; e += 2) {
              const float2 w = fma_f32x2(make_float2(pt[r], pt[r]), vf[e / 2],
                                         make_float2(accf[r4 + r][e], accf[r4 + r][e + 1]));
              accf[r4 + r][e] = w.x;
              accf[r4 + r][e + 1] = w.y;
            }
        }
      }
    }
    __syncwarp();  // the slot is refilled at the top of the next tile
    if (++stage == C::STAGES) stage = 0;

    // ---- the item, or this share's part of it, ends here
    const bool ends = now.tile + 1 == now.tiles;
    if (ends || now.u + 1 == u1) {
      const bool starts = now.u - now.tile >= u0;  // the share has the item's first tile
      const bool whole = starts && ends;
      const int part = 2 * me + (first_segment ? 0 : 1);
      if (starts && lane == 0) {
        const int64_t item = static_cast<int64_t>(now.b) * p.hkv + now.head;
        p.joins[item * 2] = ends ? -1 : part;
        p.joins[item * 2 + 1] =
            static_cast<int32_t>((now.u - now.tile + now.tiles - 1) / share);
      }
      T* op = static_cast<T*>(p.out) + now.b * p.out_batch +
              static_cast<int64_t>(now.head) * G * p.out_head;
      float* wp = p.ws + static_cast<int64_t>(part) * G * D;
      float* ml = p.ws + static_cast<int64_t>(2 * p.warps) * G * D + static_cast<int64_t>(part) * G * 2;
      if constexpr (MMA) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float l = l_run[r];
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          const int row = g + r * 8;
          if (row >= G) continue;
          if (whole) {
            const float inv = 1.f / l;
#pragma unroll
            for (int j = 0; j < NDT; ++j)
              *reinterpret_cast<uint32_t*>(op + row * p.out_head + j * 8 + 2 * tq) =
                  float2_to_pair<T>(o[j][r * 2] * inv, o[j][r * 2 + 1] * inv);
          } else {
#pragma unroll
            for (int j = 0; j < NDT; ++j)
              *reinterpret_cast<float2*>(wp + row * D + j * 8 + 2 * tq) =
                  make_float2(o[j][r * 2], o[j][r * 2 + 1]);
            if (tq == 0) *reinterpret_cast<float2*>(ml + row * 2) = make_float2(m_run[r], l);
          }
        }
      } else {
#pragma unroll
        for (int r = 0; r < GMAX; ++r) {
          if (r >= G) continue;
          float l = l_run[r];
#pragma unroll
          for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (whole)
              op[r * p.out_head + lane * E + e] = from_float<T>(accf[r][e] / l);
            else
              wp[r * D + lane * E + e] = accf[r][e];
          if (!whole && lane == 0) *reinterpret_cast<float2*>(ml + r * 2) = make_float2(m_run[r], l);
        }
      }
      fresh = true;
      first_segment = false;
    }
    advance(p, now);
  }
}

// Sum of the parts s0, s0 + step, ... of one row, brought to their largest
// maximum; a lane holds D / 32 dims.  The loads of U parts do not depend on one another.
template <int E, int U>
__device__ __forceinline__ void join_parts(const PagedDecodeParams& p, const float* mls, int first,
                                           int w0, int n, int s0, int step, int row, int lane,
                                           float (&acc)[E], float& mx, float& den) {
  mx = -FLT_MAX;
  den = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (; s0 < n; s0 += U * step) {
    float2 ml[U];
    float x[U][E];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int s = s0 + i * step;
      ml[i] = make_float2(-FLT_MAX, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = 0.f;
      if (s < n) {
        // The first part, then the first slots of the warps up to the last.
        const int64_t at = static_cast<int64_t>(s == 0 ? first : 2 * (w0 + s)) * p.group + row;
        ml[i] = *reinterpret_cast<const float2*>(mls + at * 2);
        if constexpr (E == 4) {
          const float4 v = *reinterpret_cast<const float4*>(p.ws + at * (E * 32) + lane * 4);
          x[i][0] = v.x; x[i][1] = v.y; x[i][2] = v.z; x[i][3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(p.ws + at * (E * 32) + lane * 2);
          x[i][0] = v.x; x[i][1] = v.y;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float m_new = fmaxf(mx, ml[i].x);
      const float c = exp2f((mx - m_new) * p.unit), f = exp2f((ml[i].x - m_new) * p.unit);
      mx = m_new;
      den = fmaf(ml[i].y, f, den * c);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(x[i][e], f, acc[e] * c);
    }
  }
}

// Joins the parts of every item that was cut, in share order, and writes the
// zeros of empty sequences.  A CTA has join_rows query heads of one KV head:
// four where there are many rows (and so few parts of each), a warp each; one
// where there are few.  An item of many parts is joined by the W warps together,
// row by row.
template <typename T, int D, int W, int U>  // W warps, U parts at once
__global__ void __launch_bounds__(32 * W) paged_join_kernel(const PagedDecodeParams p) {
  constexpr int E = D / 32;
  __shared__ float sm_acc[W][D];
  __shared__ float2 sm_ml[W];
  griddep_launch_dependents();
  griddep_wait();
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  const int G = p.group, per_head = (G + p.join_rows - 1) / p.join_rows;
  const int head = blockIdx.x / per_head, b = blockIdx.y;
  const int row0 = (blockIdx.x - head * per_head) * p.join_rows;
  const int rows = min(p.join_rows, G - row0);
  T* op = static_cast<T*>(p.out) + b * p.out_batch +
          (static_cast<int64_t>(head) * G + row0) * p.out_head;
  const int2 join =
      *reinterpret_cast<const int2*>(p.joins + (static_cast<int64_t>(b) * p.hkv + head) * 2);
  if (p.seq_lens[b] <= 0 || p.kv.max_pages == 0) {
    for (int i = static_cast<int>(threadIdx.x); i < rows * D; i += 32 * W)
      op[(i / D) * p.out_head + i % D] = from_float<T>(0.f);
    return;
  }
  if (join.x < 0) return;
  const int w0 = join.x / 2, n = join.y - w0 + 1;
  const float* mls = p.ws + static_cast<int64_t>(2 * p.warps) * G * D;
  float acc[E], mx, den;
  if (rows > 1 && n <= 16) {
    if (warp < rows) {
      join_parts<E, U>(p, mls, join.x, w0, n, 0, 1, row0 + warp, lane, acc, mx, den);
#pragma unroll
      for (int e = 0; e < E; ++e)
        op[warp * p.out_head + lane * E + e] = from_float<T>(acc[e] / den);
    }
    return;
  }
  for (int r = 0; r < rows; ++r) {
    join_parts<E, U>(p, mls, join.x, w0, n, warp, W, row0 + r, lane, acc, mx, den);
    if (r > 0) __syncthreads();  // the last row's meeting is over
#pragma unroll
    for (int e = 0; e < E; ++e) sm_acc[warp][lane * E + e] = acc[e];
    if (lane == 0) sm_ml[warp] = make_float2(mx, den);
    __syncthreads();
    for (int d = static_cast<int>(threadIdx.x); d < D; d += 32 * W) {
      float m = -FLT_MAX;
#pragma unroll
      for (int w = 0; w < W; ++w) m = fmaxf(m, sm_ml[w].x);
      float num = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = exp2f((sm_ml[w].x - m) * p.unit);
        num = fmaf(sm_acc[w][d], f, num);
        sum = fmaf(sm_ml[w].y, f, sum);
      }
      op[r * p.out_head + d] = from_float<T>(num / sum);
    }
  }
}

// ------------------------------------------------------------------ host side

// 16-bit: an item's queries and end cost about what four tiles do, a part what two
// do (one sequence of 1000 tokens: 9.6 us with shares of two, 11.3 with four; 64
// sequences of 1 to 8192: 69.8 us where an item counts as four at least, 74.2 with
// two, 88.3 with one; back to back, 352 MB a call).  fp32: the scores of a tile take
// longer than either.
static int paged_least(int dtype) { return dtype == FRN_DTYPE_F32 ? 1 : 4; }
static int paged_least_share(int dtype) { return dtype == FRN_DTYPE_F32 ? 1 : 2; }

// Every CTA resident, and no more warps than there can be shares.
static int paged_ctas(int dtype, int64_t batch, int64_t hkv, int64_t d, int64_t capacity, int sms) {
  const int64_t resident =
      static_cast<int64_t>(paged_ctas_per_sm(dtype == FRN_DTYPE_F32, static_cast<int>(d))) * sms;
  const int64_t tiles = batch * hkv * ((capacity + kTileTokens - 1) / kTileTokens);
  const int64_t least = paged_least_share(dtype);
  const int64_t shares = batch * hkv * ((tiles / (batch * hkv) + least - 1) / least);
  const int64_t most = (shares + kPagedWarps - 1) / kPagedWarps;
  return static_cast<int>(most < resident ? (most > 0 ? most : 1) : resident);
}

size_t paged_decode_workspace(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t d,
                              int64_t capacity, int sms) {
  const int64_t warps = kPagedWarps * static_cast<int64_t>(paged_ctas(dtype, batch, hkv, d, capacity, sms));
  const int64_t floats = 2 * warps * (hq / hkv) * (d + 2);
  return static_cast<size_t>((floats + 2 * batch * hkv) * 4);
}

template <typename T, int D, int GMAX>
static int launch_paged(const PagedDecodeProblem& g, PagedDecodeParams& p, cudaStream_t stream) {
  using C = PagedCfg<T, D, GMAX>;
  const bool uni = g.kv.page_size % kTileTokens == 0;
  auto kern = uni ? paged_decode_kernel<T, D, GMAX, true> : paged_decode_kernel<T, D, GMAX, false>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return set_cuda_error("cudaGetDevice");
  static bool ready[2][kMaxDevices] = {};
  if (dev >= kMaxDevices || !ready[uni][dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    if (e != cudaSuccess) return set_cuda_error("cudaFuncSetAttribute(paged decode)", e);
    if (dev < kMaxDevices) ready[uni][dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.warps / kPagedWarps));
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
  cfg.gridDim = dim3(
      static_cast<unsigned>(p.hkv * ((p.group + p.join_rows - 1) / p.join_rows)),
      static_cast<unsigned>(g.batch));
  cfg.dynamicSmemBytes = 0;
  // Few rows: twice the parts of a row at once, and from 64 parts on twice the warps
  // (32 / 8 heads of 128, one sequence of 1000 tokens, cold, 32 parts: 9.5 us with
  // the first, 10.3 with both, 9.8 with neither; of 4000, 125 parts: 11.9, 10.3,
  // 13.8; a batch of 64 sequences loses 1 us by either).
  const int64_t parts = g.kv.max_pages * g.kv.page_size / (kTileTokens * p.least_share);
  const bool few = g.batch * g.num_q_heads < sm_count(dev) / 2;
  if (few && parts > 64) {
    cfg.blockDim = dim3(2 * kPagedThreads);
    e = cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D, 2 * kPagedWarps, 8>, p);
  } else if (few && parts > 16) {
    e = cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D, kPagedWarps, 8>, p);
  } else {
    e = cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D, kPagedWarps, 4>, p);
  }
  if (e != cudaSuccess) return set_cuda_error("launch paged_join", e);
  return 0;
}

template <typename T, int D>
static int launch_paged_g(const PagedDecodeProblem& g, PagedDecodeParams& p, cudaStream_t s) {
  // fp32: one or two heads, one after the other, where four together would be
  // mostly padding (8 sequences of 8192 tokens, 8 heads of their own, 114 us: a
  // tenth less when it was taken).
  if constexpr (sizeof(T) == 4)
    if (p.group <= 2) return launch_paged<T, D, 4>(g, p, s);
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
  p.join_rows = g.batch * g.num_q_heads > 32 * sm_count(dev) ? 4 : 1;
  p.least = paged_least(g.dtype);
  p.least_share = paged_least_share(g.dtype);
  p.warps = kPagedWarps * paged_ctas(g.dtype, g.batch, g.kv.num_kv_heads, g.kv.head_dim,
                                     g.kv.max_pages * g.kv.page_size, sm_count(dev));
  p.ws = static_cast<float*>(g.workspace);
  p.joins = reinterpret_cast<int32_t*>(
      p.ws + static_cast<int64_t>(2 * p.warps) * p.group * (g.kv.head_dim + 2));
  p.qscale = g.scale * 1.4426950408889634f;  // log2(e)
  p.unit = 1.f;
  p.qsign = 1.f;
  if (g.dtype == FRN_DTYPE_F32) {
    p.qsign = g.scale < 0.f ? -1.f : 1.f;
    p.unit = p.qscale = fabsf(p.qscale);
  }
  switch (g.dtype) {
    case FRN_DTYPE_BF16: return launch_paged_d<__nv_bfloat16>(g, p, stream);
    case FRN_DTYPE_F16: return launch_paged_d<__half>(g, p, stream);
    default: return launch_paged_d<float>(g, p, stream);
  }
}

}  // namespace frn
