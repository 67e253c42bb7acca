// The weights that cached keys receive from many query rows of a request on the 5th-generation tensor cores (tcgen05): the last
// tokens of a prompt, whole prompt portions (attention_weights.cuh has the formula), over a cache in bfloat16 or in 8 bits, heads of
// 64 or 128.
//
// A key's sum needs the logarithm lse of every row's softmax sum first, so there are two launches with one inside:
//
//   rows:  a tile of 128 query rows ((token, head of the group) pairs) stays, tiles of 128 keys pass by, S = Q K^T; a thread per
//          row and half of the columns keeps the running maximum and sum;
//   keys:  a tile of 128 keys stays, tiles of query rows pass by, S^T = K Q^T; a thread per key and half of the columns adds up
//          exp2(s - lse).
//
// In both the tile that stays is the A operand, whose rows are the lanes of tensor memory, and a thread's sums run along its
// lane: no exchange between threads until the end.  The tiles that pass by are cut over the blocks of a cluster, whose sums meet in
// shared memory in the blocks' order: the same bits every time.
//
// Warps 0-3 fetch tiles (cp.async into the swizzled layout, any page size; codes of 8 bits become bfloat16 on the way, exactly, and a
// key's power of two multiplies its scores), warps 4-11 hold the sums, warp 12 issues the products.  Two stages of shared and
// tensor memory, two blocks a multiprocessor.
//
// What bounds it: the exponentials, one a score in each launch (16 a cycle and multiprocessor: 1,024 cycles a tile of 128 x 128,
// whose product takes 256).
//
// Every wait on a barrier is bounded; after a timeout the block raises JLX_STATUS_WAIT_TIMEOUT, waits for its own copies, frees its
// tensor memory and returns.
#include <cooperative_groups.h>

#include "attention_weights.cuh"
#include "mbarrier.cuh"
#include "mma_sync.cuh"

namespace cg = cooperative_groups;

#define TILE 128
#define STAGES 2
#define LOADERS 128                   // threads of the loading warps
#define FIRST_SUM_WARP (LOADERS / 32)
#define SUM_WARPS 8
#define MMA_WARP (FIRST_SUM_WARP + SUM_WARPS)
#define NTHREADS (32 * (MMA_WARP + 1))
#define COLUMNS 64                    // of a tile, a summing thread's
#define HALF_BYTES (TILE * 128)       // a tile's rows of 64 bfloat16 numbers
#define MAX_SPLITS 8

__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void umma_bf16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// A tile's rows of 128 bytes with the swizzle of that many, 8-row groups 1024 bytes apart, running along the contraction.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Bfloat16 operands, float32 accumulator, M = N = 128, both K-major.
#define IDESC ((1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TILE >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24))
// Byte offset of 16-byte chunk c (of DH / 8) of row r in a tile of two halves.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (c >> 3) * HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

struct Span {  // of a tile's query rows
  int p_min, p_max, lo_min, lo_max;
};

struct TcParams {
  WeightsParams P;
  float2* row_info;  // [N, Hq]: (score factor, -lse in base 2)
  int4* spans;       // [R, tiles of a request's rows]: Span
  int q_tiles;
};

template <int DH> struct TcTile {
  static constexpr int BYTES = DH / 64 * HALF_BYTES;
  static constexpr int SMEM = (1 + STAGES) * BYTES + 1024;
};

// What a block has besides its tiles.
struct Shared {
  uint64_t bars[3 * STAGES];        // FULL (the loaders), SFULL (the product), EMPTY (the sums)
  uint32_t tmem;
  int failed, masked[STAGES];
  int span[4];
  float4 col[STAGES][TILE];         // keys: a query row's (factor, -lse, slope, position)
  int lo[STAGES][TILE];             //       its first key
  float scale[STAGES][TILE];        // rows, 8 bits: a key's power of two
  float m[TILE], l[TILE];           // sums on their way out
};

__device__ __forceinline__ uint32_t bar_full(const Shared& sh, int s) { return smem_u32(&sh.bars[s]); }
__device__ __forceinline__ uint32_t bar_sfull(const Shared& sh, int s) { return smem_u32(&sh.bars[STAGES + s]); }
__device__ __forceinline__ uint32_t bar_empty(const Shared& sh, int s) { return smem_u32(&sh.bars[2 * STAGES + s]); }

// The flat row of query row `row` of a request and KV head in q, or -1.
__device__ __forceinline__ int q_row(const RowsParams& P, const RowsItem& it, int hk, int row) {
  const int G = P.Hq / P.Hkv, t = row / G;
  return row < it.cnt * G ? (it.n0 + t) * P.Hq + hk * G + row - t * G : -1;
}

// A warp of the loaders brings its 32 rows of a tile: lane i has row 32 w + i's place in `base` (-1: zeros).
template <int DH>
__device__ __forceinline__ void load_rows(uint32_t dst, const void* base, int flat, int w, int lane) {
  constexpr int CH = DH / 8, AT_ONCE = 32 / CH;
  const int c = lane % CH;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int r = i * AT_ONCE + lane / CH, from = __shfl_sync(0xffffffffu, flat, r);
    cp_async16(dst + chunk_at(w * 32 + r, c), reinterpret_cast<const uint8_t*>(base) + ((size_t)max(from, 0) * CH + c) * 16, from >= 0);
  }
}
// The same from codes of 8 bits.
template <int DH>
__device__ __forceinline__ void load_codes(uint8_t* dst, const void* base, int flat, int w, int lane) {
  constexpr int CH = DH / 16, AT_ONCE = 32 / CH;
  const int c = lane % CH;
  uint4 v[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int from = __shfl_sync(0xffffffffu, flat, i * AT_ONCE + lane / CH);
    v[i] = from >= 0 ? *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(base) + ((size_t)from * CH + c) * 16) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int r = w * 32 + i * AT_ONCE + lane / CH;
    const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    uint32_t o[8];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      o[2 * u] = weights_widen(x[u], 0x9180);
      o[2 * u + 1] = weights_widen(x[u], 0xb3a2);
    }
    *reinterpret_cast<uint4*>(dst + chunk_at(r, 2 * c)) = make_uint4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<uint4*>(dst + chunk_at(r, 2 * c + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
  }
}
template <int DH, bool F8>
__device__ __forceinline__ void load_keys(uint8_t* dst, const void* pages, int flat, int w, int lane) {
  if (F8) load_codes<DH>(dst, pages, flat, w, lane);
  else load_rows<DH>(smem_u32(dst), pages, flat, w, lane);
}
// What a loading thread has brought is there for the products.
__device__ __forceinline__ void loaded(uint32_t bar) {
  cp_async_commit();
  cp_async_wait<0>();
  fence_async_proxy();
  mbar_arrive(bar);
}

__device__ __forceinline__ void give_up(const WeightsParams& P, Shared& sh) {
  atomicOr(P.R.status, JLX_STATUS_WAIT_TIMEOUT);
  *(volatile int*)&sh.failed = 1;
}

// Barriers and tensor memory; every thread of the block calls it.
__device__ __forceinline__ void open_block(Shared& sh, int warp) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full(sh, s), LOADERS);
      mbar_init(bar_sfull(sh, s), 1);
      mbar_init(bar_empty(sh, s), SUM_WARPS);
    }
    sh.failed = 0;
    sh.span[0] = sh.span[2] = 0x7fffffff;
    sh.span[1] = sh.span[3] = (int)0x80000000;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(smem_u32(&sh.tmem), STAGES * TILE);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
__device__ __forceinline__ void close_block(Shared& sh, int warp) {
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) tmem_dealloc(sh.tmem, STAGES * TILE);
}

// The issuing thread: stage t's product of the tile that stays (`a`) with the one that passes by.
template <int DH>
__device__ __forceinline__ void products(const WeightsParams& P, Shared& sh, uint32_t a, uint32_t b, int n_tiles) {
  int t = 0;
  for (; t < n_tiles; ++t) {
    const int s = t % STAGES;
    if (!mbar_wait(bar_full(sh, s), (t / STAGES) & 1)) { give_up(P, sh); break; }
    tc_fence_after();
#pragma unroll
    for (int kk = 0; kk < DH / 16; ++kk) {
      const uint32_t off = (kk >> 2) * HALF_BYTES + (kk & 3) * 32;
      umma_bf16(sh.tmem + s * TILE, desc_k_major(a + off), desc_k_major(b + s * TcTile<DH>::BYTES + off), IDESC, kk != 0);
    }
    umma_commit(bar_sfull(sh, s));
  }
  if (t-- > 0) mbar_wait(bar_sfull(sh, t % STAGES), (t / STAGES) & 1);  // tensor memory is given up after the last one
}

// A summing warp waits for tile t (and for what the loaders wrote beside it).
__device__ __forceinline__ bool await_scores(const WeightsParams& P, Shared& sh, int t, int lane) {
  const int s = t % STAGES;
  const bool ok = mbar_wait(bar_full(sh, s), (t / STAGES) & 1) && mbar_wait(bar_sfull(sh, s), (t / STAGES) & 1);
  if (__all_sync(0xffffffffu, ok)) {
    tc_fence_after();
    return true;
  }
  if (lane == 0) give_up(P, sh);
  return false;
}
__device__ __forceinline__ void release_scores(Shared& sh, int t, int lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar_empty(sh, t % STAGES));
}
__device__ __forceinline__ bool await_stage(const WeightsParams& P, Shared& sh, int t, int lane) {
  if (t < STAGES) return true;
  const bool ok = mbar_wait(bar_empty(sh, t % STAGES), (t / STAGES - 1) & 1);
  if (__all_sync(0xffffffffu, ok) && !*(volatile int*)&sh.failed) return true;
  if (!ok) give_up(P, sh);
  return false;
}

// ----------------------------------------------------------------------------------------- rows: the softmax sums
template <int DH, bool F8>
__global__ void __launch_bounds__(NTHREADS, 2) attention_weights_rows_kernel(const TcParams T) {
  JLX_TL(TL_ATTN_PREFILL);
  const WeightsParams& P = T.P;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(16) Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t *a_p = smem, *b_p = smem + TcTile<DH>::BYTES;
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x % P.splits, tile = blockIdx.x / P.splits, r = blockIdx.y / P.R.Hkv, hk = blockIdx.y - r * P.R.Hkv;
  const int G = P.R.Hq / P.R.Hkv, row0 = tile * TILE;
  RowsItem it;
  if (!weights_request(P, r, it)) return;
  const int n_rows = min(it.cnt * G - row0, TILE);
  if (n_rows <= 0) return;
  open_block(sh, warp);
  // the tile's rows together
  if (warp >= FIRST_SUM_WARP && warp < FIRST_SUM_WARP + 4) {
    const int row = (warp - FIRST_SUM_WARP) * 32 + lane, p = P.R.positions[it.n0 + (row0 + min(row, n_rows - 1)) / G], lo = rows_first_key(P.R, p);
    const int a = __reduce_min_sync(0xffffffffu, p), b = __reduce_max_sync(0xffffffffu, p);
    const int c = __reduce_min_sync(0xffffffffu, lo), d = __reduce_max_sync(0xffffffffu, lo);
    if (lane == 0) {
      atomicMin(&sh.span[0], a);
      atomicMax(&sh.span[1], b);
      atomicMin(&sh.span[2], c);
      atomicMax(&sh.span[3], d);
    }
  }
  __syncthreads();
  const int p_min = sh.span[0], lo_min = sh.span[2], lo_max = sh.span[3];
  if (tid == 0 && split == 0 && hk == 0) T.spans[(size_t)r * T.q_tiles + tile] = make_int4(p_min, sh.span[1], lo_min, lo_max);
  int end_all = rows_end(P.R, it, sh.span[1]);
  if (end_all > min(P.W.max_kv, P.W.width)) end_all = 0;  // (the other launch leaves the request out)
  const int start = lo_min / TILE * TILE, all = end_all > start ? (end_all - start + TILE - 1) / TILE : 0;
  const int per = (all + P.splits - 1) / P.splits, t0 = min(split * per, all), n_tiles = min(per, all - t0), key0 = start + t0 * TILE;
  const int* table = P.R.block_table + (size_t)r * P.R.bt_stride;

  if (warp < FIRST_SUM_WARP) {
    auto key_row = [&](int t) {
      const int place = key0 + t * TILE + warp * 32 + lane;
      return t < n_tiles && place >= lo_min && place < end_all ? rows_cache_row(P.R, table, hk, place) : -1;
    };
    load_rows<DH>(smem_u32(a_p), P.R.q, q_row(P.R, it, hk, row0 + warp * 32 + lane), warp, lane);
    int flat = key_row(0);
    for (int t = 0; t < n_tiles; ++t) {
      const int s = t % STAGES, place0 = key0 + t * TILE;
      if (!await_stage(P, sh, t, lane)) break;
      if (F8) sh.scale[s][warp * 32 + lane] = flat >= 0 ? fp8_scale(P.R.scales[flat]) : 0.f;
      if (tid == 0) sh.masked[s] = place0 < lo_max || place0 + TILE > min(p_min + 1, end_all);
      load_keys<DH, F8>(b_p + s * TcTile<DH>::BYTES, P.R.pages, flat, warp, lane);
      flat = key_row(t + 1);
      loaded(bar_full(sh, s));
    }
    cp_async_commit();
    cp_async_wait<0>();  // (a block without tiles still has the one that stays)
  } else if (warp == MMA_WARP) {
    if (lane == 0) products<DH>(P, sh, smem_u32(a_p), smem_u32(b_p), n_tiles);
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = (warp - FIRST_SUM_WARP) >> 2, row = quarter * 32 + lane;
    const RowsToken tok = rows_token(P.R, it, row0 + min(row, n_rows - 1), hk);
    const int p_last = min(tok.p, end_all - 1);
    const bool bent = P.R.cap_log2 > 0.f || P.R.slopes || !(tok.sc > 0.f);
    const float f = bent ? 1.f : tok.sc;  // what brings the numbers below to base-2 units
    float m = ROWS_NEG_BIG, l = 0.f;
    for (int t = 0; t < n_tiles; ++t) {
      if (!await_scores(P, sh, t, lane)) break;
      const int s = t % STAGES;
      const bool masked = sh.masked[s];
#pragma unroll 1
      for (int c0 = half * COLUMNS; c0 < (half + 1) * COLUMNS; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(sh.tmem + ((uint32_t)(quarter * 32) << 16) + s * TILE + c0, v);
        tmem_ld_wait();
        if (F8) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 k = *reinterpret_cast<const float4*>(&sh.scale[s][c0 + c]);
            v[c] = __float_as_uint(__uint_as_float(v[c]) * k.x);
            v[c + 1] = __float_as_uint(__uint_as_float(v[c + 1]) * k.y);
            v[c + 2] = __float_as_uint(__uint_as_float(v[c + 2]) * k.z);
            v[c + 3] = __float_as_uint(__uint_as_float(v[c + 3]) * k.w);
          }
        }
        const int place = key0 + t * TILE + c0;
        if (bent) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            float x = __uint_as_float(v[c]) * tok.sc;
            if (P.R.cap_log2 > 0.f) x = P.R.cap_log2 * cap_tanh(x);
            v[c] = __float_as_uint(x - tok.slope * (float)(tok.p - place - c));
          }
        }
        if (masked) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (place + c < tok.lo || place + c > p_last) v[c] = __float_as_uint(-INFINITY);
        }
        float top = m;
#pragma unroll
        for (int c = 0; c < 32; ++c) top = fmaxf(top, __uint_as_float(v[c]));
        l *= rows_exp2((m - top) * f);
        m = top;
        const float at = -top * f;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 32; ++c) sum[c & 1] += rows_exp2(fmaf(__uint_as_float(v[c]), f, at));
        l += sum[0] + sum[1];
      }
      release_scores(sh, t, lane);
    }
    m = l == 0.f ? ROWS_NEG_BIG : m * f;
    // the halves of a row, then (below) the blocks of the cluster
    if (half == 1) {
      sh.m[row] = m;
      sh.l[row] = l;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * SUM_WARPS) : "memory");
    if (half == 0) {
      const float top = fmaxf(m, sh.m[row]);
      sh.l[row] = l * rows_exp2(m - top) + sh.l[row] * rows_exp2(sh.m[row] - top);
      sh.m[row] = top;
    }
  }
  close_block(sh, warp);
  cluster.sync();
  const int share = (TILE + P.splits - 1) / P.splits, row = split * share + tid;
  if (tid < share && row < n_rows) {
    float m = ROWS_NEG_BIG, l = 0.f;
    for (int q = 0; q < P.splits; ++q) m = fmaxf(m, *cluster.map_shared_rank(&sh.m[row], q));
    for (int q = 0; q < P.splits; ++q) l += *cluster.map_shared_rank(&sh.l[row], q) * rows_exp2(*cluster.map_shared_rank(&sh.m[row], q) - m);
    const RowsToken tok = rows_token(P.R, it, row0 + row, hk);
    if (P.R.sink) l += exp2f(P.R.sink[tok.head] * LOG2E - m);  // (a row that sees nothing: infinite)
    T.row_info[(size_t)tok.n * P.R.Hq + tok.head] = make_float2(tok.sc, l == 0.f ? -INFINITY : -(m + log2f(l)));
  }
  cluster.sync();
}

// ----------------------------------------------------------------------------------------- keys: their weights
template <int DH, bool F8>
__global__ void __launch_bounds__(NTHREADS, 2) attention_weights_keys_kernel(const TcParams T) {
  JLX_TL(TL_ATTN_PREFILL);
  const WeightsParams& P = T.P;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(16) Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t *a_p = smem, *b_p = smem + TcTile<DH>::BYTES;
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x % P.splits, key0 = blockIdx.x / P.splits * TILE, r = blockIdx.y / P.R.Hkv, hk = blockIdx.y - r * P.R.Hkv;
  const size_t out_row = blockIdx.y;
  const int G = P.R.Hq / P.R.Hkv;
  RowsItem it;
  auto leave = [&]() { weights_copy(P, out_row, key0, min(key0 + TILE, P.W.width), split * NTHREADS + tid, P.splits * NTHREADS); };
  if (!weights_request(P, r, it)) { leave(); return; }
  const int tiles = (it.cnt * G + TILE - 1) / TILE, limit = min(P.W.max_kv, P.W.width);
  const int4* spans = T.spans + (size_t)r * T.q_tiles;
  // row tiles that see some of these keys, every splits-th of them this block's
  auto sees = [&](const int4& s) { return s.y >= key0 && s.z < key0 + TILE; };
  int n_tiles = 0, any = 0, bad = 0, end_all = 0, first = 0x7fffffff;
  for (int t = tid; t < (tiles + NTHREADS - 1) / NTHREADS * NTHREADS; t += NTHREADS) {
    const int4 s = t < tiles ? spans[t] : make_int4(0, -1, 0, 0);
    bad |= __syncthreads_or(s.y >= limit);
    any |= __syncthreads_or(sees(s));
    n_tiles += __syncthreads_count(sees(s) && t % P.splits == split);
    end_all = max(end_all, s.y + 1);
    if (t < tiles) first = min(first, s.z);
  }
  if (bad || !any) {  // (the whole cluster)
    if (bad && tid == 0) atomicOr(P.R.status, JLX_STATUS_BAD_PAGE);
    leave();
    return;
  }
  open_block(sh, warp);
  atomicMax(&sh.span[1], end_all);
  atomicMin(&sh.span[2], first);
  __syncthreads();
  end_all = min(sh.span[1], rows_capacity(P.R));
  first = sh.span[2];
  const int* table = P.R.block_table + (size_t)r * P.R.bt_stride;

  if (warp < FIRST_SUM_WARP) {
    const int place = key0 + warp * 32 + lane;
    load_keys<DH, F8>(a_p, P.R.pages, place >= first && place < end_all ? rows_cache_row(P.R, table, hk, place) : -1, warp, lane);
    int t = 0;
    bool ok = true;
    for (int base = split; base < tiles && ok; base += 32 * P.splits) {
      // a lane looks at one of 32 row tiles
      const int mine = base + lane * P.splits;
      const int4 s_mine = mine < tiles ? spans[mine] : make_int4(0, -1, 0, 0);
      uint32_t todo = __ballot_sync(0xffffffffu, mine < tiles && sees(s_mine));
      const uint32_t masked = __ballot_sync(0xffffffffu, s_mine.x < min(key0 + TILE, end_all) - 1 || s_mine.w > key0 || (mine + 1) * TILE > it.cnt * G);
      for (; todo; todo &= todo - 1, ++t) {
        const int i = __ffs(todo) - 1, row = (base + i * P.splits) * TILE + warp * 32 + lane, s = t % STAGES;
        const int flat = q_row(P.R, it, hk, row);
        float4 col = make_float4(0.f, -INFINITY, 0.f, 0.f);
        int lo = 0x7fffffff;
        if (flat >= 0) {
          const float2 info = T.row_info[flat];
          const int p = P.R.positions[it.n0 + row / G];
          col = make_float4(info.x, info.y, P.R.slopes ? P.R.slopes[hk * G + row % G] * LOG2E : 0.f, __int_as_float(p));
          lo = rows_first_key(P.R, p);
        }
        ok = await_stage(P, sh, t, lane);
        if (!ok) break;
        sh.col[s][warp * 32 + lane] = col;
        sh.lo[s][warp * 32 + lane] = lo;
        if (tid == 0) sh.masked[s] = masked >> i & 1;
        load_rows<DH>(smem_u32(b_p + s * TcTile<DH>::BYTES), P.R.q, flat, warp, lane);
        loaded(bar_full(sh, s));
      }
    }
    cp_async_commit();
    cp_async_wait<0>();  // (a block without tiles still has the one that stays)
  } else if (warp == MMA_WARP) {
    if (lane == 0) products<DH>(P, sh, smem_u32(a_p), smem_u32(b_p), n_tiles);
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = (warp - FIRST_SUM_WARP) >> 2, row = quarter * 32 + lane, place = key0 + row;
    const bool bent = P.R.cap_log2 > 0.f || P.R.slopes;
    float ks = 1.f;
    if (F8) {
      const int flat = place >= first && place < end_all ? rows_cache_row(P.R, table, hk, place) : -1;
      ks = flat >= 0 ? fp8_scale(P.R.scales[flat]) : 0.f;
    }
    float sum[2] = {0.f, 0.f};
    for (int t = 0; t < n_tiles; ++t) {
      if (!await_scores(P, sh, t, lane)) break;
      const int s = t % STAGES;
      const bool masked = sh.masked[s];
#pragma unroll 1
      for (int c0 = half * COLUMNS; c0 < (half + 1) * COLUMNS; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(sh.tmem + ((uint32_t)(quarter * 32) << 16) + s * TILE + c0, v);
        tmem_ld_wait();
        if (masked || bent) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float4 q = sh.col[s][c0 + c];
            const int p = __float_as_int(q.w);
            float x = __uint_as_float(v[c]);
            if (F8) x *= ks;
            x *= q.x;
            if (P.R.cap_log2 > 0.f) x = P.R.cap_log2 * cap_tanh(x);
            x = x - q.z * (float)(p - place) + q.y;
            sum[c & 1] += place >= sh.lo[s][c0 + c] && place <= p ? rows_exp2(x) : 0.f;
          }
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float2 q = *reinterpret_cast<const float2*>(&sh.col[s][c0 + c]);
            float x = __uint_as_float(v[c]);
            if (F8) x *= ks;
            sum[c & 1] += rows_exp2(fmaf(x, q.x, q.y));
          }
        }
      }
      release_scores(sh, t, lane);
    }
    if (half == 1) sh.l[row] = sum[0] + sum[1];
    asm volatile("bar.sync 1, %0;" ::"n"(32 * SUM_WARPS) : "memory");
    if (half == 0) sh.l[row] += sum[0] + sum[1];
  }
  close_block(sh, warp);
  cluster.sync();
  const int share = (TILE + P.splits - 1) / P.splits, row = split * share + tid, place = key0 + row;
  if (tid < share && row < TILE && place < P.W.width) {
    float w = 0.f;
    if (place < end_all)
      for (int q = 0; q < P.splits; ++q) w += *cluster.map_shared_rank(&sh.l[row], q);
    const size_t at = out_row * P.W.width + place;
    P.W.out[at] = (P.W.add ? P.W.add[at] : 0.f) + w;
  }
  cluster.sync();
}

// -------------------------------------------------------------------------------------------- host
template <typename Kernel>
static int launch_tc(Kernel kernel, int smem, dim3 grid, int splits, const TcParams& T, cudaStream_t stream) {
  JLX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(NTHREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  JLX_CUDA(cudaLaunchKernelEx(&cfg, kernel, T));
  return 0;
}

template <int DH, bool F8>
static int launch_both(TcParams& T, int rows_splits, int keys_splits, cudaStream_t stream) {
  const unsigned pairs = (unsigned)(T.P.R.n_requests * T.P.R.Hkv);
  T.P.splits = rows_splits;
  if (int e = launch_tc(attention_weights_rows_kernel<DH, F8>, TcTile<DH>::SMEM, dim3((unsigned)(T.q_tiles * rows_splits), pairs), rows_splits, T, stream)) return e;
  T.P.splits = keys_splits;
  return launch_tc(attention_weights_keys_kernel<DH, F8>, TcTile<DH>::SMEM, dim3((unsigned)((T.P.W.width + TILE - 1) / TILE * keys_splits), pairs), keys_splits, T, stream);
}

// Scratch: float2 [N * Hq], then (on 16 bytes) int4 [R * ceil(max_count * G / 128)].
JLX_API int jlx_attention_weights_tc(const RowsArgs* rows_args, const WeightsArgs* args, int rows_splits, int keys_splits, void* stream_) {
  TcParams T;
  if (int e = rows_params(*rows_args, T.P.R)) return e;
  T.P.W = *args;
  T.P.buf_keys = 0;
  const RowsParams& R = T.P.R;
  JLX_REQUIRE(rows_splits >= 1 && rows_splits <= MAX_SPLITS && keys_splits >= 1 && keys_splits <= MAX_SPLITS, "attention_weights: %d and %d blocks share tiles", rows_splits, keys_splits);
  JLX_REQUIRE((long long)R.n_requests * R.Hkv <= 65535, "attention_weights: %d requests of %d KV heads are too many for a launch", R.n_requests, R.Hkv);
  JLX_REQUIRE((long long)R.N * R.Hq < (1ll << 31), "attention_weights: %d rows of %d heads are too many", R.N, R.Hq);
  JLX_REQUIRE(T.P.W.scratch && ((uintptr_t)T.P.W.scratch & 15) == 0, "attention_weights: scratch is needed, on 16 bytes");
  T.row_info = reinterpret_cast<float2*>(T.P.W.scratch);
  T.spans = reinterpret_cast<int4*>(T.P.W.scratch + ((size_t)R.N * R.Hq * 2 + 3) / 4 * 4);
  T.q_tiles = (int)(((long long)R.max_count * (R.Hq / R.Hkv) + TILE - 1) / TILE);
  cudaStream_t stream = (cudaStream_t)stream_;
  if (rows_args->dh == 128) return R.scales ? launch_both<128, true>(T, rows_splits, keys_splits, stream) : launch_both<128, false>(T, rows_splits, keys_splits, stream);
  return R.scales ? launch_both<64, true>(T, rows_splits, keys_splits, stream) : launch_both<64, false>(T, rows_splits, keys_splits, stream);
}
