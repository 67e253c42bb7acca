// The weights that cached keys receive from many query rows of a request on the 5th-generation tensor cores (tcgen05): the last
// tokens of a prompt, whole prompt portions (attention_weights.cuh has the formula), over a cache in bfloat16 or in 8 bits, heads of
// 64 or 128.
//
// A key's sum needs the logarithm lse of every row's softmax sum first, so there are two launches with one inside:
//
//   rows:  a tile of 128 query rows ((token, head of the group) pairs) stays, tiles of 128 keys pass by, S = Q K^T; two threads
//          per row keep the running maximum and sum;
//   keys:  a tile of 128 keys stays, tiles of 128 query rows pass by, S^T = K Q^T; two threads per key add up exp2(s - lse).
//
// In both the tile that stays is the A operand, whose rows are the lanes of tensor memory, and a thread's sums run along its lane,
// over half of the columns: no exchange between threads until the end.  The tiles that pass by are cut over
// the blocks of a cluster, whose sums meet in shared memory in the blocks' order: the same bits every time.
//
// Warps 0-3 fetch tiles (cp.async into the swizzled layout, any page size; codes of 8 bits become bfloat16 on the way, exactly, and a
// key's power of two multiplies its scores), warps 4-11 hold the sums, one thread issues the products.  Two blocks a multiprocessor.
//
// What bounds it: the exponentials, one a score in each launch (16 a cycle and multiprocessor: 1,024 cycles a tile of 128 x 128,
// whose product takes 256), at 80 % of that rate while a block works; then the way of a block to its first scores (8,000 cycles) and
// rounds of blocks that do not come out even.  Measured (B200, 40 heads on 8 of 128): 2,048 tokens behind 1,500 191 us, 277 TFLOP/s;
// the last 32 tokens of 8 sessions of up to 8,192 keys 115 us.
// Tried and slower: tiles of 64 passing by, whose products are accepted no faster than those of 128 (244 and 165 us); the tile that stays in
// tensor memory; exponentials by a polynomial for a quarter or half of them (219 and 245 us for 212: the instructions it takes are as scarce).
//
// Every wait on a barrier is bounded; after a timeout the block raises JLX_STATUS_WAIT_TIMEOUT, waits for its own copies, frees its
// tensor memory and returns.
#include <cooperative_groups.h>
#include <stddef.h>

#include "attention_weights.cuh"
#include "mbarrier.cuh"
#include "mma_sync.cuh"

namespace cg = cooperative_groups;

#define TILE 128                      // rows of the tile that stays
#define PASS 128                      // of one that passes by
// Whoever waits on a barrier waits for every one of its phases in turn: a parity cannot tell a phase from the one two before.
#define LOADERS 4                     // loading warps: two for the even tiles, two for the odd ones
#define STAGES 2                      // tiles in shared memory, free again after their product
#define BUFS 2                        // products in tensor memory
// What stands beside a tile is read until its sums are done.  Its place is written again when tile t - STAGES has had its product,
// which waited for the sums of tile t - STAGES - BUFS: SLOTS places need no barrier that says they are free.
#define SLOTS (STAGES + BUFS)
#define FIRST_SUM_WARP LOADERS
#define SUM_WARPS 8
#define MMA_WARP (FIRST_SUM_WARP + SUM_WARPS)
#define NTHREADS (32 * (MMA_WARP + 1))
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
#define IDESC ((1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(PASS >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24))
// Byte offset of 16-byte chunk c (of DH / 8) of row r in a tile: entries 0-63 and 64-127 lie in halves of their own.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (c >> 3) * (PASS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

// Two float32 operations per instruction (IEEE, as their one-value forms).
__device__ __forceinline__ uint64_t pack2(float a, float b) { return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32); }
__device__ __forceinline__ float low2(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high2(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t exp2_unit2(uint64_t x) { return pack2(rows_exp2(low2(x)), rows_exp2(high2(x))); }

struct TcParams {
  WeightsParams P;
  float2* row_info;  // [N, Hq]: (score factor, -lse in base 2)
  int4* spans;       // [R, tiles of a request's rows]: the smallest and largest position, and first key, of its rows
  int q_tiles;
  int key_tiles;     // that a block has one after the other
};

template <int DH> struct TcTile {
  static constexpr int BYTES = DH * 2 * PASS;
  static constexpr int SMEM = (1 + STAGES) * BYTES + 1024;
};

// mbar_wait that sleeps until the phase ends or 20 us are over: polls would take issue slots from the sums.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < JLX_WAIT_LIMIT / 64; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
    if (ok) return true;
  }
  return false;
}

// What a block has besides its tiles.
struct Shared {
  uint64_t bars[2 * STAGES + 2 * BUFS + SLOTS + 1];  // FULL (the loaders), EMPTY, SFULL (the product), FREE (the sums), BESIDE (the loaders), the tile that stays
  uint32_t tmem;
  int failed, masked[SLOTS], columns[SLOTS];
  int span[4];
  // of a tile that passes by.  keys: a query row's score factor, -lse, slope, position and first key; rows, 8 bits: a key's power of two
  alignas(16) float factor[SLOTS][PASS];
  alignas(16) float lse[SLOTS][PASS];
  alignas(16) int pos[SLOTS][PASS];
  alignas(16) int lo[SLOTS][PASS];
  float slope[SLOTS][PASS];
  float m[TILE], l[TILE];           // sums on their way out
};

static_assert(offsetof(Shared, factor) % 16 == 0 && offsetof(Shared, lse) % 16 == 0 && offsetof(Shared, pos) % 16 == 0 && offsetof(Shared, lo) % 16 == 0 && alignof(Shared) == 16, "four columns' numbers are one load");

__device__ __forceinline__ uint32_t bar_full(const Shared& sh, int s) { return smem_u32(&sh.bars[s]); }
__device__ __forceinline__ uint32_t bar_empty(const Shared& sh, int s) { return smem_u32(&sh.bars[STAGES + s]); }
__device__ __forceinline__ uint32_t bar_sfull(const Shared& sh, int t) { return smem_u32(&sh.bars[2 * STAGES + t % BUFS]); }
__device__ __forceinline__ uint32_t bar_free(const Shared& sh, int t) { return smem_u32(&sh.bars[2 * STAGES + BUFS + t % BUFS]); }
__device__ __forceinline__ uint32_t bar_beside(const Shared& sh, int t) { return smem_u32(&sh.bars[2 * STAGES + 2 * BUFS + t % SLOTS]); }
__device__ __forceinline__ uint32_t bar_stays(const Shared& sh) { return smem_u32(&sh.bars[2 * STAGES + 2 * BUFS + SLOTS]); }
__device__ __forceinline__ uint32_t scores_at(const Shared& sh, int t) { return sh.tmem + t % BUFS * PASS; }

// The flat row of query row `row` of a request and KV head in q, or -1.
__device__ __forceinline__ int q_row(const RowsParams& P, const RowsItem& it, int hk, int row) {
  const int G = P.Hq / P.Hkv, t = row / G;
  return row < it.cnt * G ? (it.n0 + t) * P.Hq + hk * G + row - t * G : -1;
}

// A warp brings 32 rows of a tile, from row0 (a multiple of 32) on: lane i has the place in `base` of row row0 + i (-1: zeros).  Eight
// lanes have 128 bytes of a row, whose places in the tile are two patterns in turn: few instructions stand beside the copies.
template <int DH>
__device__ __forceinline__ void load_rows(uint32_t dst, int row0, const void* base, int flat, int lane) {
  const int r = lane >> 3, c = lane & 7;
  const uint32_t at[2] = {dst + (row0 + r) * 128 + ((c ^ r) << 4), dst + (row0 + r) * 128 + ((c ^ (r + 4)) << 4)};
  const uint8_t* src = reinterpret_cast<const uint8_t*>(base) + c * 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int from = __shfl_sync(0xffffffffu, flat, i * 4 + r);
    const uint8_t* p = src + (size_t)max(from, 0) * (DH * 2);
#pragma unroll
    for (int h = 0; h < DH / 64; ++h) cp_async16(at[i & 1] + i * 512 + h * (PASS * 128), p + h * 128, from >= 0);
  }
}
// The same from codes of 8 bits, through registers.
template <int DH>
__device__ __forceinline__ void load_codes(uint8_t* dst, int row0, const void* base, int flat, int lane) {
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
    const int r = row0 + i * AT_ONCE + lane / CH;
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
template <int DH, bool CODES>
__device__ __forceinline__ void load_part(uint8_t* dst, int row0, const void* base, int flat, int lane) {
  if (CODES) load_codes<DH>(dst, row0, base, flat, lane);
  else load_rows<DH>(smem_u32(dst), row0, base, flat, lane);
}
// What a thread has brought of a tile is there for the products.
__device__ __forceinline__ void loaded(uint32_t bar) {
  asm volatile("cp.async.wait_all;" ::: "memory");
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
      mbar_init(bar_full(sh, s), 32 * LOADERS / 2);
      mbar_init(bar_empty(sh, s), 1);
    }
    for (int b = 0; b < BUFS; ++b) {
      mbar_init(bar_sfull(sh, b), 1);
      mbar_init(bar_free(sh, b), SUM_WARPS);
    }
    for (int t = 0; t < SLOTS; ++t) mbar_init(bar_beside(sh, t), 32 * LOADERS / 2);
    mbar_init(bar_stays(sh), TILE);
    sh.failed = 0;
    sh.span[0] = sh.span[2] = 0x7fffffff;
    sh.span[1] = sh.span[3] = (int)0x80000000;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(smem_u32(&sh.tmem), 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
__device__ __forceinline__ void close_block(Shared& sh, int warp) {
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) tmem_dealloc(sh.tmem, 256);
}

// The issuing thread: the products of the tile that stays (the `stays`-th of the block) with those that pass by, [t, end).
template <int DH>
__device__ __forceinline__ void products(const WeightsParams& P, Shared& sh, uint32_t a, int t, int end, int stays) {
  const int begin = t;
  bool ok = t < end && bar_wait(bar_stays(sh), stays & 1);
  for (; t < end && ok; ++t) {
    const int s = t % STAGES;
    ok = (t < BUFS || bar_wait(bar_free(sh, t - BUFS), ((t - BUFS) / BUFS) & 1)) && bar_wait(bar_full(sh, s), (t / STAGES) & 1);
    if (!ok) break;
    tc_fence_after();
#pragma unroll
    for (int kk = 0; kk < DH / 16; ++kk) {  // 16 entries: 32 bytes of the rows
      const uint32_t at = a + (kk >> 2) * (PASS * 128) + (kk & 3) * 32;
      umma_bf16(scores_at(sh, t), desc_k_major(at), desc_k_major(at + (1 + s) * TcTile<DH>::BYTES), IDESC, kk != 0);
    }
    umma_commit(bar_sfull(sh, t));
    umma_commit(bar_empty(sh, s));
  }
  if (t > begin) bar_wait(bar_sfull(sh, t - 1), ((t - 1) / BUFS) & 1);  // tensor memory is given up after the last one
  if (!ok && begin < end) give_up(P, sh);
}

// A summing warp waits for tile t (and for what its loader wrote beside it).
__device__ __forceinline__ bool await_scores(const WeightsParams& P, Shared& sh, int t, int lane) {
  const bool ok = bar_wait(bar_beside(sh, t), (t / SLOTS) & 1) && bar_wait(bar_sfull(sh, t), (t / BUFS) & 1);
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
  if (lane == 0) mbar_arrive(bar_free(sh, t));
}
__device__ __forceinline__ bool await_stage(const WeightsParams& P, Shared& sh, int t, int lane) {
  if (t < STAGES) return true;
  const bool ok = bar_wait(bar_empty(sh, t % STAGES), (t / STAGES - 1) & 1);
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
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // the last tiles of the rows see the most keys: they come first
  const int split = blockIdx.x % P.splits, pair = blockIdx.x / P.splits, r = pair / P.R.Hkv, hk = pair - r * P.R.Hkv, tile = T.q_tiles - 1 - blockIdx.y;
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
    const int c = __reduce_min_sync(0xffffffffu, p < 0 ? 0x7fffffff : lo), d = __reduce_max_sync(0xffffffffu, lo);  // (a row that sees nothing has no first key)
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
  const int start = lo_min / PASS * PASS, all = end_all > start ? (end_all - start + PASS - 1) / PASS : 0;
  const int per = (all + P.splits - 1) / P.splits, t0 = min(split * per, all), n_tiles = min(per, all - t0), key0 = start + t0 * PASS;
  const int* table = P.R.block_table + (size_t)r * P.R.bt_stride;

  if (warp < FIRST_SUM_WARP) {
    const int part = (warp >> 1) * 64;
    for (int t = warp & 1; t < n_tiles; t += 2) {
      const int s = t % STAGES, place0 = key0 + t * PASS;
      int flat[2];
      float scale[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int place = place0 + part + h * 32 + lane;
        flat[h] = place >= lo_min && place < end_all ? rows_cache_row(P.R, table, hk, place) : -1;
        if (F8) scale[h] = flat[h] >= 0 ? fp8_scale(P.R.scales[flat[h]]) : 0.f;
      }
      if (!await_stage(P, sh, t, lane)) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (F8) sh.factor[t % SLOTS][part + h * 32 + lane] = scale[h];
        load_part<DH, F8>(smem + (1 + s) * TcTile<DH>::BYTES, part + h * 32, P.R.pages, flat[h], lane);
      }
      if (tid < 64) sh.masked[t % SLOTS] = place0 < lo_max || place0 + PASS > min(p_min + 1, end_all);
      mbar_arrive(bar_beside(sh, t));
      loaded(bar_full(sh, s));
    }
  } else if (warp == MMA_WARP) {
    if (lane == 0) products<DH>(P, sh, smem_u32(smem), 0, n_tiles, 0);
    __syncwarp();
  } else {
    // (rows of a tile that is not full begin at another quarter of the lanes in every block: its warps are of another scheduler)
    const int quarter = warp & 3, half = (warp - FIRST_SUM_WARP) >> 2, row = ((quarter + blockIdx.x) & 3) * 32 + lane;
    const RowsToken tok = rows_token(P.R, it, row0 + min(row, n_rows - 1), hk);
    const int p_last = min(tok.p, end_all - 1);
    const bool bent = P.R.cap_log2 > 0.f || P.R.slopes || !(tok.sc > 0.f), idle = row - lane >= n_rows;
    const float f = bent ? 1.f : tok.sc;  // what brings the numbers below to base-2 units
    const uint64_t f2 = pack2(f, f);
    if (half == 0) {  // (lane i of a quarter has row `row`)
      load_rows<DH>(smem_u32(smem), quarter * 32, P.R.q, q_row(P.R, it, hk, row0 + row), lane);
      loaded(bar_stays(sh));
    }
    float m = ROWS_NEG_BIG, l = 0.f;
    for (int t = 0; t < n_tiles; ++t) {
      if (!await_scores(P, sh, t, lane)) break;
      const int s = t % SLOTS;
      const bool masked = sh.masked[s];
#pragma unroll 1
      for (int c0 = half * (PASS / 2); c0 < (half + 1) * (PASS / 2) && !idle; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(scores_at(sh, t) + ((uint32_t)(quarter * 32) << 16) + c0, v);
        tmem_ld_wait();
        if (F8) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 k = *reinterpret_cast<const float4*>(&sh.factor[s][c0 + c]);
            v[c] = __float_as_uint(__uint_as_float(v[c]) * k.x);
            v[c + 1] = __float_as_uint(__uint_as_float(v[c + 1]) * k.y);
            v[c + 2] = __float_as_uint(__uint_as_float(v[c + 2]) * k.z);
            v[c + 3] = __float_as_uint(__uint_as_float(v[c + 3]) * k.w);
          }
        }
        const int place = key0 + t * PASS + c0;
        if (bent) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            float x = __uint_as_float(v[c]) * tok.sc;
            if (P.R.cap_log2 > 0.f) x = P.R.cap_log2 * weights_tanh(x);
            v[c] = __float_as_uint(x - tok.slope * (float)(tok.p - place - c));
          }
        }
        if (masked) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (place + c < tok.lo || place + c > p_last) v[c] = __float_as_uint(-INFINITY);
        }
        float top = m, top1 = ROWS_NEG_BIG;
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          top = max3(top, __uint_as_float(v[c]), __uint_as_float(v[c + 1]));
          top1 = max3(top1, __uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
        }
        top = fmaxf(top, top1);
        l *= rows_exp2((m - top) * f);
        m = top;
        const uint64_t at2 = pack2(-top * f, -top * f);
        uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 32; c += 2)
          sum[c >> 1 & 1] = add2(sum[c >> 1 & 1], exp2_unit2(fma2((uint64_t)v[c] | (uint64_t)v[c + 1] << 32, f2, at2)));
        sum[0] = add2(sum[0], sum[1]);
        l += low2(sum[0]) + high2(sum[0]);
      }
      release_scores(sh, t, lane);
    }
    m = l == 0.f ? ROWS_NEG_BIG : m * f;
    // the halves' sums of a row, then (below) the blocks' of the cluster
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
  if (P.splits > 1) cluster.sync();
  const int share = (TILE + P.splits - 1) / P.splits, row = split * share + tid;
  if (tid < share && row < n_rows) {
    float m = sh.m[row], l = sh.l[row];
    if (P.splits > 1) {
      float mq[MAX_SPLITS], lq[MAX_SPLITS];
#pragma unroll
      for (int q = 0; q < MAX_SPLITS; ++q) {
        mq[q] = q < P.splits ? *cluster.map_shared_rank(&sh.m[row], q) : ROWS_NEG_BIG;
        lq[q] = q < P.splits ? *cluster.map_shared_rank(&sh.l[row], q) : 0.f;
      }
#pragma unroll
      for (int q = 0; q < MAX_SPLITS; ++q) m = fmaxf(m, mq[q]);
      l = 0.f;
#pragma unroll
      for (int q = 0; q < MAX_SPLITS; ++q) l += lq[q] * rows_exp2(mq[q] - m);
    }
    const RowsToken tok = rows_token(P.R, it, row0 + row, hk);
    if (P.R.sink) l += exp2f(P.R.sink[tok.head] * LOG2E - m);  // (a row that sees nothing: infinite)
    T.row_info[(size_t)tok.n * P.R.Hq + tok.head] = make_float2(tok.sc, l == 0.f ? -INFINITY : -(m + log2f(l)));
  }
  if (P.splits > 1) cluster.sync();
}

// ----------------------------------------------------------------------------------------- keys: their weights
// A block has T.key_tiles tiles of keys one after the other (more than one only without other blocks to share them with, and with at
// most 32 tiles of rows): the row tiles of the next one are on their way while this one's weights are added up.
template <int DH, bool F8>
__global__ void __launch_bounds__(NTHREADS, 2) attention_weights_keys_kernel(const TcParams T) {
  JLX_TL(TL_ATTN_PREFILL);
  const WeightsParams& P = T.P;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(16) Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // (the first keys are seen by the most rows, and come first)
  const int split = blockIdx.x % P.splits, pair = blockIdx.x / P.splits, r = pair / P.R.Hkv, hk = pair - r * P.R.Hkv;
  const int keys0 = blockIdx.y * T.key_tiles * TILE, keys1 = min(keys0 + T.key_tiles * TILE, P.W.width);
  const size_t out_row = pair;
  const int G = P.R.Hq / P.R.Hkv;
  RowsItem it;
  auto leave = [&]() { weights_copy(P, out_row, keys0, keys1, split * NTHREADS + tid, P.splits * NTHREADS); };
  if (!weights_request(P, r, it)) { leave(); return; }
  const int rows = it.cnt * G, tiles = (rows + PASS - 1) / PASS, limit = min(P.W.max_kv, P.W.width);
  const int4* spans = T.spans + (size_t)r * T.q_tiles;
  // row tiles that see some of a tile's keys , every splits-th of them this block's
  auto sees = [](const int4& s, int key0, int width) { return s.y >= key0 && s.z < key0 + width; };
  auto span_of = [&](int t) { return t < tiles ? spans[t] : make_int4(0, -1, 0, 0); };
  int any = 0, bad = 0, end_all = 0, first = 0x7fffffff;
  for (int t = tid; t < tiles; t += NTHREADS) {
    const int4 s = span_of(t);
    bad |= s.y >= limit;
    any |= sees(s, keys0, keys1 - keys0);
    end_all = max(end_all, s.y + 1);
    first = min(first, s.z);
  }
  const int4 mine0 = span_of(split + lane * P.splits);  // of the first 32 of this block's
  bad = __syncthreads_or(bad);
  any = __syncthreads_or(any);
  if (bad || !any) {  // (the whole cluster)
    if (bad && tid == 0) atomicOr(P.R.status, JLX_STATUS_BAD_PAGE);
    leave();
    return;
  }
  open_block(sh, warp);
  end_all = __reduce_max_sync(0xffffffffu, end_all);
  first = __reduce_min_sync(0xffffffffu, first);
  if (lane == 0) {
    atomicMax(&sh.span[1], end_all);
    atomicMin(&sh.span[2], first);
  }
  __syncthreads();
  end_all = min(sh.span[1], rows_capacity(P.R));
  first = sh.span[2];
  const int* table = P.R.block_table + (size_t)r * P.R.bt_stride;
  const int step = 32 * P.splits;
  // this block's row tiles that see a tile of keys; the whole warp asks
  auto count = [&](int key0) {
    int n = __popc(__ballot_sync(0xffffffffu, sees(mine0, key0, TILE)));
    for (int base = split + step; base < tiles; base += step) n += __popc(__ballot_sync(0xffffffffu, sees(span_of(base + lane * P.splits), key0, TILE)));
    return n;
  };

  if (warp < FIRST_SUM_WARP) {
    const int part = (warp >> 1) * 64;
    int t = 0;
    bool ok = true;
    for (int key0 = keys0; key0 < keys1 && ok; key0 += TILE)
      for (int base = split; base < tiles && ok; base += step) {
        // a lane looks at one of 32 row tiles
        const int4 span = base == split ? mine0 : span_of(base + lane * P.splits);
        uint32_t todo = __ballot_sync(0xffffffffu, sees(span, key0, TILE));
        const uint32_t masked = __ballot_sync(0xffffffffu, span.x < min(key0 + TILE, end_all) - 1 || span.w > key0);
        for (; todo; todo &= todo - 1, ++t) {
          if ((t ^ warp) & 1) continue;
          const int i = __ffs(todo) - 1, row0 = (base + i * P.splits) * PASS + part, s = t % STAGES;
          int flat[2], p[2] = {-1, -1}, lo[2] = {0x7fffffff, 0x7fffffff};
          float2 info[2] = {make_float2(0.f, -INFINITY), make_float2(0.f, -INFINITY)};
          float slope[2] = {0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = row0 + h * 32 + lane;
            flat[h] = q_row(P.R, it, hk, row);
            if (flat[h] < 0) continue;
            info[h] = T.row_info[flat[h]];
            p[h] = P.R.positions[it.n0 + row / G];
            if (P.R.slopes) slope[h] = P.R.slopes[hk * G + row % G] * LOG2E;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (flat[h] >= 0) lo[h] = rows_first_key(P.R, p[h]);
          ok = await_stage(P, sh, t, lane);
          if (!ok) break;
          const int slot = t % SLOTS;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = part + h * 32 + lane;
            load_rows<DH>(smem_u32(smem + (1 + s) * TcTile<DH>::BYTES), part + h * 32, P.R.q, flat[h], lane);
            sh.factor[slot][at] = info[h].x;
            sh.lse[slot][at] = info[h].y;
            sh.slope[slot][at] = slope[h];
            sh.pos[slot][at] = p[h];
            sh.lo[slot][at] = lo[h];
          }
          if (tid < 64) {
            sh.masked[slot] = masked >> i & 1;
            sh.columns[slot] = min(rows - row0, PASS);
          }
          mbar_arrive(bar_beside(sh, t));
          loaded(bar_full(sh, s));
        }
      }
  } else if (warp == MMA_WARP) {
    int t = 0, stays = 0;
    for (int key0 = keys0; key0 < keys1; key0 += TILE) {
      const int n = count(key0);
      if (n == 0) continue;
      if (lane == 0) products<DH>(P, sh, smem_u32(smem), t, t + n, stays);
      __syncwarp();
      t += n;
      ++stays;
    }
  } else {
    const int quarter = warp & 3, half = (warp - FIRST_SUM_WARP) >> 2, row = quarter * 32 + lane;
    const bool bent = P.R.cap_log2 > 0.f || P.R.slopes, own_factor = P.R.attn_scale != 0.f, narrow = P.R.chunk > 0 || P.R.window > 0;
    const float* add = P.W.add ? P.W.add + out_row * P.W.width : nullptr;
    float* out = P.W.out + out_row * P.W.width;
    auto key_at = [&](int place) { return place >= first && place < min(end_all, keys1) ? rows_cache_row(P.R, table, hk, place) : -1; };
    int t0 = 0, next = key_at(keys0 + row);
    for (int key0 = keys0; key0 < keys1; key0 += TILE) {
      const int place = key0 + row, n = count(key0), flat = next;
      float* other = (key0 - keys0) / TILE & 1 ? sh.m : sh.l;  // the other half's sums, one tile's beside the next one's
      const bool writes = P.splits == 1 && half == 0 && place < keys1;
      const float before = writes && add ? add[place] : 0.f;
      float ks = 1.f;
      if (n > 0) {
        if (F8) ks = flat >= 0 ? fp8_scale(P.R.scales[flat]) : 0.f;
        if (half == 0) {
          load_part<DH, F8>(smem, quarter * 32, P.R.pages, flat, lane);
          loaded(bar_stays(sh));
        }
      }
      next = key_at(place + TILE);  // (asked for a tile ahead: the table and the key would be a chain)
      const uint64_t ks2 = own_factor ? pack2(ks, ks) : pack2(ks * P.R.scale_log2, ks * P.R.scale_log2);
      uint64_t sum[2] = {0ull, 0ull};
      for (int t = t0; t < t0 + n; ++t) {
        if (!await_scores(P, sh, t, lane)) break;
        const int s = t % SLOTS;
        const bool masked = sh.masked[s];
        const int columns = sh.columns[s];  // (what lies behind them is zeros times the key, and not looked at)
#pragma unroll 1
        for (int c0 = half * (PASS / 2); c0 < min((half + 1) * (PASS / 2), columns); c0 += 32) {
          uint32_t v[32];
          tmem_ld32(scores_at(sh, t) + ((uint32_t)(quarter * 32) << 16) + c0, v);
          tmem_ld_wait();
          if (bent) {
            float more = 0.f;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const int p = sh.pos[s][c0 + c];
              float x = __uint_as_float(v[c]);
              if (F8) x *= ks;
              x *= sh.factor[s][c0 + c];
              if (P.R.cap_log2 > 0.f) x = P.R.cap_log2 * weights_tanh(x);
              x = x - sh.slope[s][c0 + c] * (float)(p - place) + sh.lse[s][c0 + c];
              more += place >= sh.lo[s][c0 + c] && place <= p ? rows_exp2(x) : 0.f;
            }
            sum[0] = add2(sum[0], pack2(more, 0.f));
          } else if (masked || c0 + 32 > columns) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 f = *reinterpret_cast<const float4*>(&sh.factor[s][c0 + c]), lse = *reinterpret_cast<const float4*>(&sh.lse[s][c0 + c]);
              const int4 p = *reinterpret_cast<const int4*>(&sh.pos[s][c0 + c]);
              const int4 lo = narrow ? *reinterpret_cast<const int4*>(&sh.lo[s][c0 + c]) : make_int4(0, 0, 0, 0);
              const float x = fmaf(__uint_as_float(v[c]) * ks, f.x, lse.x), y = fmaf(__uint_as_float(v[c + 1]) * ks, f.y, lse.y);
              const float z = fmaf(__uint_as_float(v[c + 2]) * ks, f.z, lse.z), w = fmaf(__uint_as_float(v[c + 3]) * ks, f.w, lse.w);
              sum[0] = add2(sum[0], exp2_unit2(pack2(place <= p.x && place >= lo.x ? x : -INFINITY, place <= p.y && place >= lo.y ? y : -INFINITY)));
              sum[1] = add2(sum[1], exp2_unit2(pack2(place <= p.z && place >= lo.z ? z : -INFINITY, place <= p.w && place >= lo.w ? w : -INFINITY)));
            }
          } else {
            // (a column's numbers cost every warp a trip through shared memory: the factor only where rows have their own)
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const ulonglong2 lse = *reinterpret_cast<const ulonglong2*>(&sh.lse[s][c0 + c]);
              uint64_t x = (uint64_t)v[c] | (uint64_t)v[c + 1] << 32, y = (uint64_t)v[c + 2] | (uint64_t)v[c + 3] << 32;
              if (own_factor) {
                const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(&sh.factor[s][c0 + c]);
                if (F8) {
                  x = mul2(x, ks2);
                  y = mul2(y, ks2);
                }
                x = fma2(x, f.x, lse.x);
                y = fma2(y, f.y, lse.y);
              } else {
                x = fma2(x, ks2, lse.x);
                y = fma2(y, ks2, lse.y);
              }
              sum[0] = add2(sum[0], exp2_unit2(x));
              sum[1] = add2(sum[1], exp2_unit2(y));
            }
          }
        }
        release_scores(sh, t, lane);
      }
      t0 += n;
      sum[0] = add2(sum[0], sum[1]);
      const float w = low2(sum[0]) + high2(sum[0]);
      if (half == 1) other[row] = w;
      asm volatile("bar.sync 1, %0;" ::"n"(32 * SUM_WARPS) : "memory");  // (and every product with the tile that stayed is done)
      const float both = half == 0 ? w + other[row] : 0.f;
      if (writes) out[place] = before + (place < end_all ? both : 0.f);
      if (P.splits > 1 && half == 0) sh.l[row] = both;  // (its only tile)
    }
  }
  close_block(sh, warp);
  if (P.splits == 1) return;
  cluster.sync();
  const int share = (TILE + P.splits - 1) / P.splits, row = split * share + tid, place = keys0 + row;
  if (tid < share && row < TILE && place < keys1) {
    float w[MAX_SPLITS];
#pragma unroll
    for (int q = 0; q < MAX_SPLITS; ++q) w[q] = q < P.splits ? *cluster.map_shared_rank(&sh.l[row], q) : 0.f;
#pragma unroll
    for (int q = 1; q < MAX_SPLITS; ++q) w[0] += w[q];
    const size_t at = out_row * P.W.width + place;
    P.W.out[at] = (P.W.add ? P.W.add[at] : 0.f) + (place < end_all ? w[0] : 0.f);
  }
  cluster.sync();
}

// out = add at the places from `from` on, which no request's keys reach.  (Within the launch above every 128 of them took a block of their
// own with nothing to do: 128 rows over 4096 keys into 131,072 places 99 us for 23.)
#define COPY_PLACES 4096
__global__ void __launch_bounds__(256) attention_weights_behind_kernel(const WeightsParams P, int from) {
  JLX_TL(TL_ATTN_PREFILL);
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int first = from + blockIdx.y * COPY_PLACES;
  weights_copy(P, blockIdx.x, first, min(first + COPY_PLACES, P.W.width), threadIdx.x, 256);
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
  // tiles of the keys that requests may have; what lies behind them is copied, unless it is there
  const int block = T.key_tiles * TILE, keys = T.P.W.max_kv < T.P.W.width ? T.P.W.max_kv : T.P.W.width, key_blocks = (keys + block - 1) / block;
  const int behind = T.P.W.add == T.P.W.out ? 0 : T.P.W.width - key_blocks * block;
  const unsigned pairs = (unsigned)(T.P.R.n_requests * T.P.R.Hkv);
  T.P.splits = rows_splits;
  if (int e = launch_tc(attention_weights_rows_kernel<DH, F8>, TcTile<DH>::SMEM, dim3(pairs * (unsigned)rows_splits, (unsigned)T.q_tiles), rows_splits, T, stream)) return e;
  T.P.splits = keys_splits;
  if (int e = launch_tc(attention_weights_keys_kernel<DH, F8>, TcTile<DH>::SMEM, dim3(pairs * (unsigned)keys_splits, (unsigned)key_blocks), keys_splits, T, stream)) return e;
  if (behind > 0) JLX_CUDA(jlx_launch_pdl(attention_weights_behind_kernel, dim3(pairs, (unsigned)((behind + COPY_PLACES - 1) / COPY_PLACES)), dim3(256), 0, stream, T.P, key_blocks * block));
  return 0;
}

// Scratch: float2 [N * Hq], then (on 16 bytes) int4 [R * ceil(max_count * G / 128)].
JLX_API int jlx_attention_weights_tc(const RowsArgs* rows_args, const WeightsArgs* args, int rows_splits, int keys_splits, int key_tiles, void* stream_) {
  TcParams T;
  T.key_tiles = key_tiles;
  if (int e = rows_params(*rows_args, T.P.R)) return e;
  T.P.W = *args;
  T.P.buf_keys = T.P.rows = 0;
  T.P.page_shift = -1;
  const RowsParams& R = T.P.R;
  JLX_REQUIRE(rows_splits >= 1 && rows_splits <= MAX_SPLITS && keys_splits >= 1 && keys_splits <= MAX_SPLITS, "attention_weights: %d and %d blocks share tiles", rows_splits, keys_splits);
  JLX_REQUIRE((long long)R.n_requests * R.Hkv * MAX_SPLITS < (1ll << 31), "attention_weights: %d requests of %d KV heads are too many for a launch", R.n_requests, R.Hkv);
  JLX_REQUIRE(((long long)R.max_count * (R.Hq / R.Hkv) + TILE - 1) / TILE <= 65535 && ((long long)T.P.W.width + TILE - 1) / TILE <= 65535, "attention_weights: %d tokens or %d places of a request are too many for a launch", R.max_count, T.P.W.width);
  JLX_REQUIRE(key_tiles == 1 || (key_tiles > 1 && keys_splits == 1 && (long long)R.max_count * (R.Hq / R.Hkv) <= 32 * PASS), "attention_weights: %d tiles of keys a block", key_tiles);
  JLX_REQUIRE((long long)R.N * R.Hq < (1ll << 31), "attention_weights: %d rows of %d heads are too many", R.N, R.Hq);
  JLX_REQUIRE(T.P.W.scratch && ((uintptr_t)T.P.W.scratch & 15) == 0, "attention_weights: scratch is needed, on 16 bytes");
  T.row_info = reinterpret_cast<float2*>(T.P.W.scratch);
  T.spans = reinterpret_cast<int4*>(T.P.W.scratch + ((size_t)R.N * R.Hq * 2 + 3) / 4 * 4);
  T.q_tiles = (int)(((long long)R.max_count * (R.Hq / R.Hkv) + TILE - 1) / TILE);
  cudaStream_t stream = (cudaStream_t)stream_;
  if (rows_args->dh == 128) return R.scales ? launch_both<128, true>(T, rows_splits, keys_splits, stream) : launch_both<128, false>(T, rows_splits, keys_splits, stream);
  return R.scales ? launch_both<64, true>(T, rows_splits, keys_splits, stream) : launch_both<64, false>(T, rows_splits, keys_splits, stream);
}
