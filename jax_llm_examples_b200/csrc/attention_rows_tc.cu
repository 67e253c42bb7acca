// Grouped-query attention of many query rows of an item over the paged cache on the 5th-generation tensor cores (tcgen05), head
// sizes 64 and 128: drafted trees and prompt portions, over a cache in bfloat16 or in 8 bits (attention_rows.cuh has mask and formula).
//
// A block takes 128 or 256 query rows of one item and KV head, (token, head of the group) pairs token by token, so that every key
// is read once for that many rows, and one range of their keys in tiles of 128.  Two groups of eight softmax warps work a product
// apart, each with 128 columns of tensor memory for its scores and as many for its output: with more than 128 rows each group has
// 128 of them and every tile, else both have the same rows, one the even tiles and the other the odd ones, and their sums and
// outputs are joined at the end.  Per group and tile:
//   S = Q K^T    tcgen05.mma from shared memory into tensor memory
//   P            PARTS threads per query row read their parts of its scores, keep the reference of the exponents and the sum
//                in 32-bit, and write the weights as 16-bit numbers over the first half of S
//   O += P V     tcgen05.mma with P in tensor memory and V from shared memory as an MN-major operand
// Products run in the order of their issue: a group's next score product, which overwrites S and P, is issued after its O += P V.
// Warp 0 issues the keys' copies, warp 1 the products, warp 2 the values' copies, warp 3 fetches scales, the last four warps
// prepare values (below).
//
// What bounds it: a group's turn of about 4,500 cycles, of which 1,250 are the exponentials (1,024 at the unit's rate), 1,000 the
// rest of the softmax, 600 (8 bits) the keys' scales and 1,800 the wait for the two products: their 16 instructions are accepted
// one in 95 cycles from one thread, 1,520 a tile.  So 2,250 a tile of 128 by 128, where exponentials and products would take
// 1,024 each, side by side.  Measured (B200): 2,048 tokens after 1,500, 40 heads on 8 of 128, 8 bits: 185 us, 571 TFLOP/s, 34 %
// of the bfloat16 peak; trees of 32 tokens on 8 requests of up to 8,192 keys, bfloat16: 94 us, 347 TFLOP/s; of 64 tokens on 16
// requests of up to 12,000, 32 heads, 8 bits: 275 us, 551 TFLOP/s.
// Tried and slower: one group of sixteen warps on 128 rows with two buffers of scores (227, 114 and 325 us); then one block per
// multiprocessor that takes an equal share of all tiles (247, 112 and 293: its join and the change from piece to piece cost what
// the shares gained); a warp for each group's products beside one for all copies (228, 108 and 357).
//
// 8 bits: the keys' codes are an operand as they lie in the cache.  Queries are two: each entry (its row's largest brought to
// 2^7 .. 2^8 by a power of two) as e4m3, and what is left of it as e5m2; the remainder of eight bits after the nearest four is
// a whole number up to 8 of the entry's last unit, which e5m2 holds (three bits), so both products add up in one accumulator to
// that of the bfloat16 query.  That is exact for entries from 2^-6 on, 2^-13 of the row's largest; below, e4m3's steps no longer
// shrink, the remainder has up to eight bits, and an entry is off by up to 2^-14: 2^-21 of the row's largest.  The e4m3 product
// has twice the rate: two cost what one of bfloat16 does, and no key is converted.  A key's power of two multiplies its column
// of scores.  The values become bfloat16, code times scale, which it holds exactly, once per tile and block: a code's seven bits
// are a bfloat16 number's exponent and mantissa but for a factor of 2^120, which the multiplication with the scale takes along.
// (Tried and slower: values' scales kept out of the operand, as exponents added to the keys' scores and taken out of the sum:
// the three numbers a key that every softmax thread then reads take 1,500 cycles of a tile's shared-memory bandwidth.)
// Weights are rounded to bfloat16 for the product with the values (2^-8 of each at most); sums are 32-bit.  Over 8 bits, too: one
// product takes one type, and the values' scales need bfloat16's exponents; float16 weights would ask for the scales in the scores
// (see above).  Against 64 bits the output is off by 0.0016 to 0.0019 of its norm, of which its own rounding makes 0.0014.
//
// Masks: only tiles that some row does not see wholly look at them.  In such a tile a value that is not finite is taken out
// (a product would spread 0 * infinity over all rows) and added to the rows that do see it at the end; of rows of the cache
// outside the range finite numbers reach a product at most, with weights of zero (8 bits: zeros).
//
// Every wait on a barrier is bounded; after a timeout the block raises JLX_STATUS_WAIT_TIMEOUT, waits (bounded) for its own
// copies, frees its tensor memory and returns.
#include "attention_rows.cuh"
#include "mbarrier.cuh"

#define BQ 128           // query rows of a group
#define BROWS (2 * BQ)   // of a block
#define BKV 128          // keys per tile
#define PARTS 2          // softmax threads per query row and group: each takes BKV / PARTS of a tile's keys
#define CP (BKV / PARTS)
#define SOFTMAX0 4       // first softmax warp: the first group's 4 * PARTS, then the second's
#define AUX0 (SOFTMAX0 + 8 * PARTS)  // first of the four warps that prepare values
#define AUX 128
#define NTHREADS (AUX0 * 32 + AUX)
// Registers: the block is launched with 80 a thread (the most that 768 threads may have); the four softmax warpgroups take more,
// the two others give it up: 4 * 96 + 2 * 48 = 6 * 80.
#define REGS_SOFTMAX 96
#define REGS_OTHERS 48
#define GROWTH 16.0f     // how far a row's maximum may outgrow its reference (in powers of two) before O is rescaled
#define SLOTS 4          // tiles whose scales are kept

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
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
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_f16_a_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two float32 operations per instruction (IEEE, as their one-value forms).
__device__ __forceinline__ uint64_t pack2(float a, float b) { return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32); }
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

// Shared-memory matrix descriptors for tiles whose rows are 128 (or 64) bytes with the swizzle of that many, 8-row groups side
// by side.  K-major: a row runs along K.  MN-major: along the operand's N direction, rows are K steps; blocks of 64 numbers
// along N are `lbo_bytes` apart.
template <int ROW> __device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(8 * ROW >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)(ROW == 128 ? 2 : 4) << 61);
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr, uint32_t lbo_bytes) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(lbo_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptors: float32 accumulator, M = 128, N = n; operand formats a, b (kind::f16: 0 float16, 1 bfloat16;
// kind::f8f6f4: 0 e4m3, 1 e5m2); A K-major, B K- or MN-major.
__host__ __device__ constexpr uint32_t make_idesc(uint32_t a, uint32_t b, uint32_t b_mn_major, uint32_t n) {
  return (1u << 4) | (a << 7) | (b << 10) | (b_mn_major << 16) | ((n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// Byte offset of 16-byte chunk c of row r in a swizzled tile of rows of ROW bytes.
template <int ROW> __device__ __forceinline__ uint32_t swizzled(int r, int c) {
  return ROW == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

#define HALF_BYTES (128 * 128)  // 128 rows of 128 bytes
template <int DH, bool F8> struct TcTile {
  static constexpr int ROW = F8 ? DH : 128;                  // bytes of a row of queries or keys as the score product sees it
  static constexpr int HALVES = F8 ? 1 : DH / 64;            // bfloat16: entries 0-63, 64-127 lie in tiles of their own
  static constexpr int PART = 128 * ROW;                     // such a tile
  static constexpr int Q = F8 ? 2 * PART : HALVES * PART;    // a group's queries (8 bits: first parts, what is left), two of them
  static constexpr int K = HALVES * PART;                    // a tile of keys
  static constexpr int KS = DH == 64 ? 4 : F8 ? 3 : 2;       // tiles of keys in flight
  static constexpr int V = DH / 64 * HALF_BYTES;             // a tile of values as an operand, two of them
  static constexpr int VS = F8 && DH == 64 ? 3 : 2;          // tiles of values in flight (8 bits: of their codes)
  static constexpr int RAW = F8 ? PART : 0;                  // a tile of values' codes
  static constexpr int SCALES = F8 ? SLOTS * BKV * 5 : 0;    // [SLOTS] the keys' scales; [SLOTS] the values' bytes
  static constexpr int SMEM = 2 * Q + KS * K + 2 * V + VS * RAW + SCALES + 1024;
  static constexpr int STEPS = F8 ? 2 * DH / 32 : DH / 16;   // score products of a tile
  static constexpr int OC = DH / PARTS;                      // columns of its group's O that a softmax thread rescales
  static constexpr int OE = DH / (2 * PARTS);                // columns of the sum of both that it stores
};

template <int DH, bool F8>
__global__ void __launch_bounds__(NTHREADS, 1) attention_rows_tc_kernel(const __grid_constant__ CUtensorMap map, const RowsParams P, int box_rows, int row_block, int row_tiles) {
  JLX_TL(TL_ATTN_PREFILL);
  using T = TcTile<DH, F8>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t *q_p = smem, *k_p = q_p + 2 * T::Q, *v_p = k_p + T::KS * T::K, *raw_p = v_p + 2 * T::V;
  float* scales_p = reinterpret_cast<float*>(raw_p + T::VS * T::RAW);
  uint8_t* bytes_p = reinterpret_cast<uint8_t*>(scales_p + SLOTS * BKV);
  // barriers (each use flips a phase bit; t = a tile's number)
  enum { B_QREADY = 0,    // Q is in shared memory
         B_KFULL = 1,     // [KS] K of tile t has landed                  stage t % KS, phase t / KS
         B_KEMPTY = 5,    // [KS] the score product of tile t is done
         B_VFULL = 9,     // [VS] V of tile t (or its codes) has landed   stage t % VS, phase t / VS
         B_RAWEMPTY = 12, // [VS] the codes have been read
         B_VREADY = 15,   // [2] V of tile t is an operand
         B_VEMPTY = 17,   // [2] the product with P of tile t is done
         B_SFULL = 19,    // [2] S of tile t is complete
         B_PREADY = 21,   // [2] P of tile t is in tensor memory, its group's O rescaled
         B_ODONE = 23,    // both O are complete (once)
         B_MEET = 24,     // [2][4] the threads of a group and quarter of the rows have met
         B_END = 32,      // [4] the threads of a quarter of the rows, of both groups (once)
         B_SCALES = 36,   // [SLOTS] the scales of tile t are there        slot t % SLOTS, phase t / SLOTS
         B_SCFREE = 40,   // [SLOTS] they have been read
         N_BARS = 44 };
  __shared__ __align__(8) uint64_t bars[N_BARS];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed, any_bad, span[4];
  __shared__ float xmax[2][2][PARTS][BQ];  // [meeting parity][group][part][row]: what the threads of a row exchange
  __shared__ float ends[2][BQ];            // [group][row]: the references at the end
  __shared__ int4 toks[BROWS];          // the rows' tokens: index, position, first key, slope
  __shared__ int item_s[4];
  __shared__ float q_exp[BROWS];           // 8 bits: the power of two that a query row was divided by
  pdl_launch_dependents_if_small();
  pdl_wait();
  const uint32_t bar0 = smem_u32(&bars[0]);
  auto BAR = [bar0](int i) { return bar0 + 8u * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // an item's ranges, heads and row tiles side by side, then the next item: the items' order (the longest first, say) is the blocks'
  const int unit = blockIdx.x / P.splits, split = blockIdx.x - unit * P.splits, item_i = unit / (P.Hkv * row_tiles);
  const int hk = unit % (P.Hkv * row_tiles) / row_tiles, row0 = unit % row_tiles * row_block;
  RowsItem it;
  if (!rows_tokens(P, item_i, it)) return;
  const int G = P.Hq / P.Hkv, n_rows = min(it.cnt * G - row0, row_block);
  if (n_rows <= 0) return;
  const bool by_rows = n_rows > BQ;
  // asked for now, needed after the request's description: the tokens' positions, and the queries (four neighbouring threads of
  // the softmax warps bring a row into shared memory)
  const bool softmax = warp >= SOFTMAX0 && warp < AUX0;
  const int q_row = (threadIdx.x - SOFTMAX0 * 32) >> 2, q_part = threadIdx.x & 3;
  int p_mine = 0;
  uint4 q_mine[2][DH / 32];
  if (threadIdx.x < BROWS) p_mine = P.positions[it.n0 + (row0 + min((int)threadIdx.x, n_rows - 1)) / G];
  if (softmax) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int row = row0 + min(g * BQ + q_row, n_rows - 1), t = row / G, head = hk * G + row - t * G;
      const uint4* src = reinterpret_cast<const uint4*>(P.q + ((size_t)(it.n0 + t) * P.Hq + head) * DH + q_part * (DH / 4));
      if (g == 0 || by_rows)
#pragma unroll
        for (int u = 0; u < DH / 32; ++u) q_mine[g][u] = src[u];
    }
  }
  if (!rows_request(P, it)) return;

  if (threadIdx.x == 0) {
    for (int i = 0; i < N_BARS; ++i) {
      int count = 1;  // a transaction count or a tcgen05.commit, but:
      if (i == B_QREADY) count = 256 * PARTS;
      if (i >= B_PREADY && i < B_PREADY + 2) count = 128 * PARTS;
      if ((i >= B_RAWEMPTY && i < B_RAWEMPTY + 3) || (i >= B_VREADY && i < B_VREADY + 2)) count = AUX;
      if (i >= B_MEET && i < B_MEET + 8) count = 32 * PARTS;
      if (i >= B_END && i < B_END + 4) count = 64 * PARTS;
      if (i >= B_SCALES && i < B_SCALES + SLOTS) count = 32;
      mbar_init(BAR(i), count);
    }
    failed = any_bad = 0;
    item_s[0] = it.r;
    item_s[1] = it.base;
    item_s[2] = it.drafted;
    item_s[3] = it.n0;
    span[0] = span[2] = 0x7fffffff;
    span[1] = span[3] = (int)0x80000000;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (threadIdx.x < BROWS) {
    const int lo = rows_first_key(P, p_mine);
    const int a = __reduce_min_sync(0xffffffffu, lo), b = __reduce_max_sync(0xffffffffu, lo);
    const int c = __reduce_min_sync(0xffffffffu, p_mine), d = __reduce_max_sync(0xffffffffu, p_mine);
    if (lane == 0) {
      atomicMin(&span[0], a);
      atomicMax(&span[1], b);
      atomicMin(&span[2], c);
      atomicMax(&span[3], d);
    }
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), 512);  // S of even and odd tiles, O of even and odd tiles: 128 columns each
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot, tm_o = tmem + 256;
  // the item's keys and this block's equal part of their tiles
  const int first = P.cu_q ? min(span[0], it.base) : span[0], end_all = rows_end(P, it, span[3]);
  const int full_lo = span[1], full_hi = P.cu_q ? it.base : span[2] + 1;  // keys in between are seen by every row
  const int start = first / BKV * BKV, per = max((end_all - start + BKV * P.splits - 1) / (BKV * P.splits), 0) * BKV, range0 = start + split * per;
  const int begin = max(first, range0), end = min(end_all, range0 + per);
  const int n_tiles = end > begin ? (end - range0 + BKV - 1) / BKV : 0;
  const int* table = P.block_table + (size_t)it.r * P.bt_stride;
  const int v_off = P.Hkv * P.page_size;
  auto masked_tile = [&](int place0) { return place0 < full_lo || place0 + BKV > min(full_hi, end) || place0 < begin; };

  if (!softmax) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHERS));
  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------------------------ copies: warp 0 keys, warp 2 values
    // Keys are free again after their score product, values after the product with P (or their conversion).  Lane i has the
    // place of box i of a tile; the block table's entry is asked for two tiles before the copy that needs it.
    // (Asking for tiles into L2 ahead of that costs as much of the copy engine's time as a copy: 20 % of the kernel's.)
    const int which = warp >> 1, boxes = BKV / box_rows, stages = which ? T::VS : T::KS, off = which ? v_off : 0;
    auto find_page = [&](int t) {
      const int pi = (range0 + t * BKV + lane * box_rows) / P.page_size;
      return lane < boxes && t < n_tiles && pi < P.bt_stride ? table[pi] : -1;
    };
    int page = find_page(0), page_next = find_page(1), t = 0;
    bool ok = true;
    for (; t < n_tiles; ++t) {
      const int place = range0 + t * BKV + lane * box_rows, st = t % stages;
      const bool there = rows_page_there(P, page);
      if (!there && lane < boxes && place < end && place + box_rows > begin) atomicOr(P.status, JLX_STATUS_BAD_PAGE);
      if (!there) page = P.num_pages;
      const int row = (page * 2 * P.Hkv + hk) * P.page_size + place % P.page_size + off;
      page = page_next;
      page_next = find_page(t + 2);
      if (t >= stages) ok = mbar_wait(BAR((which ? (F8 ? B_RAWEMPTY : B_VEMPTY) : B_KEMPTY) + st), (t / stages - 1) & 1);
      ok = __all_sync(0xffffffffu, ok && !*(volatile int*)&failed);
      if (!ok) break;
      const uint32_t bar = BAR((which ? B_VFULL : B_KFULL) + st);
      uint32_t dst = smem_u32(which ? (F8 ? raw_p + st * T::RAW : v_p + st * T::V) : k_p + st * T::K);
      if (lane == 0) mbar_expect_tx(bar, BKV * DH * (F8 ? 1 : 2));
      for (int i = 0; i < boxes; ++i) {
        const int r = __shfl_sync(0xffffffffu, row, i);
        if (lane == 0) {
          tma_load_2d(dst, &map, 0, r, bar);
          if (T::HALVES == 2) tma_load_2d(dst + HALF_BYTES, &map, 64, r, bar);
        }
        dst += box_rows * T::ROW;
      }
    }
    if (!ok) {  // let the copies in flight land before the block's shared memory is given up
      for (int i = max(0, t - stages); i < t; ++i) mbar_wait(BAR((which ? B_VFULL : B_KFULL) + i % stages), (i / stages) & 1);
      if (lane == 0) {
        atomicOr(P.status, JLX_STATUS_WAIT_TIMEOUT);
        failed = 1;
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------ products
    if (lane == 0 && n_tiles > 0) {
      bool ok = mbar_wait(BAR(B_QREADY), 0);
      // Step u is group u & 1's: of tile u / 2 if the groups share the tiles, of tile u if they take them in turn.
      const int steps = by_rows ? 2 * n_tiles : n_tiles;
      auto issue_qk = [&](int u) {
        const int g = u & 1, t = by_rows ? u >> 1 : u, sk = t % T::KS;
        if (ok && !(by_rows && g)) {
          ok = mbar_wait(BAR(B_KFULL + sk), (t / T::KS) & 1);
          if (F8 && ok) ok = mbar_wait(BAR(B_SCALES + t % SLOTS), (t / SLOTS) & 1);  // (whoever sees S complete may read the scales)
        }
        if (!ok) return;
        tc_fence_after();
        const uint32_t q_s = smem_u32(q_p) + (by_rows ? g * T::Q : 0), k_s = smem_u32(k_p) + sk * T::K;
#pragma unroll
        for (int kk = 0; kk < T::STEPS; ++kk) {
          if (F8) {  // first parts, then what is left: steps of 32 entries
            const int part = kk / (DH / 32);
            const uint32_t off = kk % (DH / 32) * 32;
            umma_f8(tmem + g * 128, desc_k_major<T::ROW>(q_s + part * T::PART + off), desc_k_major<T::ROW>(k_s + off), make_idesc(part, 0, 0, BKV), kk != 0);
          } else {   // steps of 16 entries
            const uint32_t off = (kk >> 2) * HALF_BYTES + (kk & 3) * 32;
            umma_f16(tmem + g * 128, desc_k_major<T::ROW>(q_s + off), desc_k_major<T::ROW>(k_s + off), make_idesc(1, 1, 0, BKV), kk != 0);
          }
        }
        umma_commit(BAR(B_SFULL + g));
        if (!by_rows || g) umma_commit(BAR(B_KEMPTY + sk));
      };
      issue_qk(0);
      if (steps > 1) issue_qk(1);
      for (int u = 0; u < steps && ok; ++u) {
        const int g = u & 1, t = by_rows ? u >> 1 : u, st = t & 1;
        if (!(by_rows && g)) ok = mbar_wait(BAR(B_VREADY + st), (t >> 1) & 1);
        if (ok) ok = mbar_wait(BAR(B_PREADY + g), (u >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t v_s = smem_u32(v_p) + st * T::V;
#pragma unroll
        for (int kk = 0; kk < BKV / 16; ++kk)  // P: 16 keys = 8 columns of tensor memory; V: 16 keys = 16 rows of 128 bytes
          umma_f16_a_tmem(tm_o + g * 128, tmem + g * 128 + kk * 8, desc_mn_major(v_s + kk * 16 * 128, HALF_BYTES), make_idesc(1, 1, 1, DH), (u >> 1 | kk) != 0);
        if (!by_rows || g) {
          umma_commit(BAR(B_VEMPTY + st));
          if (F8) umma_commit(BAR(B_SCFREE + t % SLOTS));
        }
        if (u + 2 < steps) issue_qk(u + 2);
      }
      if (ok) umma_commit(BAR(B_ODONE));
      if (!ok) {
        atomicOr(P.status, JLX_STATUS_WAIT_TIMEOUT);
        failed = 1;
      }
    }
  } else if (F8 && warp == 3) {
    // ------------------------------------------------------------------------------ scales: four keys of a tile a lane
    // Their rows' table entries are asked for two tiles ahead, their bytes one.  (As small bulk copies beside the values' their
    // issue took 2,000 cycles a tile.)
    auto find_page = [&](int t) {
      const int pi = (range0 + t * BKV + lane * 4) / P.page_size;
      return t < n_tiles && pi < P.bt_stride ? table[pi] : -1;
    };
    auto fetch = [&](int t, int page, uint32_t& k, uint32_t& v) {
      const int place = range0 + t * BKV + lane * 4;
      k = v = 0u;
      if (!rows_page_there(P, page)) return;
      const uint8_t* src = P.scales + (size_t)((page * 2 * P.Hkv + hk) * P.page_size + place % P.page_size);
      k = *reinterpret_cast<const uint32_t*>(src);
      v = *reinterpret_cast<const uint32_t*>(src + v_off);
    };
    uint32_t k = 0, v = 0, k_next = 0, v_next = 0;
    if (n_tiles > 0) fetch(0, find_page(0), k, v);
    int page = find_page(1), page_next = 0;
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      page_next = find_page(t + 2);
      if (t + 1 < n_tiles) fetch(t + 1, page, k_next, v_next);
      if (t >= SLOTS) ok = __all_sync(0xffffffffu, mbar_wait(BAR(B_SCFREE + t % SLOTS), (t / SLOTS - 1) & 1));
      if (!ok) break;
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = (k >> (8 * i)) & 0xff;
        w[i] = a == FP8_BAD ? 0x7fc00000u : a << 23;
      }
      *reinterpret_cast<uint4*>(scales_p + (t % SLOTS) * BKV + lane * 4) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint32_t*>(bytes_p + (t % SLOTS) * BKV + lane * 4) = v;
      mbar_arrive(BAR(B_SCALES + t % SLOTS));
      k = k_next;
      v = v_next;
      page = page_next;
    }
    if (!ok && lane == 0) {
      atomicOr(P.status, JLX_STATUS_WAIT_TIMEOUT);
      failed = 1;
    }
  } else if (warp >= AUX0) {
    // ------------------------------------------------------------------------------ values as an operand
    const int i0 = threadIdx.x - AUX0 * 32;  // the key of every tile
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      const int st = t & 1, sr = t % T::VS, place0 = range0 + t * BKV;
      ok = mbar_wait(BAR(B_VFULL + sr), (t / T::VS) & 1);
      if (F8 && ok) ok = mbar_wait(BAR(B_SCALES + t % SLOTS), (t / SLOTS) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint8_t* v = v_p + st * T::V;
      if (F8) {
        const int bv = bytes_p[(t % SLOTS) * BKV + i0];
        if (t >= 2) ok = __all_sync(0xffffffffu, mbar_wait(BAR(B_VEMPTY + st), ((t >> 1) - 1) & 1));
        if (!ok) break;
        const uint8_t* raw = raw_p + sr * T::RAW;
        // 2^(120 + e) in two factors: together they leave bfloat16's range only where e > 7.  Rows outside the range (their
        // codes may be anything) count for nothing, whatever their byte; a row without codes is NaN for all rows that see it:
        // at once if all do, at the end if some do not.
        const bool in = place0 + i0 >= begin && place0 + i0 < end;
        const int e = in ? min(bv, 254) - 127 : 0;
        uint32_t f = (uint32_t)min(120 + e, 127) + 127, h = (uint32_t)max(e - 7, 0) + 127;
        f = (f << 7) | (f << 23);
        h = (h << 7) | (h << 23);
        if (!in || bv == FP8_BAD) f = 0u;  // (every code is a finite number to the product)
        uint32_t all = 0u;
        if (in && bv == FP8_BAD) {
          if (masked_tile(place0)) *(volatile int*)&any_bad = 1;
          else all = 0x7fc07fc0u;
        }
        const __nv_bfloat162 f2 = *reinterpret_cast<const __nv_bfloat162*>(&f), h2 = *reinterpret_cast<const __nv_bfloat162*>(&h);
        // two codes, each with its sign in the byte above, -> two numbers: the sign and seven bits to their places in one shift
        auto widen = [&](uint32_t x, uint32_t select) {
          uint32_t y;
          asm("prmt.b32 %0, %1, %1, %2;" : "=r"(y) : "r"(x), "r"(select));
          y = (y << 4) & 0x87f087f0u;
          const __nv_bfloat162 z = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&y), f2);
          return *reinterpret_cast<const uint32_t*>(&z);
        };
        auto further = [&](uint32_t x) {
          const __nv_bfloat162 z = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), h2);
          return *reinterpret_cast<const uint32_t*>(&z);
        };
#pragma unroll
        for (int c0 = 0; c0 < DH / 16; c0 += 4) {
          uint4 x[4];  // (fetched together: a store would hold the next fetch back)
#pragma unroll
          for (int c = 0; c < 4; ++c) x[c] = *reinterpret_cast<const uint4*>(raw + swizzled<T::ROW>(i0, c0 + c));
          uint8_t* half = v + (c0 >> 2) * HALF_BYTES;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
            uint32_t o[8];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              o[2 * u] = widen(w[u], 0x9180);
              o[2 * u + 1] = widen(w[u], 0xb3a2);
            }
            if (__builtin_expect(e > 7, 0)) {
#pragma unroll
              for (int u = 0; u < 8; ++u) o[u] = further(o[u]);
            }
            if (__builtin_expect(all != 0u, 0)) {
#pragma unroll
              for (int u = 0; u < 8; ++u) o[u] = all;
            }
            *reinterpret_cast<uint4*>(half + swizzled<128>(i0, c * 2)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(half + swizzled<128>(i0, c * 2 + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        fence_async_proxy();
        mbar_arrive(BAR(B_RAWEMPTY + sr));
      } else if (masked_tile(place0)) {
        bool bad = false;
#pragma unroll 1
        for (int x = i0; x < DH / 64 * BKV * 8; x += AUX) {  // (consecutive threads: chunks of a row)
          const int i = (x >> 3) & (BKV - 1);
          uint4* at = reinterpret_cast<uint4*>(v + (x >> 10) * HALF_BYTES + swizzled<128>(i, x & 7));
          uint32_t w[4] = {at->x, at->y, at->z, at->w};
          bool here = false;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            if ((w[y] & 0x7f80u) == 0x7f80u) { w[y] &= 0xffff0000u; here = true; }
            if ((w[y] & 0x7f800000u) == 0x7f800000u) { w[y] &= 0xffffu; here = true; }
          }
          if (here) {
            *at = make_uint4(w[0], w[1], w[2], w[3]);
            bad = true;
          }
        }
        if (bad) *(volatile int*)&any_bad = 1;
        fence_async_proxy();
      }
      mbar_arrive(BAR(B_VREADY + st));
    }
    if (!ok && lane == 0) {
      atomicOr(P.status, JLX_STATUS_WAIT_TIMEOUT);
      failed = 1;
    }
  }
  } else {
    // ------------------------------------------------------------------------------ queries, softmax, rescale, store
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if (g && !by_rows) break;
      const int i = q_row, part = q_part;
      const uint4 (&x)[DH / 32] = q_mine[g];
      uint8_t* dst = q_p + g * T::Q;
      if (F8) {
        float top = 0.f;
#pragma unroll
        for (int u = 0; u < DH / 32; ++u) {
          const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&x[u]);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float2 f = __bfloat1622float2(h[y]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = max(min((int)(__float_as_uint(top) >> 23) - 127, 120), -110) - 7;
        const float in = fp8_pow2(-e);
        if (part == 0) q_exp[g * BQ + i] = top == INFINITY ? __int_as_float(0x7fc00000) : fp8_pow2(e);  // (no codes for an infinite entry: the scores are NaN)
#pragma unroll
        for (int u = 0; u < DH / 64; ++u) {  // 16 entries: a chunk of each part
          uint32_t hi[4], left[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&x[2 * u + (w >> 1)]) + (w & 1) * 2;
            const float2 f0 = __bfloat1622float2(h[0]), f1 = __bfloat1622float2(h[1]);
            const float a = f0.x * in, b = f0.y * in, c = f1.x * in, d = f1.y * in;
            hi[w] = fp8x4_from_float(a, b, c, d);
            uint32_t back[2];
            fp8x4_to_half(hi[w], back[0], back[1]);
            const float2 g0 = __half22float2(*reinterpret_cast<const __half2*>(&back[0])), g1 = __half22float2(*reinterpret_cast<const __half2*>(&back[1]));
            left[w] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a - g0.x, b - g0.y), __NV_SATFINITE, __NV_E5M2) |
                      (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c - g1.x, d - g1.y), __NV_SATFINITE, __NV_E5M2) << 16;
          }
          *reinterpret_cast<uint4*>(dst + swizzled<T::ROW>(i, part * (DH / 64) + u)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(dst + T::PART + swizzled<T::ROW>(i, part * (DH / 64) + u)) = make_uint4(left[0], left[1], left[2], left[3]);
        }
      } else {
#pragma unroll
        for (int u = 0; u < DH / 32; ++u) {
          const int c = part * (DH / 32) + u;
          *reinterpret_cast<uint4*>(dst + (c >> 3) * HALF_BYTES + swizzled<128>(i, c & 7)) = x[u];
        }
      }
    }
    fence_async_proxy();
    mbar_arrive(BAR(B_QREADY));
    // A warp reaches the tensor-memory lanes [32 * (warp & 3), +32), so PARTS warps of a group share each quarter of the query
    // rows and split a tile's keys among them.  The threads of a row and group meet once per tile to agree on the row's maximum;
    // each keeps the sum of its own part.
    const int quarter = warp & 3, group = (warp - SOFTMAX0) / (4 * PARTS), part = ((warp - SOFTMAX0) >> 2) % PARTS, row = quarter * 32 + lane;
    const int block_row = by_rows ? group * BQ + row : row;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16, o_addr = tm_o + group * 128 + lane_addr;
    const int col0 = part * CP;
    // What only masked tiles and the end need waits in shared memory: 64 scores leave a thread 32 registers for all else, and
    // the first-level cache is too small for spilled ones.
    float sc;
    {
      const RowsToken tok = rows_token(P, it, row0 + min(block_row, n_rows - 1), hk);
      toks[block_row] = make_int4(tok.n, tok.p, tok.lo, __float_as_int(tok.slope));
      sc = tok.sc;
    }
    auto token = [&]() {
      const volatile int* x = reinterpret_cast<const volatile int*>(&toks[block_row]);
      RowsToken tok;
      tok.n = x[0];
      tok.p = x[1];
      tok.lo = x[2];
      tok.slope = __int_as_float(x[3]);
      const int r = row0 + min(block_row, n_rows - 1), G = P.Hq / P.Hkv;
      tok.head = hk * G + r % G;
      return tok;
    };
    auto item = [&]() {
      const volatile int* x = item_s;
      RowsItem it;
      it.r = x[0];
      it.base = x[1];
      it.drafted = x[2];
      it.n0 = x[3];
      return it;
    };
    const bool capped = P.cap_log2 > 0.f, bent = capped || P.slopes;
    bool ok = mbar_wait(BAR(B_QREADY), 0);  // (every row's power of two has been written)
    if (F8) sc *= *(volatile float*)&q_exp[block_row];
    // The row's factor waits for the exponents (raw * sc - ref is one instruction) where it is positive, so that scores have
    // their maximum where the raw ones have it, and nothing is done to the scores in between.
    const bool late = sc > 0.f && !bent;
    const float in = late ? 1.f : sc, out = late ? sc : 1.f;
    float m = ROWS_NEG_BIG, l = 0.f;
    const int turns = by_rows ? n_tiles : (n_tiles + 1 - group) >> 1;
    for (int turn = 0; turn < turns && ok; ++turn) {
      const int t = by_rows ? turn : 2 * turn + group, place0 = range0 + t * BKV;
      ok = mbar_wait(BAR(B_SFULL + group), turn & 1);  // (the products of the group's last tile, issued before it, are complete too)
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_addr = tmem + group * 128 + lane_addr;
      // Masked tiles, capped scores, distance biases and factors that are not positive: the scores are made final in tensor
      // memory first, 16 at a time.  (Beside the 64 scores below their code made the others' registers spill: 10 % of the kernel.)
      const bool special = masked_tile(place0) || !late;
      if (__builtin_expect(special, 0)) {
        const RowsToken tok = token();
        const RowsItem it = item();
#pragma unroll 1
        for (int c0 = col0; c0 < col0 + CP; c0 += 16) {
          uint32_t v[16];
          tmem_ld16(s_addr + c0, v);
          tmem_ld_wait();
          const int place = place0 + c0;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float x = __uint_as_float(v[c]) * in;
            if (F8) x *= scales_p[(t % SLOTS) * BKV + c0 + c];
            v[c] = __float_as_uint(x);
          }
          if (capped) {
            // the polynomial where no score of the warp lies outside its range (a NaN does: it keeps to the general form)
            float far = 0.f;
#pragma unroll
            for (int c = 0; c < 16; ++c) far = __uint_as_float(v[c]) == __uint_as_float(v[c]) ? fmaxf(far, fabsf(__uint_as_float(v[c]))) : INFINITY;
            if (!__any_sync(0xffffffffu, far > 1.f)) {
#pragma unroll
              for (int c = 0; c < 16; ++c) v[c] = __float_as_uint(P.cap_log2 * cap_tanh_small(__uint_as_float(v[c])));
            } else {
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const float x = __uint_as_float(v[c]);
                v[c] = __float_as_uint(x == x ? P.cap_log2 * cap_tanh(x) : x);
              }
            }
          }
          // which of these keys the row's token sees: those at cached places from its first one on (up to its own, or before the tree) ...
          const int hi = P.cu_q ? min(it.base, end) : min(tok.p + 1, end), from = max(max(tok.lo, begin) - place, 0), to = min(hi - place, 16);
          uint32_t sees = to > from ? (0xffffu >> (16 - (to - from))) << from : 0u;
          if (P.cu_q && place + 16 > it.base) {  // ... and the drafted ones of its mask
            const int j0 = place - it.base, words = P.words, n = min(it.drafted, end - it.base);
            const int* mask = P.masks + (size_t)tok.n * words;
            const int w0 = j0 >> 5, sh = j0 & 31;  // (bits j0 .. j0 + 15 lie in two words)
            const uint32_t a = w0 >= 0 && w0 < words ? (uint32_t)mask[w0] : 0u, b = w0 + 1 >= 0 && w0 + 1 < words ? (uint32_t)mask[w0 + 1] : 0u;
            uint32_t bits = __funnelshift_r(a, b, sh);
            const int cut0 = max(max(-j0, begin - place), 0), cut1 = min(n - j0, 16);
            bits &= cut1 > cut0 ? (0xffffu >> (16 - (cut1 - cut0))) << cut0 : 0u;
            if (tok.lo > 0)
              for (uint32_t left = bits; left; left &= left - 1) {
                const int c = __ffs(left) - 1;
                if (P.positions[P.cu_q[it.r] + j0 + c] < tok.lo) bits &= ~(1u << c);
              }
            sees |= bits;
          }
          if (P.slopes) {
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              int key_pos = place + c;
              if (P.cu_q && key_pos >= it.base) key_pos = key_pos - it.base < it.drafted ? P.positions[P.cu_q[it.r] + key_pos - it.base] : 0;
              v[c] = __float_as_uint(fmaf(-tok.slope, (float)(tok.p - key_pos), __uint_as_float(v[c])));
            }
          }
#pragma unroll
          for (int c = 0; c < 16; ++c) v[c] = (sees >> c) & 1 ? v[c] : 0xff800000u;
          __syncwarp();
          tmem_st16(s_addr + c0, v);
        }
        tmem_st_wait();
      }
      uint32_t v[CP];
      tmem_ld32(s_addr + col0, v);
      tmem_ld32(s_addr + col0 + 32, v + 32);
      tmem_ld_wait();
      if (F8 && !special) {
#pragma unroll
        for (int c = 0; c < CP; c += 4) {
          const ulonglong2 ks = *reinterpret_cast<const ulonglong2*>(scales_p + (t % SLOTS) * BKV + col0 + c);
          const uint64_t w[2] = {ks.x, ks.y};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint64_t f = mul2(w[u],
                                    pack2(__uint_as_float(v[c + 2 * u]), __uint_as_float(v[c + 2 * u + 1])));
            v[c + 2 * u] = (uint32_t)f;
            v[c + 2 * u + 1] = (uint32_t)(f >> 32);
          }
        }
      }
      float mx4[4] = {ROWS_NEG_BIG, ROWS_NEG_BIG, ROWS_NEG_BIG, ROWS_NEG_BIG};  // four chains instead of one long one
#pragma unroll
      for (int c = 0; c < CP; c += 2) mx4[(c >> 1) & 3] = max3(mx4[(c >> 1) & 3], __uint_as_float(v[c]), __uint_as_float(v[c + 1]));
      float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      // the row's maximum over all parts (double-buffered by the meeting's parity: a partner may be a tile ahead)
      const int mp = turn & 1;
      xmax[mp][group][part][row] = mx;
      mbar_arrive(BAR(B_MEET + 4 * group + quarter));
      ok = mbar_wait(BAR(B_MEET + 4 * group + quarter), mp);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
#pragma unroll
      for (int q = 0; q < PARTS; ++q) mx = fmaxf(mx, xmax[mp][group][q][row]);
      // While no row of this quarter has grown by more than GROWTH beyond its reference, the references stay and O is not
      // rescaled, which takes 700 cycles and more.  All threads of these rows decide alike: they hold the same references.  8 bits:
      // the weights may exceed 1 (up to 2^16: 32-bit sums and bfloat16 weights lose nothing by it).  Bfloat16 caches: a new
      // reference lies that much above what the headroom for large values asks for.
      mx = mx > 0.5f * ROWS_NEG_BIG ? mx * out + (F8 ? 0.f : ROWS_HEADROOM) : ROWS_NEG_BIG;
      const float top = mx;
      mx = fmaxf(m, mx);
      if (__all_sync(0xffffffffu, mx - m <= (F8 ? GROWTH : 0.f))) mx = m;
      else if (!F8) mx = fmaxf(m, top + GROWTH);
      const float corr = m == mx ? 1.f : rows_exp2(m - mx);
      const uint64_t out2 = pack2(out, out), mx2 = pack2(-mx, -mx);
      float rs4[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t packed[CP / 2];
#pragma unroll
      for (int c = 0; c < CP; c += 4) {
        const uint64_t e0 = fma2(pack2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), out2, mx2), e1 = fma2(pack2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])), out2, mx2);
        const float p0 = rows_exp2(__uint_as_float((uint32_t)e0)), p1 = rows_exp2(__uint_as_float((uint32_t)(e0 >> 32)));
        const float p2 = rows_exp2(__uint_as_float((uint32_t)e1)), p3 = rows_exp2(__uint_as_float((uint32_t)(e1 >> 32)));
        rs4[0] += p0; rs4[1] += p1; rs4[2] += p2; rs4[3] += p3;
        const __nv_bfloat162 a = __floats2bfloat162_rn(p0, p1), b = __floats2bfloat162_rn(p2, p3);
        packed[c >> 1] = *reinterpret_cast<const uint32_t*>(&a);
        packed[(c >> 1) + 1] = *reinterpret_cast<const uint32_t*>(&b);
      }
      // P over the first half of this S buffer: keys 2c and 2c + 1 in column c (the partners have read their scores: they met
      // after their loads)
      tmem_st32(s_addr + part * (CP / 2), packed);
      l = fmaf(l, corr, (rs4[0] + rs4[1]) + (rs4[2] + rs4[3]));
      m = mx;
      if (turn > 0 && !__all_sync(0xffffffffu, corr == 1.f)) {
#pragma unroll
        for (int c0 = 0; c0 < T::OC; c0 += 32) {
          uint32_t o[32];
          tmem_ld32(o_addr + part * T::OC + c0, o);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
          tmem_st32(o_addr + part * T::OC + c0, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(BAR(B_PREADY + group));
    }
    // the end: the last products, what the groups have joined, the store.  Both groups' last meetings must be over before xmax is
    // written again: the last product comes after all of them.
    if (ok && n_tiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(BAR(B_ODONE), 0));
    if (ok) {
      tc_fence_after();
      xmax[0][group][part][row] = l;
      if (part == 0) ends[group][row] = m;
      mbar_arrive(BAR(B_END + quarter));
      ok = __all_sync(0xffffffffu, mbar_wait(BAR(B_END + quarter), 0));
    }
    if (ok) {
      // Rows of its own: a thread stores half of its row from its group's O.  Shared rows: a quarter of it, from both.
      float f0 = 1.f, f1 = 0.f, total = xmax[0][group][0][row] + xmax[0][group][1][row];
      uint32_t o_first = o_addr;
      int col = part * T::OC;
      if (!by_rows) {
        m = fmaxf(ends[0][row], ends[1][row]);
        f0 = rows_exp2(ends[0][row] - m);
        f1 = rows_exp2(ends[1][row] - m);
        total = fmaf(xmax[0][1][0][row] + xmax[0][1][1][row], f1, (xmax[0][0][0][row] + xmax[0][0][1][row]) * f0);
        o_first = tm_o + lane_addr;
        col = (group * PARTS + part) * T::OE;
      }
      const bool both = !by_rows && n_tiles > 1, bad = *(volatile int*)&any_bad;
      const int col_end = col + (by_rows ? T::OC : T::OE);
      const RowsToken tok = token();
      const RowsItem it = item();
      const size_t at = (size_t)(tok.n + (P.splits > 1 ? rows_part_shift(P, item_i, it.n0) : 0)) * P.Hq + tok.head;
      const float inv = P.splits > 1 ? 1.f : rows_inverse(P, m, total, tok.head);
      if (P.splits > 1 && col == 0 && block_row < n_rows) P.part_ml[at * P.splits + split] = make_float2(m, total);
#pragma unroll 1
      for (; col < col_end; col += 16) {
        __syncwarp();
        uint32_t o[16], o1[16];
        if (n_tiles > 0) {
          tmem_ld16(o_first + col, o);
          if (both) tmem_ld16(tm_o + lane_addr + 128 + col, o1);
          tmem_ld_wait();
        }
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float x = n_tiles > 0 ? __uint_as_float(o[c]) * f0 : 0.f;
          o[c] = __float_as_uint(both ? fmaf(__uint_as_float(o1[c]), f1, x) : x);
        }
        if (block_row >= n_rows) continue;
        if (bad) {  // the values that were taken out, for the rows that see them
          for (int place = begin; place < end; ++place) {
            int key_pos;
            if (!masked_tile(place / BKV * BKV) || !rows_sees(P, it, tok.n, tok.p, tok.lo, place, key_pos)) continue;
            const int row_c = rows_cache_row(P, table, hk, place);
            if (row_c < 0) continue;
            if (F8 && P.scales[row_c + v_off] != FP8_BAD) continue;
            const bf16* vp = reinterpret_cast<const bf16*>(P.pages) + (size_t)(row_c + v_off) * DH + col;
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const float y = F8 ? __int_as_float(0x7fc00000) : __bfloat162float(vp[c]);
              if (!isfinite(y)) o[c] = __float_as_uint(__uint_as_float(o[c]) + y);
            }
          }
        }
        if (P.splits > 1) {
          float4* dst = reinterpret_cast<float4*>(P.part_o + (at * P.splits + split) * DH + col);
#pragma unroll
          for (int c = 0; c < 16; c += 4)
            dst[c >> 2] = make_float4(__uint_as_float(o[c]), __uint_as_float(o[c + 1]), __uint_as_float(o[c + 2]), __uint_as_float(o[c + 3]));
        } else {
          uint4* dst = reinterpret_cast<uint4*>(P.out + at * DH + col);
#pragma unroll
          for (int c = 0; c < 16; c += 8) {
            uint4 x;
            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&x);
#pragma unroll
            for (int u = 0; u < 4; ++u) h[u] = __floats2bfloat162_rn(__uint_as_float(o[c + 2 * u]) * inv, __uint_as_float(o[c + 2 * u + 1]) * inv);
            dst[c >> 3] = x;
          }
        }
      }
    }
    if (!ok && lane == 0) {
      atomicOr(P.status, JLX_STATUS_WAIT_TIMEOUT);
      failed = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// -------------------------------------------------------------------------------------------- host
template <int DH, bool F8>
static int launch_tc(const RowsParams& P, int box_rows, int row_block, int row_tiles, cudaStream_t stream) {
  static unsigned long long allowed = 0;  // a bit per device: the attribute belongs to the device's context
  int dev = 0;
  JLX_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(allowed >> dev & 1)) {
    JLX_CUDA(cudaFuncSetAttribute(attention_rows_tc_kernel<DH, F8>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcTile<DH, F8>::SMEM));
    if (dev < 64) allowed |= 1ull << dev;
  }
  CUtensorMap map;
  if (int rc = rows_map(P, DH, F8, box_rows, &map)) return rc;
  const long long blocks = (long long)P.n_items * P.splits * P.Hkv * row_tiles;
  JLX_REQUIRE(blocks < (1ll << 31), "attention over rows: too many items or rows");
  JLX_CUDA(jlx_launch_pdl(attention_rows_tc_kernel<DH, F8>, dim3((unsigned)blocks), dim3(NTHREADS), TcTile<DH, F8>::SMEM, stream, map, P, box_rows, row_block, row_tiles));
  return 0;
}

JLX_API int jlx_attention_rows_tc(const RowsArgs* a, cudaStream_t stream) {
  RowsParams P;
  if (rows_params(*a, P)) return 1;
  JLX_REQUIRE(a->page_size % 16 == 0 && ((uintptr_t)a->scales & 15) == 0, "attention over rows (tcgen05): needs pages of a multiple of 16 tokens and scales on a 16-byte boundary");
  if (P.n_items == 0) return 0;
  const int rows = a->max_count * (P.Hq / P.Hkv), box_rows = P.page_size % 64 == 0 ? 64 : P.page_size % 32 == 0 ? 32 : 16;
  JLX_REQUIRE(P.splits == 1 || (P.part_o && P.part_ml), "attention over rows: scratch for the ranges is missing");
  JLX_REQUIRE(a->row_block == BQ || a->row_block == BROWS, "attention over rows (tcgen05): %d rows a block (128 or 256)", a->row_block);
  const int row_tiles = (rows + a->row_block - 1) / a->row_block;
  const int rc = a->dh == 128 ? (P.scales ? launch_tc<128, true>(P, box_rows, a->row_block, row_tiles, stream) : launch_tc<128, false>(P, box_rows, a->row_block, row_tiles, stream))
                              : (P.scales ? launch_tc<64, true>(P, box_rows, a->row_block, row_tiles, stream) : launch_tc<64, false>(P, box_rows, a->row_block, row_tiles, stream));
  if (rc || P.splits == 1) return rc;
  return a->dh == 128 ? launch_rows_join<128>(P, a->max_count, stream) : launch_rows_join<64>(P, a->max_count, stream);
}
