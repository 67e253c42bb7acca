// Grouped-query attention of up to 16 query rows a block of an item and KV head over the paged cache, held in bfloat16 or in 8
// bits: single decoded tokens and small drafted trees (attention_rows.cuh has mask and formula), head sizes 64 and 128.  It reads
// every key once and computes little with it: bytes bound it, and the instructions that stand between a byte and a product.
//
// A block takes one range of an item's keys, in tiles of 64: a warp of its own fetches them up to STAGES tiles ahead, by TMA
// where pages hold whole boxes of 16, 32 or 64 rows (a lane per box: its entry of the block table, a tile ahead, and a few
// copies), else by cp.async, row by row (any page size; that warp then sets the pace).  Four warps take 16 keys of every tile
// each and meet only at the end.
//
// The products are transposed, S^T = K Q^T and O^T = V^T P^T: keys and entries fill the 16 rows of a tensor-core tile and the
// query rows its 8 columns, of which a group of 5 heads wastes 3, not 11 of 16.  That halves products, scores, exponentials and
// accumulators against query rows as rows (590 -> 280 instructions a warp and tile, 160 -> 100 registers), which is what lets
// the warps keep up with the memory.
//
// 8 bits: codes go to the tensor cores as float16, which holds every one of them; no number of the cache is rounded.  A key's
// power of two multiplies its row of scores.  A value's is added to its key's exponent: with a_j = s_j + e_j the weights
// w_j = 2^(a_j - ref) and the sum  sum w_j 2^-e_j  give  out = sum w_j code_j / sum w_j 2^-e_j,  so that float16 rounds each
// weight by 2^-11 of it at most, or by 2^-25 where it is below 2^-14: keys whose weight times scale is below 2^-25 of the
// row's largest add to the sum and no longer to the values, of which they are at most as small a part.  (Scales lie within
// 2^-60 .. 2^60: no product leaves the 32-bit range.)  Queries are brought to float16 by a power of two per row, which makes the
// largest entry 2^7 .. 2^8: entries above 2^-24 of it are exact, smaller ones off by 2^-32 of it at most.
// Bfloat16 caches: probabilities are rounded to bfloat16 for the product with the values (2^-8 of each at most).  Sums and
// outputs are 32-bit in both.
//
// The contraction index of a product may run in any order that both operands share, and this is what makes codes cheap: the 16
// codes that a thread reads at once (16 bytes of a key) serve four steps of the score product, whose query fragments are
// gathered in that order; of the values a transposing load of byte pairs gives two keys' codes of two neighbouring entries,
// which a byte permutation turns into an operand whose rows are the even, then the odd entries.
//
// The reference `ref` of a row's exponents is not its running maximum: it moves, with a rescaling of the outputs, only when a
// score outgrows it by 2^GROWTH (weights up to 64: no trouble for float16 or a 32-bit sum), so a tile costs one vote instead of
// a maximum over all its keys.  Over a bfloat16 cache it moves by as much beyond the headroom that keeps large values' sums finite.
//
// Ranges of one item (few items, long contexts) are a thread-block cluster of up to 8: they leave their sums in shared memory
// and each reads its share of the others' there, no second kernel and no scratch.  More ranges than that go through scratch.
//
// What bounds it: in long caches the instructions between a byte and a product (a tile's 280 a warp), in short ones a block's way to its first tile (page, position, key: 2 us) and the launch.  Measured
// (B200, 40 heads on 8 of 128, 8 bits): 64 requests of up to 8,192 keys 153 us, 5.35 TB/s, 82 % of the copy rate; 8 of up to
// 30,000 78 us, 5.05 TB/s; one of 700 13 us with its call, 8.4 on the device.
// Tried and slower: 8-bit score products (the conversion of queries' remainders costs more than the codes'), a reference taken
// from the tile before with a second pass where it fails, exponentials by a polynomial.
#include <cooperative_groups.h>
#include <cuda.h>

#include "attention_rows.cuh"
#include "mbarrier.cuh"
#include "mma_sync.cuh"

#define KT 64           // keys per tile
#define GROWTH 6.0f
#define CONSUMERS 4     // warps with 16 keys of a tile each
#define MAX_CLUSTER 8

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit numbers, two of a row per thread, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Where 16-byte chunk c of row `row` lies in a tile of KT rows of CH chunks: as TMA's swizzle of rows of 64 or 128 bytes puts
// it; rows of 256 bytes are two halves of 128.
template <int CH> __device__ __forceinline__ int chunk_at(int row, int c) {
  if (CH == 4) return row * 4 + (c ^ ((row >> 1) & 3));
  return (c >> 3) * KT * 8 + row * 8 + ((c & 7) ^ (row & 7));
}
// The key at position i of eight in the products: two keys whose four chunks a quarter of a warp reads at once (positions 2i
// and 2i + 1) then differ in bit 2 of the swizzle, and fall on different banks.
__device__ __forceinline__ int key_at(int i) { return (i >> 1) | ((i & 1) << 2); }

template <int DH, bool F8, int NG> struct FewTile {
  static constexpr int ELEM = F8 ? 1 : 2;
  static constexpr int CH = DH * ELEM / 16;     // 16-byte chunks per row
  static constexpr int BYTES = KT * DH * ELEM;  // keys or values of a tile
  static constexpr int STAGES = DH * ELEM >= 256 ? 3 : 4;
  static constexpr int SCALE_BYTES = F8 ? 2 * KT : 0;  // per stage: the keys' scale bytes, the values'
  static constexpr int LD = DH + 4;             // floats between rows of the outputs as the warps leave them
  static constexpr int RING = STAGES * (2 * BYTES + SCALE_BYTES);
  static constexpr int MERGE = (CONSUMERS + 1) * 8 * NG * (LD * 4 + 8);
  static constexpr int SMEM = (RING > MERGE ? RING : MERGE) + 1024;  // (up to 1 KB for the alignment)
};

// The scales of a box whose page is missing: copied like any other's.  (What the fetching warp does between a free stage and its
// copies counts: fewer bytes to wait for in such tiles, with plain stores of zeros, took 87 us for 78 with 8 requests of up to
// 30,000 keys, copies from a row of their own 82, a branch around them 80.)
__device__ __align__(16) uint8_t no_scales[KT];

// NG: groups of 8 query rows (1, 2).  Registers for as many blocks of a multiprocessor as its shared memory has room for (heads of
// 128 in bfloat16, two groups: 209 registers and one block otherwise, six requests of 4,000 keys 25 us for 20).
template <int DH, bool F8, int NG>
__global__ void __launch_bounds__((CONSUMERS + 1) * 32, DH == 128 && NG == 2 ? 2 : 3) attention_few_kernel(const __grid_constant__ CUtensorMap map, const RowsParams P, int clustered, int box_rows) {
  JLX_TL(TL_ATTN_DECODE);
  using T = FewTile<DH, F8, NG>;
  constexpr int CH = T::CH, STAGES = T::STAGES, ROWS = 8 * NG;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);  // where the swizzle's pattern starts
  __shared__ __align__(8) uint64_t bars[2 * STAGES];
  __shared__ int4 row_tok[ROWS];   // (token, head, position, first key) of the block's rows
  __shared__ float2 row_sc[ROWS];  // (score factor, slope)
  __shared__ int any_bad;
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int split = blockIdx.x % P.splits, item_i = blockIdx.x / P.splits;
  const int tiles_y = gridDim.y / P.Hkv, hk = blockIdx.y / tiles_y, row0 = (blockIdx.y - hk * tiles_y) * ROWS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  RowsItem it;
  if (!rows_tokens(P, item_i, it)) return;
  const int G = P.Hq / P.Hkv, n_rows = min(it.cnt * G - row0, ROWS);
  if (n_rows <= 0) return;
  // every warp looks at the rows itself (at most 16): what they see together, and (warp 0) their description for all
  const RowsToken tok = rows_token(P, it, row0 + min(lane, n_rows - 1), hk);
  if (!rows_request(P, it)) return;
  const uint32_t bar0 = smem_u32(bars);
  auto FULL = [&](int s) { return bar0 + 8u * s; };
  auto EMPTY = [&](int s) { return bar0 + 8u * (STAGES + s); };
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(FULL(s), box_rows ? 1 : F8 ? 33 : 32);  // TMA's bytes; else every lane's copies, and the scales' store
      mbar_init(EMPTY(s), CONSUMERS);
    }
    any_bad = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0 && lane < ROWS) {
    row_tok[lane] = make_int4(tok.n, tok.head, tok.p, tok.lo);
    row_sc[lane] = make_float2(tok.sc, tok.slope);
  }
  const int lo_min = __reduce_min_sync(0xffffffffu, tok.lo), lo_max = __reduce_max_sync(0xffffffffu, tok.lo);
  const int p_min = __reduce_min_sync(0xffffffffu, tok.p), p_max = __reduce_max_sync(0xffffffffu, tok.p);
  const int first = P.cu_q ? min(lo_min, it.base) : lo_min, end_all = rows_end(P, it, p_max);
  const int full_lo = lo_max, full_hi = P.cu_q ? it.base : p_min + 1;  // keys in between are seen by every row
  // equal ranges of whole tiles (an item's own: a short request's blocks are as short as each other)
  const int start = first / KT * KT, per = max((end_all - start + KT * P.splits - 1) / (KT * P.splits), 0) * KT, range0 = start + split * per;
  const int begin = max(first, range0), end = min(end_all, range0 + per);
  const int n_tiles = end > begin ? (end - range0 + KT - 1) / KT : 0;
  const int* table = P.block_table + (size_t)it.r * P.bt_stride;
  const int v_off = P.Hkv * P.page_size;  // rows between a key and its value
  auto k_tile = [&](int s) { return smem + s * 2 * T::BYTES; };
  auto scales_of = [&](int s) { return smem + STAGES * 2 * T::BYTES + s * T::SCALE_BYTES; };
  __syncthreads();

  float m[NG][2], l[NG][2];
  float o[NG][DH / 16][4];
  if (warp == CONSUMERS) {
    // ------------------------------------------------------------------------------ the fetching warp
    bool ok = true;
    if (box_rows) {
      // lane i has box i of every tile
      const int boxes = KT / box_rows;
      auto find_page = [&](int t) {
        const int pi = (range0 + t * KT + lane * box_rows) / P.page_size;
        return lane < boxes && t < n_tiles && pi < P.bt_stride ? table[pi] : -1;
      };
      int page = find_page(0);
      int t = 0;
#pragma unroll 1
      for (; t < n_tiles; ++t) {
        const int s = t % STAGES;
        if (t >= STAGES) ok = mbar_wait(EMPTY(s), (t / STAGES - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(FULL(s), 2 * T::BYTES + T::SCALE_BYTES);
        __syncwarp();
        if (lane < boxes) {
          const int place = range0 + t * KT + lane * box_rows;
          const bool there = rows_page_there(P, page);
          if (!there && place < end && place + box_rows > begin) atomicOr(P.status, JLX_STATUS_BAD_PAGE);
          if (!there) page = P.num_pages;
          const int row = (page * 2 * P.Hkv + hk) * P.page_size + place % P.page_size, to_v = there ? v_off : 0;
          const uint8_t* bytes = there ? P.scales + row : no_scales;
          const uint32_t dst = smem_u32(k_tile(s)) + lane * box_rows * (CH == 4 ? 64 : 128);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
#pragma unroll
            for (int h = 0; h < (CH + 7) / 8; ++h) tma_load_2d(dst + w * T::BYTES + h * KT * 128, &map, h * 128 / T::ELEM, row + w * v_off, FULL(s));
            if (F8) bulk_load(smem_u32(scales_of(s)) + w * KT + lane * box_rows, bytes + w * to_v, box_rows, FULL(s));
          }
        }
        page = find_page(t + 1);
      }
      if (!ok)  // let the copies in flight land before the block's shared memory is given up
        for (int u = max(0, t - STAGES); u < t; ++u) mbar_wait(FULL(u % STAGES), (u / STAGES) & 1);
    } else {
    // Lane i knows the rows of keys 2i and 2i + 1 of the tile; each copy instruction takes 32 / CH rows.  The scales of a tile
    // are loaded before its copies are issued and stored a tile later, when they have come.
    auto find_rows = [&](int t) {
      const int place = range0 + t * KT + 2 * lane;
      return make_int2(t < n_tiles && place >= begin && place < end ? rows_cache_row(P, table, hk, place) : -1,
                       t < n_tiles && place + 1 >= begin && place + 1 < end ? rows_cache_row(P, table, hk, place + 1) : -1);
    };
    auto put_scales = [&](int t, const int4& bytes) {
      uint8_t* sc = scales_of(t % STAGES);
      *reinterpret_cast<uint16_t*>(sc + 2 * lane) = (uint16_t)(bytes.x | bytes.y << 8);
      *reinterpret_cast<uint16_t*>(sc + KT + 2 * lane) = (uint16_t)(bytes.z | bytes.w << 8);
      __syncwarp();
      if (lane == 0) mbar_arrive(FULL(t % STAGES));
    };
    int2 row = find_rows(0);
    int4 bytes_before = make_int4(0, 0, 0, 0);
#pragma unroll 1
    for (int t = 0; t < n_tiles; ++t) {
      const int s = t % STAGES;
      if (t >= STAGES) ok = mbar_wait(EMPTY(s), (t / STAGES - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      int4 bytes = make_int4(0, 0, 0, 0);
      if (F8) {
        bytes.x = row.x >= 0 ? P.scales[row.x] : 0;
        bytes.y = row.y >= 0 ? P.scales[row.y] : 0;
        bytes.z = row.x >= 0 ? P.scales[row.x + v_off] : 0;
        bytes.w = row.y >= 0 ? P.scales[row.y + v_off] : 0;
      }
      const uint32_t dst0 = smem_u32(k_tile(s));
      const int c = lane % CH;
#pragma unroll 8
      for (int i = 0; i < KT * CH / 32; ++i) {
        const int j = i * (32 / CH) + lane / CH;
        const int rx = __shfl_sync(0xffffffffu, row.x, j >> 1), ry = __shfl_sync(0xffffffffu, row.y, j >> 1);
        const int r = (j & 1) ? ry : rx;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(P.pages) + ((size_t)max(r, 0) * CH + c) * 16;
        const uint32_t dst = dst0 + chunk_at<CH>(j, c) * 16;
        cp_async16(dst, src, r >= 0);
        cp_async16(dst + T::BYTES, src + (r >= 0 ? (size_t)v_off * CH * 16 : 0), r >= 0);
      }
      cp_async_arrive(FULL(s));
      row = find_rows(t + 1);
      if (F8) {
        if (t > 0) put_scales(t - 1, bytes_before);
        bytes_before = bytes;
      }
    }
    if (F8 && ok && n_tiles > 0) put_scales(n_tiles - 1, bytes_before);
    cp_async_commit();
    cp_async_wait<0>();  // nothing is in flight when the ring is used for something else
    }
    if (!ok && lane == 0) atomicOr(P.status, JLX_STATUS_WAIT_TIMEOUT);
  } else {
    // ------------------------------------------------------------------------------ the computing warps
    // queries: column g of group ng is row 8 ng + g, its entries in the order of the scores' contraction
    uint32_t qf[NG][DH / 16][2];
    float sc[NG][2], slope[NG][2];
    int4 tk[NG][2];
#pragma unroll
    for (int ng = 0; ng < NG; ++ng) {
      const int4 of = row_tok[8 * ng + g];
      const bf16* q = P.q + ((size_t)of.x * P.Hq + of.y) * DH;
      int e = 0;
      if (F8) {
        uint4 a[DH / 64][2];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < DH / 64; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            a[i][u] = *reinterpret_cast<const uint4*>(q + i * 64 + t4 * 16 + u * 8);
            const __nv_bfloat162* pa = reinterpret_cast<const __nv_bfloat162*>(&a[i][u]);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float2 f = __bfloat1622float2(pa[x]);
              top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the row's power of two: its largest entry into [2^7, 2^8)
        e = max(min((int)(__float_as_uint(top) >> 23) - 127, 120), -110) - 7;
        const float in = fp8_pow2(-e);
#pragma unroll
        for (int i = 0; i < DH / 64; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const __nv_bfloat162* pa = reinterpret_cast<const __nv_bfloat162*>(&a[i][w >> 1]) + (w & 1) * 2;
            const float2 f0 = __bfloat1622float2(pa[0]), f1 = __bfloat1622float2(pa[1]);
            const __half2 h0 = __floats2half2_rn(f0.x * in, f0.y * in), h1 = __floats2half2_rn(f1.x * in, f1.y * in);
            qf[ng][i * 4 + w][0] = *reinterpret_cast<const uint32_t*>(&h0);
            qf[ng][i * 4 + w][1] = *reinterpret_cast<const uint32_t*>(&h1);
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < DH / 16; ++ks) {
          qf[ng][ks][0] = *reinterpret_cast<const uint32_t*>(q + ks * 16 + t4 * 2);
          qf[ng][ks][1] = *reinterpret_cast<const uint32_t*>(q + ks * 16 + t4 * 2 + 8);
        }
      }
      // this thread's scores are those of rows 2 t4 and 2 t4 + 1 of the group
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 2 * t4 + c, er = __shfl_sync(0xffffffffu, e, r * 4);
        tk[ng][c] = row_tok[8 * ng + r];
        const float2 f = row_sc[8 * ng + r];
        sc[ng][c] = F8 ? f.x * fp8_pow2(er) : f.x;
        slope[ng][c] = f.y;
        m[ng][c] = ROWS_NEG_BIG;
        l[ng][c] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < DH / 16; ++i) o[ng][i][0] = o[ng][i][1] = o[ng][i][2] = o[ng][i][3] = 0.f;
    }
    const bool capped = P.cap_log2 > 0.f, bent = capped || P.slopes;
    const int key0 = warp * 16;
    const int kg = key0 + key_at(g), kl = key0 + key_at(lane & 7);
    bool ok = true;

#pragma unroll 1
    for (int t = 0; t < n_tiles; ++t) {
      const int st = t % STAGES, place0 = range0 + t * KT;
      const bool masked = place0 < full_lo || place0 + KT > min(full_hi, end) || place0 < begin;
      ok = mbar_wait(FULL(st), (t / STAGES) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint8_t* kt = k_tile(st);
      uint8_t* vt = k_tile(st) + T::BYTES;
      if (__builtin_expect(masked, 0)) {
        // A value that is not finite leaves the tile before the product (a warp reads its own keys' values only).  Codes of rows
        // outside the range may be anything, those of rows inside are numbers.
        bool any = false;
#pragma unroll 1
        for (int i = lane; i < 16 * CH; i += 32) {
          const int place = place0 + key0 + i / CH;
          uint4* at = reinterpret_cast<uint4*>(vt + chunk_at<CH>(key0 + i / CH, i % CH) * 16);
          if (place < begin || place >= end) {
            *at = make_uint4(0u, 0u, 0u, 0u);
          } else if (!F8) {
            uint32_t w[4] = {at->x, at->y, at->z, at->w};
            bool bad = false;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              if ((w[u] & 0x7f80u) == 0x7f80u) { w[u] &= 0xffff0000u; bad = true; }
              if ((w[u] & 0x7f800000u) == 0x7f800000u) { w[u] &= 0xffffu; bad = true; }
            }
            if (bad) {
              *at = make_uint4(w[0], w[1], w[2], w[3]);
              any = true;
            }
          }
        }
        if (any) any_bad = 1;
        // (the stage's next copies are writes of the asynchronous proxy: these stores have to be ordered before them, too)
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      // ---- S^T: two keys (g, g + 8) x two rows per thread and group; two chains of products
      float s[NG][2][4];
#pragma unroll
      for (int ng = 0; ng < NG; ++ng)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[ng][u][0] = s[ng][u][1] = s[ng][u][2] = s[ng][u][3] = 0.f;
      if (F8) {
#pragma unroll
        for (int b = 0; b < DH / 64; ++b) {
          const uint4 c0 = *reinterpret_cast<const uint4*>(kt + chunk_at<CH>(kg, b * 4 + t4) * 16);
          const uint4 c1 = *reinterpret_cast<const uint4*>(kt + chunk_at<CH>(kg + 8, b * 4 + t4) * 16);
          const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a[4];
            fp8x4_to_half(w0[w], a[0], a[2]);
            fp8x4_to_half(w1[w], a[1], a[3]);
#pragma unroll
            for (int ng = 0; ng < NG; ++ng) mma_f16(s[ng][w & 1], a, qf[ng][b * 4 + w][0], qf[ng][b * 4 + w][1]);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < DH / 16; ++ks) {
          uint32_t a[4];
          ldmatrix_x4(smem_u32(kt + chunk_at<CH>(kl + ((lane >> 3) & 1) * 8, ks * 2 + (lane >> 4)) * 16), a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int ng = 0; ng < NG; ++ng) mma_bf16(s[ng][ks & 1], a, qf[ng][ks][0], qf[ng][ks][1]);
        }
      }
      // ---- base-2 exponents of the weights, and which of them count
      float ks0 = 1.f, ks1 = 1.f, ve0 = 0.f, ve1 = 0.f, vi0 = 1.f, vi1 = 1.f;  // keys' scales; values' exponents and 2^-exponent
      if (F8) {
        const uint8_t* sp = scales_of(st) + kg;
        const int bk0 = sp[0], bk1 = sp[8], bv0 = fp8_weight_byte(sp[KT]), bv1 = fp8_weight_byte(sp[KT + 8]);
        ks0 = fp8_scale(bk0);
        ks1 = fp8_scale(bk1);
        ve0 = bv0 == FP8_BAD ? __int_as_float(0x7fc00000) : (float)(bv0 - 127);
        ve1 = bv1 == FP8_BAD ? __int_as_float(0x7fc00000) : (float)(bv1 - 127);
        vi0 = __int_as_float((254 - min(bv0, 254)) << 23);  // (finite for any byte: a masked key's weight is 0 and stays 0)
        vi1 = __int_as_float((254 - min(bv1, 254)) << 23);
      }
      float x[NG][4];
#pragma unroll
      for (int ng = 0; ng < NG; ++ng)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float raw = s[ng][0][e] + s[ng][1][e];
          x[ng][e] = F8 ? raw * (sc[ng][e & 1] * (e < 2 ? ks0 : ks1)) : raw * sc[ng][e & 1];
        }
      // (one branch around all that most tiles do without: a jump over each element's part of it costs an instruction fetch)
      if (__builtin_expect(masked || bent, 0)) {
#pragma unroll
        for (int ng = 0; ng < NG; ++ng)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = x[ng][e];
            if (capped) v = v == v ? P.cap_log2 * cap_tanh(v) : v;
            int key_pos;
            const int4 k = tk[ng][e & 1];
            const int place = place0 + kg + (e < 2 ? 0 : 8);
            const bool sees = place >= begin && place < end && rows_sees(P, it, k.x, k.z, k.w, place, key_pos);
            x[ng][e] = sees ? fmaf(-slope[ng][e & 1], (float)(k.z - key_pos), v) : -INFINITY;
          }
      }
      bool grown = false;
#pragma unroll
      for (int ng = 0; ng < NG; ++ng)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (F8) x[ng][e] = x[ng][e] == -INFINITY ? x[ng][e] : x[ng][e] + (e < 2 ? ve0 : ve1);  // (a masked key's scale may be anything)
          grown |= x[ng][e] > m[ng][e & 1] + (F8 ? GROWTH : -ROWS_HEADROOM);
        }
      if (__builtin_expect(__any_sync(0xffffffffu, grown), 0)) {
#pragma unroll
        for (int ng = 0; ng < NG; ++ng) {
          float corr[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(x[ng][c], x[ng][c + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            mx = fmaxf(m[ng][c], F8 ? mx : mx + (ROWS_HEADROOM + GROWTH));
            corr[c] = rows_exp2(m[ng][c] - mx);
            m[ng][c] = mx;
            l[ng][c] *= corr[c];
          }
#pragma unroll
          for (int i = 0; i < DH / 16; ++i) {
            o[ng][i][0] *= corr[0]; o[ng][i][1] *= corr[1]; o[ng][i][2] *= corr[0]; o[ng][i][3] *= corr[1];
          }
        }
      }
      uint32_t pb[NG][2];
#pragma unroll
      for (int ng = 0; ng < NG; ++ng) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = rows_exp2(x[ng][e] - m[ng][e & 1]);  // (a masked key's exponent is -infinity: exactly 0)
          l[ng][e & 1] = F8 ? fmaf(w[e], e < 2 ? vi0 : vi1, l[ng][e & 1]) : l[ng][e & 1] + w[e];
        }
        if (F8) {
          const __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
          pb[ng][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h0));
          pb[ng][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h1));
        } else {
          pb[ng][0] = transpose8x8(pack_bf16(w[0], w[1]));
          pb[ng][1] = transpose8x8(pack_bf16(w[2], w[3]));
        }
      }
      // ---- O^T += V^T P^T
      if (F8) {
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
          uint32_t r[4];
          ldmatrix_x4_trans(smem_u32(vt + chunk_at<CH>(kl + ((lane >> 3) & 1) * 8, c + (lane >> 4)) * 16), r[0], r[1], r[2], r[3]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t a[4];  // rows 0-7: the chunk's even entries, rows 8-15: the odd ones
            fp8x4_to_half(__byte_perm(r[2 * u], 0, 0x3120), a[0], a[1]);
            fp8x4_to_half(__byte_perm(r[2 * u + 1], 0, 0x3120), a[2], a[3]);
#pragma unroll
            for (int ng = 0; ng < NG; ++ng) mma_f16(o[ng][c + u], a, pb[ng][0], pb[ng][1]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < DH / 16; ++i) {
          uint32_t a[4];
          ldmatrix_x4_trans(smem_u32(vt + chunk_at<CH>(kl + (lane >> 4) * 8, i * 2 + ((lane >> 3) & 1)) * 16), a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int ng = 0; ng < NG; ++ng) mma_bf16(o[ng][i], a, pb[ng][0], pb[ng][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(EMPTY(st));
    }
    if (!ok && lane == 0) atomicOr(P.status, JLX_STATUS_WAIT_TIMEOUT);
  }
  __syncthreads();  // the ring is free: the warps leave their rows in it

  float* rows_o = reinterpret_cast<float*>(smem);                                         // [CONSUMERS][ROWS][LD], then the merged rows
  float2* rows_ml = reinterpret_cast<float2*>(smem + (CONSUMERS + 1) * ROWS * T::LD * 4);  // [CONSUMERS][ROWS], then the merged rows'
  if (warp < CONSUMERS) {
#pragma unroll
    for (int ng = 0; ng < NG; ++ng)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[ng][c] += __shfl_xor_sync(0xffffffffu, l[ng][c], d);
        const int r = warp * ROWS + 8 * ng + 2 * t4 + c;
        if (g == 0) rows_ml[r] = make_float2(m[ng][c], l[ng][c]);
        float* dst = rows_o + (size_t)r * T::LD;
#pragma unroll
        for (int i = 0; i < DH / 16; ++i) {
          if (F8) *reinterpret_cast<float2*>(dst + i * 16 + 2 * g) = make_float2(o[ng][i][c], o[ng][i][2 + c]);
          else { dst[i * 16 + g] = o[ng][i][c]; dst[i * 16 + g + 8] = o[ng][i][2 + c]; }
        }
      }
  }
  __syncthreads();
  constexpr int Q4 = DH / 4;
  float* merged = rows_o + (size_t)CONSUMERS * ROWS * T::LD;
  float2* merged_ml = rows_ml + CONSUMERS * ROWS;
  auto store = [&](const int4& k, int d, float4 acc, float mm, float ll) {
    const float inv = rows_inverse(P, mm, ll, k.y);
    uint2 v;
    *reinterpret_cast<__nv_bfloat162*>(&v.x) = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
    *reinterpret_cast<__nv_bfloat162*>(&v.y) = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(P.out + ((size_t)k.x * P.Hq + k.y) * DH + d) = v;
  };
  const int part_shift = rows_part_shift(P, item_i, it.n0);
  for (int idx = tid; idx < n_rows * Q4; idx += (CONSUMERS + 1) * 32) {
    const int row = idx / Q4, d = (idx - row * Q4) * 4;
    float mm = ROWS_NEG_BIG, ll = 0.f;
#pragma unroll
    for (int w = 0; w < CONSUMERS; ++w) mm = fmaxf(mm, rows_ml[w * ROWS + row].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < CONSUMERS; ++w) {
      const float2 ml = rows_ml[w * ROWS + row];
      const float f = ml.x == mm ? 1.f : rows_exp2(ml.x - mm);  // (infinite maxima: the others count for nothing)
      const float4 v = *reinterpret_cast<const float4*>(rows_o + (size_t)(w * ROWS + row) * T::LD + d);
      ll = fmaf(ml.y, f, ll);
      acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
    }
    const int4 k = row_tok[row];
    if (!F8 && any_bad) {  // the values that were taken out, for the rows that see them
      for (int place = begin; place < end; ++place) {
        int key_pos;
        const int ts = place / KT * KT;
        if (ts >= max(full_lo, begin) && ts + KT <= min(full_hi, end)) continue;  // (a tile without masks kept them)
        if (!rows_sees(P, it, k.x, k.z, k.w, place, key_pos)) continue;
        const int row_c = rows_cache_row(P, table, hk, place);
        if (row_c < 0) continue;
        const bf16* v = reinterpret_cast<const bf16*>(P.pages) + (size_t)(row_c + v_off) * DH + d;
        const float y[4] = {__bfloat162float(v[0]), __bfloat162float(v[1]), __bfloat162float(v[2]), __bfloat162float(v[3])};
        if (!isfinite(y[0])) acc.x += y[0];
        if (!isfinite(y[1])) acc.y += y[1];
        if (!isfinite(y[2])) acc.z += y[2];
        if (!isfinite(y[3])) acc.w += y[3];
      }
    }
    if (P.splits == 1) {
      store(k, d, acc, mm, ll);
    } else if (clustered) {
      *reinterpret_cast<float4*>(merged + (size_t)row * T::LD + d) = acc;
      if (d == 0) merged_ml[row] = make_float2(mm, ll);
    } else {
      const size_t at = (size_t)(k.x + part_shift) * P.Hq + k.y;
      *reinterpret_cast<float4*>(P.part_o + (at * P.splits + split) * DH + d) = acc;
      if (d == 0) P.part_ml[at * P.splits + split] = make_float2(mm, ll);
    }
  }
  if (clustered) {
    // the ranges of the item: every block takes its share of the outputs and reads the others' sums of it
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int total = n_rows * Q4, share = (total + P.splits - 1) / P.splits;
    for (int idx = split * share + tid; idx < min(total, (split + 1) * share); idx += (CONSUMERS + 1) * 32) {
      const int row = idx / Q4, d = (idx - row * Q4) * 4;
      float2 ml[MAX_CLUSTER];
      float4 v[MAX_CLUSTER];
      float mm = ROWS_NEG_BIG, ll = 0.f;
#pragma unroll
      for (int w = 0; w < MAX_CLUSTER; ++w) {
        if (w >= P.splits) break;
        ml[w] = *cluster.map_shared_rank(&merged_ml[row], w);
        v[w] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(merged + (size_t)row * T::LD + d, w));
        mm = fmaxf(mm, ml[w].x);
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < MAX_CLUSTER; ++w) {
        if (w >= P.splits) break;
        const float f = ml[w].x == mm ? 1.f : rows_exp2(ml[w].x - mm);
        ll = fmaf(ml[w].y, f, ll);
        acc.x = fmaf(v[w].x, f, acc.x); acc.y = fmaf(v[w].y, f, acc.y); acc.z = fmaf(v[w].z, f, acc.z); acc.w = fmaf(v[w].w, f, acc.w);
      }
      store(row_tok[row], d, acc, mm, ll);
    }
    cluster.sync();  // no block leaves while its sums are read
  }
}

// -------------------------------------------------------------------------------------------- host
template <int DH, bool F8, int NG>
static int launch_few(const RowsParams& P, dim3 grid, cudaStream_t stream) {
  using T = FewTile<DH, F8, NG>;
  // boxes of whole rows within a page (and its scales, 16 bytes at a time); 0: pages too small or ragged for TMA
  int box_rows = P.page_size % 64 == 0 ? 64 : P.page_size % 32 == 0 ? 32 : P.page_size % 16 == 0 ? 16 : 0;
  if (F8 && ((uintptr_t)P.scales & 15) != 0) box_rows = 0;
  CUtensorMap map = {};
  if (box_rows) {
    if (int rc = rows_map(P, DH, F8, box_rows, &map)) return rc;
  }
  static unsigned long long allowed = 0;  // a bit per device: the attribute belongs to the device's context
  int dev = 0;
  JLX_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(allowed >> dev & 1)) {
    JLX_CUDA(cudaFuncSetAttribute(attention_few_kernel<DH, F8, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM));
    if (dev < 64) allowed |= 1ull << dev;
  }
  const int clustered = P.splits > 1 && P.splits <= MAX_CLUSTER;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((CONSUMERS + 1) * 32);
  cfg.dynamicSmemBytes = T::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = clustered ? P.splits : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = clustered ? 2 : 1;
  JLX_CUDA(cudaLaunchKernelEx(&cfg, attention_few_kernel<DH, F8, NG>, map, P, clustered, box_rows));
  return 0;
}

template <int DH, bool F8, int NG>
static int few_places(int splits) {
  using T = FewTile<DH, F8, NG>;
  int dev = 0, sms = 0, n = 0;
  bool ok = cudaFuncSetAttribute(attention_few_kernel<DH, F8, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM) == cudaSuccess;
  if (splits > 1 && splits <= MAX_CLUSTER) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits);
    cfg.blockDim = dim3((CONSUMERS + 1) * 32);
    cfg.dynamicSmemBytes = T::SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    ok = ok && cudaOccupancyMaxActiveClusters(&n, attention_few_kernel<DH, F8, NG>, &cfg) == cudaSuccess;
    n *= splits;
  } else {
    ok = ok && cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess &&
         cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attention_few_kernel<DH, F8, NG>, (CONSUMERS + 1) * 32, T::SMEM) == cudaSuccess;
    n *= sms;
  }
  if (!ok) cudaGetLastError();
  return ok && n > 0 ? n : 1;
}

// Blocks that the current device holds at once of the kernel for so many rows of a KV head, with ranges in clusters where they
// are joined there (what plans ranges asks once per kind).
JLX_API int jlx_attention_few_places(int dh, int bits8, int rows, int splits) {
  if (dh == 128)
    return bits8 ? (rows <= 8 ? few_places<128, true, 1>(splits) : few_places<128, true, 2>(splits)) : (rows <= 8 ? few_places<128, false, 1>(splits) : few_places<128, false, 2>(splits));
  return bits8 ? (rows <= 8 ? few_places<64, true, 1>(splits) : few_places<64, true, 2>(splits)) : (rows <= 8 ? few_places<64, false, 1>(splits) : few_places<64, false, 2>(splits));
}

JLX_API int jlx_attention_few(const RowsArgs* a, cudaStream_t stream) {
  RowsParams P;
  if (rows_params(*a, P)) return 1;
  if (P.n_items == 0) return 0;
  const int rows = a->max_count * (P.Hq / P.Hkv), ng = rows <= 8 ? 1 : 2;
  const long long gx = (long long)P.n_items * P.splits, gy = (long long)P.Hkv * ((rows + 8 * ng - 1) / (8 * ng));
  JLX_REQUIRE(gx < (1ll << 31) && gy <= 65535, "attention over rows: too many items or rows");
  JLX_REQUIRE(P.splits <= MAX_CLUSTER || (P.part_o && P.part_ml), "attention over rows: scratch for the ranges is missing");
  const dim3 grid((unsigned)gx, (unsigned)gy);
  const bool f8 = P.scales != nullptr;
  int rc;
  if (a->dh == 128) rc = f8 ? (ng == 1 ? launch_few<128, true, 1>(P, grid, stream) : launch_few<128, true, 2>(P, grid, stream))
                            : (ng == 1 ? launch_few<128, false, 1>(P, grid, stream) : launch_few<128, false, 2>(P, grid, stream));
  else rc = f8 ? (ng == 1 ? launch_few<64, true, 1>(P, grid, stream) : launch_few<64, true, 2>(P, grid, stream))
               : (ng == 1 ? launch_few<64, false, 1>(P, grid, stream) : launch_few<64, false, 2>(P, grid, stream));
  if (rc) return rc;
  if (P.splits > MAX_CLUSTER) return a->dh == 128 ? launch_rows_join<128>(P, a->max_count, stream) : launch_rows_join<64>(P, a->max_count, stream);
  return 0;
}
