// Low-rank adapters of many requests at once beside a shared projection: every row n has an adapter e of its own (or none), and
//
//   out[n] = y[n] + scale_e (x[n] A_e^T) B_e^T,      A_e [r, K], B_e [No, r], x [N, K], y and out [N, No].
//
// The rows come sorted by adapter (`order`), cut into tiles of one adapter each (16 rows, or 64 where an adapter has more), so that an
// adapter's matrices are read once for a tile's rows.
//
// bfloat16 (adapters_kernel): a thread-block cluster serves a tile in one launch.  Its blocks cut K: each makes the products of
// its part of x and A on the tensor cores, a warp every WK-th 32 entries of K, and their sums meet in shared memory, first of the
// block's warps, then of the cluster's blocks (each adds up a share of the numbers and hands it to all).  Then the blocks
// cut No: each multiplies its part of B with the tile's rows of rank r and adds y.  All sums go in one order.
//
// It is bound by bytes: 2 r (K + No) operations a row against 2 K + 4 No bytes of rows and 2 r (K + No) of weights a tile.  So
// mma.sync, with B, and for tiles of 16 rows x and A, straight from memory into registers: the contraction index may run in any order
// that both operands share, and with entry 8 t + i of 32 as the thread's (t = lane % 4) every operand of two products is one load of
// 16 bytes.  Tiles of 64 rows have no registers for operands that are on their way: x and A come through shared memory, four stages
// deep (2048 rows of rank 64: 35 us for 52).  Columns of the second product are dealt to a unit of four tiles in the order that
// leaves a thread with eight neighbours of a row of y.
//
// The rows of rank r between both products are 32-bit sums, which the tensor cores take as two bfloat16 numbers (off by 2^-16 of
// each at most, far below the rounding of a bfloat16 output), or as three for 32-bit outputs (2^-24).
//
// Everything else (32-bit rows, K or No no multiple of 8, rows off 16-byte boundaries) takes two plain kernels with 32-bit sums, a
// thread per column of B: 300 float32 rows of rank 64, 1024 to 1024, 37 us; 675 bfloat16 rows of rank 70, 2051 to 2053, 70.
//
// Measured (B200, among others): one row of rank 16, 5120 to 7168, 13.1 us a call, 8.2 on the device, of which the launch is 2 and each
// phase one to two trips to memory; 64 rows of 24 adapters of ranks 16 to 64 22 us; 2048 rows of rank 64, 5120 to 5120, 33.5 us (2 TB/s).
// A cluster is as large as one round of blocks allows: 2048 rows with four blocks a tile 41 us, with eight 33.
#include <cooperative_groups.h>

#include "common.cuh"
#include "mbarrier.cuh"
#include "mma_sync.cuh"

namespace cg = cooperative_groups;

#define THREADS 256
#define WARPS (THREADS / 32)
#define MAX_RANK 256
#define MAX_CLUSTER 16  // (more than 8 blocks are not portable; this is sm_100a only)

struct AdapterArgs {  // _ADAPTER_ARGS in kernels/api.py
  const void *x, *a, *b, *y;
  void* out;
  const int* order;    // [M] rows, sorted by adapter
  const int* tiles;    // [n_tiles][3] = (adapter or -1, first in `order`, count)
  const float* scale;  // [E] or null: 1
  const int* ranks;    // [E] or null: r
  float* low;          // [M, r] scratch of the plain kernels
  long long ldx, ldy, ldo;
  int N, M, E, r, K, No, n_tiles, tile_rows, type, out_type;
};

struct AdapterTile {
  int e, first, count, rank;
};
// The part of tile i that begins at row `from` and holds `rows` at most; false: nothing to do.
__device__ __forceinline__ bool adapter_tile(const AdapterArgs& P, int i, int from, int rows, AdapterTile& t) {
  t.e = P.tiles[3 * i];
  t.first = P.tiles[3 * i + 1] + from;
  t.count = min(P.tiles[3 * i + 2] - from, rows);
  if (t.count <= 0 || t.first < 0 || t.first + t.count > P.M || t.e >= P.E) return false;
  if (t.e < 0 && P.out == P.y) return false;
  t.rank = t.e < 0 ? 0 : P.ranks ? min(max(P.ranks[t.e], 0), P.r) : P.r;
  return true;
}
__device__ __forceinline__ int adapter_row(const AdapterArgs& P, const AdapterTile& t, int i) {
  const int n = i < t.count ? P.order[t.first + i] : -1;
  return n < P.N ? n : -1;
}

// ------------------------------------------------------------------------------------ bfloat16
// The first n of eight entries (n <= 0: none).
__device__ __forceinline__ uint4 first_of(uint4 v, int n) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] &= n >= 2 * i + 2 ? 0xffffffffu : n == 2 * i + 1 ? 0xffffu : 0u;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// entries between rows of the shared arrays: rows fall on different banks
__host__ __device__ constexpr int low_stride(int rank_cols) { return rank_cols + 8; }

// A row of rank r (its parts `apart` entries from each other) times a row of B, in 32 bits.
template <int PARTS>
__device__ __forceinline__ float whole_entry(const bf16* l, int apart, const bf16* b, int rank) {
  float sum = 0.f;
#pragma unroll 1
  for (int k = 0; k < rank; ++k) {
    float v = 0.f;
#pragma unroll
    for (int p = PARTS - 1; p >= 0; --p) v += __bfloat162float(l[p * apart + k]);
    sum = fmaf(v, __bfloat162float(b[k]), sum);
  }
  return sum;
}

template <typename TY> struct Eight;
template <> struct Eight<bf16> {
  uint4 v;
  __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void add_store(bf16* p, const float* d) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    uint4 w;
    uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      u[i] = pack_bf16(f.x + d[2 * i], f.y + d[2 * i + 1]);
    }
    *reinterpret_cast<uint4*>(p) = w;
  }
  __device__ __forceinline__ void store(bf16* p) { *reinterpret_cast<uint4*>(p) = v; }
};
template <> struct Eight<float> {
  float4 v[2];
  __device__ __forceinline__ void load(const float* p) {
    v[0] = reinterpret_cast<const float4*>(p)[0];
    v[1] = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void add_store(float* p, const float* d) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(v[i].x + d[4 * i], v[i].y + d[4 * i + 1], v[i].z + d[4 * i + 2], v[i].w + d[4 * i + 3]);
  }
  __device__ __forceinline__ void store(float* p) {
    reinterpret_cast<float4*>(p)[0] = v[0];
    reinterpret_cast<float4*>(p)[1] = v[1];
  }
};

// Stages of x and A in shared memory.
template <int MT, int RC, int WK> struct Stage {
  static constexpr int SUBS = WK > 4 ? WK / 4 : 1, K = 64 * SUBS;
  static constexpr int X_CHUNKS = SUBS * MT * 16 * 8, A_CHUNKS = SUBS * RC * 8;
  static constexpr int X_BYTES = X_CHUNKS * 16, BYTES = X_BYTES + A_CHUNKS * 16, STAGES = 4;
};

// MT: tiles of 16 rows.  NT: tiles of 8 ranks that a warp has; the block's warps are WR groups of them (WR * NT * 8 >= r) times
// WK cuts of K.  PARTS: bfloat16 numbers that a 32-bit sum between the products becomes.
template <int MT, int NT, int WR, typename TY>
__global__ void __launch_bounds__(THREADS, WR * NT * 8 > 128 ? 1 : 2) adapters_kernel(const AdapterArgs P) {
  JLX_TL(TL_OTHER);
  constexpr int ROWS = 16 * MT, WK = WARPS / WR, RC = WR * NT * 8, LD = low_stride(RC);
  constexpr int PARTS = sizeof(TY) == 4 ? 3 : 2;
  constexpr int STEPS = (RC + 31) / 32;  // of 32 ranks in the second product (the last one may be short)
  constexpr bool EARLY = MT == 1 && STEPS == 1;  // room in registers for what the next 32 columns need
  extern __shared__ __align__(128) uint8_t smem_raw[];
  float* meet = reinterpret_cast<float*>(smem_raw);                  // [max(WK / 2, 1)][ROWS][RC]: the warps' sums; then [ROWS][RC] of the block
  bf16* low = reinterpret_cast<bf16*>(meet + (WK > 1 ? WK / 2 : 1) * ROWS * RC);  // [PARTS][ROWS][LD]
  __shared__ int row_s[ROWS];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), me = cluster.block_rank();
  const int subs = (P.tile_rows + ROWS - 1) / ROWS, tile = blockIdx.y / subs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  if (MT == 1) pdl_launch_dependents_if_small();  // (a successor that waits beside the blocks of many rows costs them half their speed: 50 us for 33)
  pdl_wait();
  AdapterTile t;
  if (!adapter_tile(P, tile, (blockIdx.y - tile * subs) * ROWS, ROWS, t)) return;  // (the whole cluster)
  if (tid < ROWS) row_s[tid] = adapter_row(P, t, tid);
  __syncthreads();
  const bf16 *x = reinterpret_cast<const bf16*>(P.x), *a = reinterpret_cast<const bf16*>(P.a), *b = reinterpret_cast<const bf16*>(P.b);
  const TY* y = reinterpret_cast<const TY*>(P.y);
  TY* out = reinterpret_cast<TY*>(P.out);

  // what a warp takes of B (and, of few rows, of y) for 32 columns
  const int units = (P.No + 31) / 32, per_u = (units + blocks - 1) / blocks, u0 = me * per_u, u1 = min(u0 + per_u, units);
  const int col_g = (g >> 1) * 8 + (g & 1);
  struct B {
    uint4 b[STEPS][4];
    Eight<TY> y[EARLY ? 2 : 1];
  };
  B first;
  auto fetch_b = [&](int u, B& f) {
    if (u >= u1) return;
    if (t.e >= 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = u * 32 + col_g + j * 2;
        const bf16* br = b + ((size_t)t.e * P.No + n) * P.r;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const int k = s * 32 + t4 * 8;
          if (P.r & 7) {  // rows of B off 16-byte boundaries: entry by entry
            const int left = n < P.No ? t.rank - k : 0;
            const uint16_t* e = reinterpret_cast<const uint16_t*>(br + k);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (2 * i < left ? e[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)e[2 * i + 1] << 16 : 0u);
            f.b[s][j] = make_uint4(w[0], w[1], w[2], w[3]);
            continue;
          }
          f.b[s][j] = n < P.No && k < t.rank ? *reinterpret_cast<const uint4*>(br + k) : make_uint4(0, 0, 0, 0);
          if (t.rank & 7) f.b[s][j] = first_of(f.b[s][j], t.rank - k);
        }
      }
    }
    if (EARLY) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = row_s[h * 8 + g], col = u * 32 + t4 * 8;
        if (n >= 0 && col < P.No) f.y[h].load(y + (size_t)n * P.ldy + col);
      }
    }
  };

  if (t.e >= 0) {
    // ---- x A^T over this block's part of K
    const int wr = warp % WR, wk = warp / WR;
    const int chunks = (P.K + 31) / 32, per = (chunks + blocks - 1) / blocks, c0 = me * per, c1 = min(c0 + per, chunks);
    float acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
    const bf16* xr[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = row_s[m * 16 + h * 8 + g];
        xr[m][h] = n >= 0 ? x + (size_t)n * P.ldx + t4 * 8 : nullptr;
      }
    const int rank0 = wr * NT * 8 + g;
    const bf16* ar = a + ((size_t)t.e * P.r + rank0) * P.K + t4 * 8;
    struct Step {
      uint4 x[MT][2], a[NT];
    };
    auto fetch = [&](int c, Step& f) {
      const int k = c * 32;
      const bool in = c < c1 && k + t4 * 8 < P.K;
#pragma unroll
      for (int n = 0; n < NT; ++n) f.a[n] = in && rank0 + n * 8 < t.rank ? *reinterpret_cast<const uint4*>(ar + (size_t)n * 8 * P.K + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) f.x[m][h] = in && xr[m][h] ? *reinterpret_cast<const uint4*>(xr[m][h] + k) : make_uint4(0, 0, 0, 0);
    };
    auto multiply = [&](const Step& f) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint32_t f0[4] = {f.x[m][0].x, f.x[m][1].x, f.x[m][0].y, f.x[m][1].y}, f1[4] = {f.x[m][0].z, f.x[m][1].z, f.x[m][0].w, f.x[m][1].w};
          mma_bf16(acc[m][n], f0, f.a[n].x, f.a[n].y);
          mma_bf16(acc[m][n], f1, f.a[n].z, f.a[n].w);
        }
    };
    if (MT == 1 && NT <= 4) {  // a step's operands are on their way while the one before is worked on
      Step even, odd;
      fetch(c0 + wk, even);
#pragma unroll 1
      for (int c = c0 + wk; c < c1; c += 2 * WK) {
        fetch(c + WK, odd);
        multiply(even);
        fetch(c + 2 * WK, even);
        multiply(odd);
      }
    } else if (MT == 1) {
#pragma unroll 1
      for (int c = c0 + wk; c < c1; c += WK) {
        Step f;
        fetch(c, f);
        multiply(f);
      }
    } else {
      // Many rows: registers hold the sums, and no second step's operands; so both come through shared memory, STAGES - 1 stages ahead.  A
      // stage has SUBS times 64 of K, in rows of 128 bytes whose chunks of 16 are swizzled; a warp has every WK-th 16 of K.
      using S = Stage<MT, RC, WK>;
      const int k_begin = c0 * 32, k_end = min(c1 * 32, P.K), stages = (k_end - k_begin + S::K - 1) / S::K;
      const uint32_t ring = smem_u32(smem_raw);
      auto ask = [&](int st) {
        const uint32_t to = ring + (st % S::STAGES) * S::BYTES;
        const int k0 = k_begin + st * S::K;
#pragma unroll
        for (int i = 0; i < S::X_CHUNKS / THREADS; ++i) {
          const int q = i * THREADS + tid, sub = q / (ROWS * 8), row = q / 8 % ROWS, c = q & 7, k = k0 + sub * 64 + c * 8, n = row_s[row];
          const bool in = n >= 0 && k < k_end;
          cp_async16(to + (sub * ROWS + row) * 128 + ((c ^ (row & 7)) << 4), in ? x + (size_t)n * P.ldx + k : x, in);
        }
#pragma unroll
        for (int i = 0; i < (S::A_CHUNKS + THREADS - 1) / THREADS; ++i) {
          const int q = i * THREADS + tid, sub = q / (RC * 8), row = q / 8 % RC, c = q & 7, k = k0 + sub * 64 + c * 8;
          const bool in = row < t.rank && k < k_end;
          if (S::A_CHUNKS % THREADS == 0 || q < S::A_CHUNKS)
            cp_async16(to + S::X_BYTES + (sub * RC + row) * 128 + ((c ^ (row & 7)) << 4), in ? a + ((size_t)t.e * P.r + row) * P.K + k : a, in);
        }
      };
#pragma unroll
      for (int st = 0; st < S::STAGES - 1; ++st) {
        if (st < stages) ask(st);
        cp_async_commit();
      }
#pragma unroll 1
      for (int st = 0; st < stages; ++st) {
        cp_async_wait<S::STAGES - 2>();
        __syncthreads();  // (the stage has come, and the one before has been read by all)
        if (st + S::STAGES - 1 < stages) ask(st + S::STAGES - 1);
        cp_async_commit();
        const uint32_t from = ring + (st % S::STAGES) * S::BYTES;
#pragma unroll
        for (int z = 0; z < S::K / 16; z += WK) {
          const int step = z + wk, sub = step >> 2, c = (step & 3) * 2;  // its two chunks of a row
          uint32_t bf_[NT][2];
#pragma unroll
          for (int n = 0; n < NT; n += 2) {  // two tiles of 8 ranks (one: the other lanes' addresses are not used)
            const int row = (wr * NT + n) * 8 + (lane & 7) + (NT > 1 ? (lane >> 4) * 8 : 0), ch = c + (lane >> 3 & 1);
            uint32_t r0, r1, r2, r3;
            ldmatrix_x4(from + S::X_BYTES + (sub * RC + row) * 128 + ((ch ^ (row & 7)) << 4), r0, r1, r2, r3);
            bf_[n][0] = r0; bf_[n][1] = r1;
            if (NT > 1) { bf_[(n + 1) % NT][0] = r2; bf_[(n + 1) % NT][1] = r3; }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const int row = m * 16 + (lane & 15), ch = c + (lane >> 4);
            uint32_t f[4];
            ldmatrix_x4(from + (sub * ROWS + row) * 128 + ((ch ^ (row & 7)) << 4), f[0], f[1], f[2], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_bf16(acc[m][n], f, bf_[n][0], bf_[n][1]);
          }
        }
      }
      cp_async_wait<0>();
      __syncthreads();  // (the ring's memory is the sums' now)
    }
    if (EARLY) fetch_b(u0 + warp, first);  // (B's first part is on its way while the sums meet)
    // ---- the warps' sums, halved until one is left
    auto put = [&](float* to, bool add) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float2* p = reinterpret_cast<float2*>(to + (m * 16 + h * 8 + g) * RC + wr * NT * 8 + n * 8 + t4 * 2);
            if (add) {
              acc[m][n][2 * h] += p->x;
              acc[m][n][2 * h + 1] += p->y;
            } else {
              *p = make_float2(acc[m][n][2 * h], acc[m][n][2 * h + 1]);
            }
          }
    };
#pragma unroll
    for (int half = WK / 2; half > 0; half >>= 1) {
      if (wk >= half && wk < 2 * half) put(meet + (wk - half) * ROWS * RC, false);
      __syncthreads();
      if (wk < half) put(meet + wk * ROWS * RC, true);
      __syncthreads();
    }
    if (wk == 0) put(meet, false);
    cluster.sync();
    // ---- the blocks': each adds up a share and hands it to all
    const float s = P.scale ? P.scale[t.e] : 1.f;
    const int share = (ROWS * RC / 4 + blocks - 1) / blocks;
    for (int i = me * share + tid; i < min((me + 1) * share, ROWS * RC / 4); i += THREADS) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int q0 = 0; q0 < MAX_CLUSTER; q0 += 8) {
        if (q0 >= blocks) break;
        float4 w[8];  // (asked for together: each takes a trip to another multiprocessor)
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q] = q0 + q < blocks ? reinterpret_cast<const float4*>(cluster.map_shared_rank(meet, q0 + q))[i] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          v.x += w[q].x; v.y += w[q].y; v.z += w[q].z; v.w += w[q].w;
        }
      }
      float f[4] = {v.x * s, v.y * s, v.z * s, v.w * s};
      const int row = i * 4 / RC, col = i * 4 % RC;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        uint2 w = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float2 o = __bfloat1622float2(h[u]);
          f[2 * u] = isinf(o.x) ? 0.f : f[2 * u] - o.x;
          f[2 * u + 1] = isinf(o.y) ? 0.f : f[2 * u + 1] - o.y;
        }
        for (int q = 0; q < blocks; ++q) *reinterpret_cast<uint2*>(cluster.map_shared_rank(low, q) + ((size_t)p * ROWS + row) * LD + col) = w;
      }
    }
    cluster.sync();
  }

  // ---- the tile's rows times B^T, over this block's part of the columns, 32 at a time
  if (!EARLY || t.e < 0) fetch_b(u0 + warp, first);
#pragma unroll 1
  for (int u = u0 + warp; u < u1; u += WARPS) {
    const int col = u * 32 + t4 * 8;  // this thread's eight columns
    const bool mine = col < P.No;
    const B now = first;
    if (EARLY) fetch_b(u + WARPS, first);
    constexpr int TOGETHER = sizeof(TY) == 4 && MT > 2 ? 2 : MT;  // tiles of rows whose y is asked for together
    Eight<TY> yt[TOGETHER][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (!EARLY && m % TOGETHER == 0) {
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = mine ? row_s[(m + i) * 16 + h * 8 + g] : -1;
            if (row >= 0) yt[i][h].load(y + (size_t)row * P.ldy + col);
          }
      }
      Eight<TY> ys[2];
      int n[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        n[h] = mine ? row_s[m * 16 + h * 8 + g] : -1;
        ys[h] = EARLY ? now.y[h] : yt[m % TOGETHER][h];
      }
      if (t.e < 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (n[h] >= 0) ys[h].store(out + (size_t)n[h] * P.ldo + col);
        continue;
      }
      float d[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j][0] = d[j][1] = d[j][2] = d[j][3] = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p) {  // small parts first
          uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
          if (RC % 32 == 0 || s * 32 + t4 * 8 < RC) {
            const bf16* l = low + ((size_t)p * ROWS + m * 16 + g) * LD + s * 32 + t4 * 8;
            lo = *reinterpret_cast<const uint4*>(l);
            hi = *reinterpret_cast<const uint4*>(l + 8 * LD);
          }
          const uint32_t f0[4] = {lo.x, hi.x, lo.y, hi.y}, f1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma_bf16(d[j], f0, now.b[s][j].x, now.b[s][j].y);
            mma_bf16(d[j], f1, now.b[s][j].z, now.b[s][j].w);
          }
        }
      }
      // Against an infinite entry of B the small part of a number, 0 or of the other sign, makes NaN of an infinity, and so does an
      // infinite row against the zeros that fill up an adapter's ranks: sums that are not finite are made again of whole numbers, over the
      // adapter's own ranks.
      float4 total = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        total.x += d[j][0]; total.y += d[j][1]; total.z += d[j][2]; total.w += d[j][3];
      }
      if (!isfinite((total.x + total.y) + (total.z + total.w)) && mine) {
#pragma unroll 1
        for (int x = 0; x < 16; ++x) {  // (x = 4 j + i of d[j][i])
          const float whole = whole_entry<PARTS>(low + (m * 16 + (x >> 1 & 1) * 8 + g) * LD, ROWS * LD, b + ((size_t)t.e * P.No + col + (x >> 2) * 2 + (x & 1)) * P.r, t.rank);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (x == 4 * j + i && !isfinite(d[j][i])) d[j][i] = whole;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float f[8] = {d[0][2 * h], d[0][2 * h + 1], d[1][2 * h], d[1][2 * h + 1], d[2][2 * h], d[2][2 * h + 1], d[3][2 * h], d[3][2 * h + 1]};
        if (n[h] >= 0) ys[h].add_store(out + (size_t)n[h] * P.ldo + col, f);
      }
    }
    if (!EARLY) fetch_b(u + WARPS, first);
  }
}

// --------------------------------------------------------------------------- any type and alignment
#define PLAIN_ROWS 8
#define PLAIN_RANKS 4

// low[i, j] = scale x A^T for PLAIN_ROWS rows of a tile and PLAIN_RANKS ranks a block; its threads cut K.
template <typename T>
__global__ void __launch_bounds__(THREADS) adapters_low_kernel(const AdapterArgs P) {
  JLX_TL(TL_OTHER);
  __shared__ float part[WARPS][PLAIN_ROWS * PLAIN_RANKS];
  const int subs = (P.tile_rows + PLAIN_ROWS - 1) / PLAIN_ROWS, tile = blockIdx.y / subs, j0 = blockIdx.x * PLAIN_RANKS;
  AdapterTile t;
  if (!adapter_tile(P, tile, (blockIdx.y - tile * subs) * PLAIN_ROWS, PLAIN_ROWS, t) || t.e < 0) return;
  const T *x = reinterpret_cast<const T*>(P.x), *a = reinterpret_cast<const T*>(P.a) + ((size_t)t.e * P.r + j0) * P.K;
  const T* xr[PLAIN_ROWS];
#pragma unroll
  for (int i = 0; i < PLAIN_ROWS; ++i) {
    const int n = adapter_row(P, t, min(i, t.count - 1));
    xr[i] = x + (size_t)max(n, 0) * P.ldx;
  }
  float acc[PLAIN_ROWS][PLAIN_RANKS] = {};
#pragma unroll 2
  for (int k = threadIdx.x; k < P.K; k += THREADS) {
    float xv[PLAIN_ROWS], av[PLAIN_RANKS];
#pragma unroll
    for (int i = 0; i < PLAIN_ROWS; ++i) xv[i] = to_f32<T>(xr[i][k]);
#pragma unroll
    for (int j = 0; j < PLAIN_RANKS; ++j) av[j] = j0 + j < t.rank ? to_f32<T>(a[(size_t)j * P.K + k]) : 0.f;
#pragma unroll
    for (int i = 0; i < PLAIN_ROWS; ++i)
#pragma unroll
      for (int j = 0; j < PLAIN_RANKS; ++j) acc[i][j] = fmaf(xv[i], av[j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < PLAIN_ROWS; ++i)
#pragma unroll
    for (int j = 0; j < PLAIN_RANKS; ++j) {
      const float v = warp_sum(acc[i][j]);
      if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][i * PLAIN_RANKS + j] = v;
    }
  __syncthreads();
  const int i = threadIdx.x / PLAIN_RANKS, j = threadIdx.x % PLAIN_RANKS;
  if (i < t.count && i < PLAIN_ROWS && j0 + j < P.r) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += part[w][threadIdx.x];
    P.low[(size_t)(t.first + i) * P.r + j0 + j] = v * (P.scale ? P.scale[t.e] : 1.f);
  }
}

// out = y + low B^T: a thread per column, PLAIN_ROWS rows.
template <typename T, typename TY>
__global__ void __launch_bounds__(THREADS) adapters_out_kernel(const AdapterArgs P) {
  JLX_TL(TL_OTHER);
  __shared__ __align__(16) float low[MAX_RANK][PLAIN_ROWS];
  const int subs = (P.tile_rows + PLAIN_ROWS - 1) / PLAIN_ROWS, tile = blockIdx.y / subs;
  AdapterTile t;
  if (!adapter_tile(P, tile, (blockIdx.y - tile * subs) * PLAIN_ROWS, PLAIN_ROWS, t)) return;
  if (t.e >= 0)
    for (int i = threadIdx.x; i < PLAIN_ROWS * t.rank; i += THREADS) low[i % t.rank][i / t.rank] = i / t.rank < t.count ? P.low[(size_t)(t.first + i / t.rank) * P.r + i % t.rank] : 0.f;
  __syncthreads();
  const int n = blockIdx.x * THREADS + threadIdx.x;
  if (n >= P.No) return;
  float acc[PLAIN_ROWS] = {};
  const T* b = reinterpret_cast<const T*>(P.b) + ((size_t)max(t.e, 0) * P.No + n) * P.r;
#pragma unroll 4
  for (int j = 0; j < t.rank; ++j) {
    const float w = to_f32<T>(b[j]);
#pragma unroll
    for (int i = 0; i < PLAIN_ROWS; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(&low[j][i]);
      acc[i] = fmaf(v.x, w, acc[i]);
      acc[i + 1] = fmaf(v.y, w, acc[i + 1]);
      acc[i + 2] = fmaf(v.z, w, acc[i + 2]);
      acc[i + 3] = fmaf(v.w, w, acc[i + 3]);
    }
  }
#pragma unroll
  for (int i = 0; i < PLAIN_ROWS; ++i) {
    const int row = adapter_row(P, t, i);
    if (row < 0) continue;
    const TY v = reinterpret_cast<const TY*>(P.y)[(size_t)row * P.ldy + n];
    reinterpret_cast<TY*>(P.out)[(size_t)row * P.ldo + n] = t.e < 0 ? v : from_f32<TY>(to_f32<TY>(v) + acc[i]);
  }
}

// -------------------------------------------------------------------------------------------- host
template <int MT, int NT, int WR, typename TY>
static int launch_adapters(const AdapterArgs& P, int cluster, cudaStream_t stream) {
  constexpr int ROWS = 16 * MT, WK = WARPS / WR, RC = WR * NT * 8, PARTS = sizeof(TY) == 4 ? 3 : 2;
  using S = Stage<MT, RC, WK>;
  constexpr size_t sums = (size_t)(WK > 1 ? WK / 2 : 1) * ROWS * RC * 4 + (size_t)PARTS * ROWS * low_stride(RC) * 2, ring = MT > 1 ? S::STAGES * S::BYTES : 0;
  constexpr size_t smem = sums > ring ? sums : ring;
  auto kernel = adapters_kernel<MT, NT, WR, TY>;
  static_assert(smem <= 227 * 1024, "a tile's sums do not fit into shared memory");
  if (smem > 48 * 1024) JLX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  if (cluster > 8) JLX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  const int subs = (P.tile_rows + ROWS - 1) / ROWS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster, P.n_tiles * subs);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  JLX_CUDA(cudaLaunchKernelEx(&cfg, kernel, P));
  return 0;
}

template <int MT, typename TY>
static int launch_rank(const AdapterArgs& P, int cluster, cudaStream_t stream) {
  if (P.r <= 8) return launch_adapters<MT, 1, 1, TY>(P, cluster, stream);
  if (P.r <= 16) return launch_adapters<MT, 2, 1, TY>(P, cluster, stream);
  if (P.r <= 32) return launch_adapters<MT, 4, 1, TY>(P, cluster, stream);
  if (P.r <= 64) return launch_adapters<MT, 4, 2, TY>(P, cluster, stream);
  if (P.r <= 128) return launch_adapters<MT, 4, 4, TY>(P, cluster, stream);
  return launch_adapters<MT == 4 ? 2 : MT, 8, 4, TY>(P, cluster, stream);
}

static bool rows_on_16(const void* p, long long ld, int size) { return ((uintptr_t)p & 15) == 0 && ld * size % 16 == 0; }

// Whether the call takes the one-launch kernel (else the plain ones, which need `low`: kernels/api.py has the same rule).
static bool adapters_fast(const AdapterArgs& a) {
  const int size = a.out_type == JLX_F32 ? 4 : 2;
  return a.type == JLX_BF16 && a.K % 8 == 0 && a.No % 8 == 0 && rows_on_16(a.x, a.ldx, 2) && rows_on_16(a.a, 8, 2) && rows_on_16(a.b, 8, 2) && rows_on_16(a.y, a.ldy, size) &&
         rows_on_16(a.out, a.ldo, size);
}

JLX_API int jlx_adapters(const AdapterArgs* args, int sms, void* stream_) {
  const AdapterArgs& P = *args;
  cudaStream_t stream = (cudaStream_t)stream_;
  JLX_REQUIRE(P.N > 0 && P.M > 0 && P.E > 0 && P.r > 0 && P.r <= MAX_RANK && P.K > 0 && P.No > 0, "adapters: bad sizes");
  JLX_REQUIRE(P.n_tiles > 0 && (P.tile_rows == 16 || P.tile_rows == 64), "adapters: %d tiles of %d rows", P.n_tiles, P.tile_rows);
  JLX_REQUIRE((long long)P.n_tiles * (P.tile_rows / PLAIN_ROWS) <= 65535, "adapters: too many tiles (%d)", P.n_tiles);
  if (adapters_fast(P)) {
    // One round of blocks: two a multiprocessor, of ranks over 128 one.  (2048 rows of rank 256 of 20 requests: 246 us where two were
    // counted, 177; 1024 of three adapters 132 and 88.)
    const int rows = P.tile_rows == 16 ? 16 : P.r <= 128 ? 64 : 32, units = P.n_tiles * (P.tile_rows / rows);
    int cluster = MAX_CLUSTER;
    while (cluster > 1 && units * cluster > (P.r > 128 ? 1 : 2) * sms) cluster /= 2;
    if (P.out_type == JLX_F32) return P.tile_rows == 16 ? launch_rank<1, float>(P, cluster, stream) : launch_rank<4, float>(P, cluster, stream);
    return P.tile_rows == 16 ? launch_rank<1, bf16>(P, cluster, stream) : launch_rank<4, bf16>(P, cluster, stream);
  }
  JLX_REQUIRE(P.low != nullptr, "adapters: scratch is needed");
  const unsigned groups = (unsigned)(P.n_tiles * (P.tile_rows / PLAIN_ROWS));
  const dim3 low_grid((P.r + PLAIN_RANKS - 1) / PLAIN_RANKS, groups), out_grid((P.No + THREADS - 1) / THREADS, groups);
  JLX_DISPATCH_DTYPE(P.type, T, {
    adapters_low_kernel<T><<<low_grid, THREADS, 0, stream>>>(P);
    JLX_LAUNCH_CHECK("adapters_low");
    if (P.out_type == JLX_F32) adapters_out_kernel<T, float><<<out_grid, THREADS, 0, stream>>>(P);
    else adapters_out_kernel<T, bf16><<<out_grid, THREADS, 0, stream>>>(P);
  });
  JLX_LAUNCH_CHECK("adapters_out");
  return 0;
}
