// A paged cache kept to a budget: which places a request and KV head keep (kv_choose), and moving the kept rows of keys and values to the
// front of the request's pages or of other pages (kv_compact).
//
// kv_choose, of a request's L places and n = min(keep, L): the last `recent` ones, then the first `first` ones, as far as n goes, then of the
// rest those with the largest sums; ties go to the lowest place; NaN counts as the lowest sum, -0 as 0.  Places come in ascending
// order.  A sum becomes a whole number of 32 bits with the same order, places that are kept in any case the largest one; the bits of the
// smallest kept one are found eight at a time by counting (a digit's count of the places that share the digits before it), until few enough
// places share them that each can be compared with all; then the places above it, and the first so many that equal it, are
// counted and written, a warp going through a stretch of them by votes.  A cluster of blocks serves a request and KV head, each with
// a stretch of the places in registers: the sums are read once.
//
// kv_compact moves rows bit for bit.  Into other pages every row is on its own.  In place, row i's new place is at or before its old
// one: a block takes a column of 32 bytes of one plane's rows through all places in order, 1024 at a time (2048 where rows are no
// multiple of 32 bytes and the column has 16), all loads of which precede all stores; a later row's source lies behind what has been written.
//
// Both are bound by bytes, few in the first, so there by the chain of its passes: 100,001 places of one session, 4096 kept, 18.9 us a call;
// 64 sessions of up to 8192, 2048 kept, 25.5 us (62 with sums in shared memory and a scan of the block for every 512 places; digits of 11
// bits: 40).  Moving 2048 rows of 8 heads of 128 each of 32 sessions takes 94 us, 5.8 TB/s;
// in place 185: every block of a column looks up each row's place and pages for 32 bytes of it.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

#define THREADS 512
#define WARPS (THREADS / 32)
#define MAX_CLUSTER 16
#define BINS 256
#define FEW 64  // places that are compared with each other
#define MAX_KEYS 16  // sums that a thread keeps at most

struct ChooseArgs {  // _CHOOSE_ARGS in kernels/api.py
  const float* sums;   // [R, H, width]
  const int* lengths;  // [R]
  const int* keep;     // [R]
  int* places;         // [R, H, most]
  int* counts;         // [R]
  int* status;
  int R, H, width, most, first, recent;
};

// Larger numbers for larger sums, from 0x7fffff (-infinity) to 0xff800000 (infinity).
#define KEY_NONE 0u  // no place
#define KEY_NAN 1u
#define KEY_ANY 0xffffffffu  // kept in any case
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return KEY_NAN;
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// per: places of a block.  KEYS: sums of a thread, its warp's stretch 32 by 32 (0: they are read again from memory in every pass).
template <int KEYS>
__global__ void __launch_bounds__(THREADS, 2) kv_choose_kernel(const ChooseArgs P, int per) {
  JLX_TL(TL_OTHER);
  __shared__ int bins[2][BINS];  // from the largest digit on
  __shared__ uint32_t mine_few[FEW], few[FEW], found_edge;
  __shared__ int warp_sums[WARPS], found[3], n_few, warp_kept[2][WARPS], mine[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), me = cluster.block_rank(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int row = blockIdx.y, r = row / P.H;
  int L = P.lengths[r], n = P.keep[r];
  if (L < 0 || L > P.width || n < 0 || min(n, L) > P.most) {
    if (tid == 0) atomicOr(P.status, JLX_STATUS_BAD_LENGTH);
    L = min(max(L, 0), P.width);
  }
  n = min(min(max(n, 0), L), P.most);
  const int recent = min(P.recent, n), first = min(P.first, n - recent);
  if (me == 0 && tid == 0 && row == r * P.H) P.counts[r] = n;
  const float* sums = P.sums + (size_t)row * P.width;
  int* places = P.places + (size_t)row * P.most;
  for (int i = n + me * THREADS + tid; i < P.most; i += blocks * THREADS) places[i] = -1;
  // this block's places, and of them a warp's
  const int p1 = min((me + 1) * per, L), stretch = (per + 32 * WARPS - 1) / (32 * WARPS) * 32;
  const int w0 = min(me * per + warp * stretch, p1), w1 = min(w0 + stretch, p1);
  auto look = [&](int i) {
    const int p = w0 + i * 32 + lane;
    if (p >= w1) return KEY_NONE;
    return p < first || p >= L - recent ? KEY_ANY : ordered(sums[p]);
  };
  uint32_t held[KEYS > 0 ? KEYS : 1];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) held[i] = look(i);
  const int steps = KEYS > 0 ? KEYS : stretch / 32;
  auto key = [&](int i) { return KEYS > 0 ? held[KEYS > 0 ? i : 0] : look(i); };
  // the smallest one that is kept, and how many of the places with just that one
  uint32_t edge = KEY_NONE, mask = 0u;
  int left = 0;
  if (n > 0 && n < L) {
    left = n;
    for (int shift = 24, half = 0;; shift -= 8, half ^= 1) {
      if (tid < BINS) bins[half][tid] = 0;
      if (tid == 0) n_few = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < steps; ++i) {
        const uint32_t k = key(i);
        if (k != KEY_NONE && (k & mask) == edge) atomicAdd(&bins[half][~k >> shift & 255], 1);
      }
      if (blocks > 1) cluster.sync();  // (the counts of the digit before last have been read everywhere, too)
      else __syncthreads();
      if (tid < BINS) {  // a digit a thread
        int c = 0;
        if (blocks > 1) {
#pragma unroll
          for (int q0 = 0; q0 < MAX_CLUSTER; q0 += 8) {
            if (q0 >= blocks) break;
            int v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = q0 + q < blocks ? *cluster.map_shared_rank(&bins[half][tid], q0 + q) : 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) c += v[q];
          }
        } else {
          c = bins[half][tid];
        }
        int above = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, above, o);
          if (lane >= o) above += y;
        }
        if (lane == 31) warp_sums[warp] = above;
        asm volatile("bar.sync 1, %0;" ::"n"(BINS) : "memory");
        above += __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0) - c;  // places with a larger digit
        if (above < left && above + c >= left) {
          found[0] = 255 - tid;
          found[1] = left - above;
          found[2] = c;
        }
      }
      __syncthreads();
      edge |= (uint32_t)found[0] << shift;
      mask |= 255u << shift;
      left = found[1];
      const int share = found[2];  // places that share the digits up to here
      if (shift == 0) break;       // (all digits: they are equal)
      if (share <= FEW) {
#pragma unroll
        for (int i = 0; i < steps; ++i) {
          const uint32_t k = key(i);
          if (k != KEY_NONE && (k & mask) == edge) mine_few[atomicAdd(&n_few, 1)] = k;
        }
        if (blocks > 1) {
          cluster.sync();
          int n_q = lane < blocks ? *cluster.map_shared_rank(&n_few, lane) : 0, at = n_q;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += y;
          }
          if (warp < blocks) {  // a warp fetches a block's
            const int count = __shfl_sync(0xffffffffu, n_q, warp), to = __shfl_sync(0xffffffffu, at, warp) - count;
            const uint32_t* from = cluster.map_shared_rank(mine_few, warp);
            for (int i = lane; i < count; i += 32) few[to + i] = from[i];
          }
        }
        __syncthreads();
        if (tid < share) {
          const uint32_t* all = blocks > 1 ? few : mine_few;
          const uint32_t k = all[tid];
          int more = 0, same = 0;
          for (int i = 0; i < share; ++i) {
            more += all[i] > k;
            same += all[i] == k;
          }
          if (more < left && more + same >= left) {  // (whoever has that sum writes the same)
            found_edge = k;
            found[0] = left - more;
          }
        }
        __syncthreads();
        edge = found_edge;
        left = found[0];
        break;
      }
    }
  }
  // ---- how many of the warp's places are above the edge, and how many equal it.  (Without an edge all places are above it, or none is kept.)
  if (n == 0) edge = KEY_ANY;
  int kept = 0, equal = 0;
#pragma unroll
  for (int i = 0; i < steps; ++i) {
    const uint32_t k = key(i);
    kept += k > edge;
    equal += k == edge;
  }
  kept = __reduce_add_sync(0xffffffffu, kept);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) {
    warp_kept[0][warp] = kept;
    warp_kept[1][warp] = equal;
  }
  __syncthreads();
  int at = 0, before = 0;  // kept places, and places equal to the edge, before the warp's: first of the block
  if (blocks > 1) {
    if (tid < 32) {
      const int a = __reduce_add_sync(0xffffffffu, lane < WARPS ? warp_kept[0][lane] : 0), e = __reduce_add_sync(0xffffffffu, lane < WARPS ? warp_kept[1][lane] : 0);
      if (lane == 0) {
        mine[0] = a;
        mine[1] = e;
      }
    }
    cluster.sync();
    const int a = lane < me ? *cluster.map_shared_rank(&mine[0], lane) : 0, e = lane < me ? *cluster.map_shared_rank(&mine[1], lane) : 0;
    at = __reduce_add_sync(0xffffffffu, a);
    before = __reduce_add_sync(0xffffffffu, e);
    cluster.barrier_arrive();  // (a block's shared memory stays until the others have read it)
  }
  at += __reduce_add_sync(0xffffffffu, lane < warp ? warp_kept[0][lane] : 0);
  before += __reduce_add_sync(0xffffffffu, lane < warp ? warp_kept[1][lane] : 0);
  at += min(before, left);  // (of those that equal it the first so many are kept)
  // ---- in order
  const uint32_t below = (1u << lane) - 1;
#pragma unroll
  for (int i = 0; i < steps; ++i) {
    const uint32_t k = key(i);
    bool take = k > edge;
    if (before < left) {  // (the warp's: some that equal it are still to be kept)
      const uint32_t same = __ballot_sync(0xffffffffu, k == edge);
      take |= k == edge && before + __popc(same & below) < left;
      before += __popc(same);
    }
    const uint32_t keep = __ballot_sync(0xffffffffu, take);
    if (take) places[at + __popc(keep & below)] = w0 + i * 32 + lane;
    at += __popc(keep);
  }
  if (blocks > 1) cluster.barrier_wait();
}

// -------------------------------------------------------------------------------------------- moving
struct CompactArgs {  // _COMPACT_ARGS in kernels/api.py
  uint8_t* pages;         // [P, 2, H, page, row_bytes]
  uint8_t* scales;        // [P, 2, H, page] or null
  const int* table;       // [R, table_width] where the rows are
  const int* into;        // [R, into_width] where they go
  const int* places;      // [R, H, most]
  const int* counts;      // [R]
  const float* sums;      // [R, H, width] or null
  float* sums_out;        // [R, H, out_width]
  int* status;
  int R, H, page, num_pages, row_bytes, table_width, into_width, most, width, out_width;
};

// The flat row of a place's key (values H * page further), or -1.
__device__ __forceinline__ int compact_row(const CompactArgs& P, const int* table, int width, int h, int place) {
  const int pi = place < 0 ? width : place / P.page;
  const int page = pi < width ? table[pi] : -1;
  return page >= 0 && page < P.num_pages ? (page * 2 * P.H + h) * P.page + (place - pi * P.page) : -1;
}
// Where row i of head h comes from and goes to; false (and the status): a page is missing, or (in place) the row would move back.
__device__ __forceinline__ bool compact_move(const CompactArgs& P, int r, int h, int i, bool in_place, int& src, int& dst) {
  const int place = P.places[((size_t)r * P.H + h) * P.most + i];
  src = compact_row(P, P.table + (size_t)r * P.table_width, P.table_width, h, place);
  dst = compact_row(P, P.into + (size_t)r * P.into_width, P.into_width, h, i);
  if (src < 0 || dst < 0 || (in_place && place < i)) {
    atomicOr(P.status, JLX_STATUS_BAD_PAGE);
    return false;
  }
  return true;
}
__device__ __forceinline__ int compact_count(const CompactArgs& P, int r) { return min(max(P.counts[r], 0), P.most); }
// A number of rows that `places` does not hold, or that `sums_out` has no room for: cut to it, and the status says so.
__device__ __forceinline__ void compact_check(const CompactArgs& P, int r) {
  const int n = P.counts[r];
  if (n < 0 || n > P.most || (P.sums && n > P.out_width)) atomicOr(P.status, JLX_STATUS_BAD_LENGTH);
}

// Sums of a request and head: a block, all loads of a stretch before its stores (sums and sums_out may be one).
__device__ __forceinline__ void compact_sums(const CompactArgs& P, int row) {
  const int r = row / P.H, n = min(compact_count(P, r), P.out_width);
  const float* from = P.sums + (size_t)row * P.width;
  float* to = P.sums_out + (size_t)row * P.out_width;
  const bool in_place = to == from;
  for (int base = 0; base < P.out_width; base += THREADS) {
    const int i = base + threadIdx.x;
    float v = 0.f;
    if (i < n) {
      const int place = P.places[(size_t)row * P.most + i];
      if (place >= 0 && place < P.width && !(in_place && place < i)) v = from[place];
      else atomicOr(P.status, JLX_STATUS_BAD_PAGE);
    }
    if (in_place) __syncthreads();
    if (i < P.out_width) to[i] = v;
    if (in_place) __syncthreads();
  }
}

// Into other pages: a block looks up where its rows come from and go to, then moves 16 bytes of both planes a thread, several rows'
// loads together.  The last grid column looks at the counts and moves sums.
#define MOVE_ROWS 128  // of a block
__global__ void __launch_bounds__(THREADS) kv_compact_kernel(const CompactArgs P) {
  JLX_TL(TL_KV_STORE);
  constexpr int AT_ONCE = 4;
  __shared__ int2 moves[MOVE_ROWS];
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int row = blockIdx.y, r = row / P.H, h = row - r * P.H;
  if (blockIdx.x == gridDim.x - 1) {
    if (h == 0 && threadIdx.x == 0) compact_check(P, r);
    if (P.sums) compact_sums(P, row);
    return;
  }
  const int i0 = blockIdx.x * MOVE_ROWS, rows = min(compact_count(P, r) - i0, MOVE_ROWS), chunks = P.row_bytes / 16;
  if (rows <= 0) return;
  if (threadIdx.x < rows) {
    int src, dst;
    moves[threadIdx.x] = compact_move(P, r, h, i0 + threadIdx.x, false, src, dst) ? make_int2(src, dst) : make_int2(-1, -1);
  }
  __syncthreads();
  const size_t plane = (size_t)P.H * P.page;  // rows between a key and its value
  if (P.scales && threadIdx.x < 2 * rows) {
    const int2 m = moves[threadIdx.x >> 1];
    const size_t off = (threadIdx.x & 1) * plane;
    if (m.x >= 0) P.scales[m.y + off] = P.scales[m.x + off];
  }
  uint4* pages = reinterpret_cast<uint4*>(P.pages);
  for (int x0 = threadIdx.x; x0 < rows * chunks; x0 += AT_ONCE * THREADS) {
    uint4 v[AT_ONCE][2];
    size_t to[AT_ONCE];
    bool moved[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int x = x0 + u * THREADS, i = x / chunks;
      moved[u] = false;
      if (x >= rows * chunks) continue;
      const int2 m = moves[i];
      const int c = x - i * chunks;
      moved[u] = m.x >= 0;
      to[u] = (size_t)max(m.y, 0) * chunks + c;
      const size_t from = (size_t)max(m.x, 0) * chunks + c;
      v[u][0] = pages[from];
      v[u][1] = pages[from + plane * chunks];
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
      if (moved[u]) {
        pages[to[u]] = v[u][0];
        pages[to[u] + plane * chunks] = v[u][1];
      }
  }
}

// In place: a block has a column of 16 or 32 bytes of a plane (grid x: the columns, the scales, the counts and sums).
__global__ void __launch_bounds__(THREADS) kv_compact_in_place_kernel(const CompactArgs P, int columns) {
  JLX_TL(TL_KV_STORE);
  constexpr int AT_ONCE = 4;
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int row = blockIdx.y, r = row / P.H, h = row - r * P.H;
  if (blockIdx.x == 2 * columns + 2) {
    if (h == 0 && threadIdx.x == 0) compact_check(P, r);
    if (P.sums) compact_sums(P, row);
    return;
  }
  const int n = compact_count(P, r), plane = blockIdx.x & 1, column = blockIdx.x >> 1;
  const size_t off = (size_t)plane * P.H * P.page;
  if (column == columns) {  // a byte a row
    if (!P.scales) return;
    for (int base = 0; base < n; base += THREADS) {
      const int i = base + threadIdx.x;
      int src, dst;
      const bool moves = i < n && compact_move(P, r, h, i, true, src, dst);
      const uint8_t v = moves ? P.scales[src + off] : 0;
      __syncthreads();
      if (moves) P.scales[dst + off] = v;
      __syncthreads();
    }
    return;
  }
  const int chunks = P.row_bytes / 16, wide = P.row_bytes % 32 == 0 ? 2 : 1, per = THREADS / wide;
  const int c = column * wide + threadIdx.x % wide, first = threadIdx.x / wide;
  for (int base = 0; base < n; base += per * AT_ONCE) {
    uint4 v[AT_ONCE];
    int to[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = base + u * per + first;
      int src, dst;
      to[u] = -1;
      if (i < n && compact_move(P, r, h, i, true, src, dst)) {
        to[u] = dst;
        v[u] = reinterpret_cast<const uint4*>(P.pages)[((size_t)src + off) * chunks + c];
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
      if (to[u] >= 0) reinterpret_cast<uint4*>(P.pages)[((size_t)to[u] + off) * chunks + c] = v[u];
    __syncthreads();
  }
}

// -------------------------------------------------------------------------------------------- host
JLX_API int jlx_kv_choose(const ChooseArgs* args, int cluster, void* stream_) {
  const ChooseArgs& P = *args;
  JLX_REQUIRE(P.R > 0 && P.H > 0 && P.width > 0 && P.most >= 0 && P.first >= 0 && P.recent >= 0, "kv_choose: bad sizes");
  JLX_REQUIRE(cluster >= 1 && cluster <= MAX_CLUSTER, "kv_choose: %d blocks a row", cluster);
  JLX_REQUIRE((long long)P.R * P.H <= 65535, "kv_choose: %d requests of %d KV heads are too many for a launch", P.R, P.H);
  const int per = (P.width + cluster - 1) / cluster, keys = (per + THREADS - 1) / THREADS;
  static_assert(BINS <= THREADS && FEW <= THREADS && MAX_CLUSTER <= WARPS, "a thread has a digit, a warp fetches a block's places");
  auto kernel = keys <= 2 ? kv_choose_kernel<2> : keys <= 4 ? kv_choose_kernel<4> : keys <= 8 ? kv_choose_kernel<8> : keys <= MAX_KEYS ? kv_choose_kernel<MAX_KEYS> : kv_choose_kernel<0>;
  if (cluster > 8) JLX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster, P.R * P.H);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = (cudaStream_t)stream_;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  JLX_CUDA(cudaLaunchKernelEx(&cfg, kernel, P, per));
  return 0;
}

JLX_API int jlx_kv_compact(const CompactArgs* args, int in_place, void* stream_) {
  const CompactArgs& P = *args;
  cudaStream_t stream = (cudaStream_t)stream_;
  JLX_REQUIRE(P.R > 0 && P.H > 0 && P.page > 0 && P.num_pages > 0 && P.row_bytes > 0 && P.row_bytes % 16 == 0 && P.most >= 0, "kv_compact: bad sizes");
  JLX_REQUIRE(((uintptr_t)P.pages & 15) == 0, "kv_compact: pages must be 16-byte aligned");
  JLX_REQUIRE(((long long)P.num_pages + 1) * 2 * P.H * P.page < (1ll << 31), "kv_compact: cache too large for 32-bit rows");
  JLX_REQUIRE((long long)P.R * P.H <= 65535, "kv_compact: %d requests of %d KV heads are too many for a launch", P.R, P.H);
  if (in_place) {
    const int columns = P.row_bytes % 32 == 0 ? P.row_bytes / 32 : P.row_bytes / 16;
    JLX_CUDA(jlx_launch_pdl(kv_compact_in_place_kernel, dim3(2 * columns + 3, P.R * P.H), dim3(THREADS), 0, stream, P, columns));
    return 0;
  }
  static_assert(2 * MOVE_ROWS <= THREADS, "a thread looks up a row, and moves a scale");
  JLX_CUDA(jlx_launch_pdl(kv_compact_kernel, dim3((P.most + MOVE_ROWS - 1) / MOVE_ROWS + 1, P.R * P.H), dim3(THREADS), 0, stream, P));
  return 0;
}
