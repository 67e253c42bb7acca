// The weights that cached keys receive from few query rows of a request: up to 16 (token, head of the group) rows a KV head, single
// decoded tokens above all (attention_weights.cuh has the formula), over a cache in bfloat16 or in 8 bits, heads of 64 or 128.
//
// A thread-block cluster serves a request and KV head; its blocks cut the keys.  Scores are made transposed, S^T = K Q^T, with
// keys as the 16 rows of a tensor-core tile and query rows as its 8 columns, and straight from memory: the contraction index may
// run in any order that both operands share, and with every fourth 16-byte chunk of a row as a thread's a key's operands of two
// products are one load, nothing passes through shared memory.  The scores stay (in shared memory, or in scratch where a range
// is too long) while every thread keeps the maximum and the sum of its share of them; when those are known of the warp, the block and
// the cluster, a key's weights are added up by one thread, in the rows' order: the same bits every time, no atomics.
//
// 8 bits: codes become float16, which holds every one of them, and a key's power of two multiplies its scores.  Queries are brought to
// float16 by a power of two per row that makes the largest entry 2^7 .. 2^8: entries above 2^-24 of it are exact, smaller ones off by
// 2^-32 of it at most.  (As bfloat16, which needs no such power, a pair of codes takes four instructions, not one.)
//
// It is bound by the keys' bytes, and by the instructions and the latency between a byte and its weight: a warp has 32 registers of
// keys on their way while it works on as many (without that 64 sessions of up to 8192 keys took 208 us).  Measured (B200, 40 heads on 8 of
// 128): those sessions 164 us, 5.2 TB/s; 8 of up to 30,000 keys in 8 bits 79 us, 2.7 TB/s; one of 700 keys 13.4 us a call, 7.5 on the
// device.  Ranges: 64 sessions with 1, 4, 8, 16 of them 195, 193, 166, 229 us.  Tried and slower: two sums a product, to halve its chain
// (registers).
#include <cooperative_groups.h>

#include "attention_weights.cuh"
#include "mma_sync.cuh"

namespace cg = cooperative_groups;

#define THREADS 128
#define WARPS (THREADS / 32)
#define EARLY 8  // of a thread's keys, whose places in `add` are asked for before the rows' sums are known
#define KT 16  // keys of a warp's tile

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
#define MAX_SPLITS 16  // (clusters of more than 8 blocks are not portable; this is sm_100a only)
#define MAX_HELD (100 * 1024)  // bytes of scores in shared memory: two blocks of the largest kind a multiprocessor, so that a cluster of 16 has places

// WHOLE: the page size is a multiple of a tile's keys, which then lie side by side.
template <int DH, bool F8, int NG, bool WHOLE>
__global__ void __launch_bounds__(THREADS, NG == 2 ? 3 : 4) attention_weights_kernel(const WeightsParams P) {
  JLX_TL(TL_ATTN_DECODE);
  constexpr int ROWS = 8 * NG, CH = DH * (F8 ? 1 : 2) / 64;  // 16-byte chunks of a key that a thread has
  constexpr int AHEAD = 4 / CH;                              // tiles of a batch: 32 registers of keys
  constexpr int REGS = F8 ? 8 : 4;                           // registers of bfloat16 pairs that a chunk becomes
  extern __shared__ __align__(16) float smem_buf[];
  __shared__ float2 ml[ROWS], part[WARPS][ROWS], factor[ROWS];  // (maximum, sum); at last (maximum of all, what the exponentials are divided by, inverted)
  cg::cluster_group cluster = cg::this_cluster();
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int split = blockIdx.x, r = blockIdx.y / P.R.Hkv, hk = blockIdx.y - r * P.R.Hkv;
  const size_t row = blockIdx.y;
  RowsItem it;
  const int everyone = split * THREADS + tid, all = P.splits * THREADS;
  if (!weights_request(P, r, it)) { weights_copy(P, row, 0, P.W.width, everyone, all); return; }
  const int G = P.R.Hq / P.R.Hkv, n_rows = min(it.cnt * G, ROWS);
  const RowsToken tok = rows_token(P.R, it, min(lane, n_rows - 1), hk);
  const int p_max = __reduce_max_sync(0xffffffffu, tok.p), end_all = rows_end(P.R, it, p_max);
  // (a row that sees nothing has no first key: under a window its 0 would stretch the range over keys that no row sees)
  const int first = __reduce_min_sync(0xffffffffu, tok.p < 0 ? max(end_all, 0) : tok.lo), start = first / KT * KT;
  // equal ranges of whole tiles
  const int per = max((end_all - start + KT * P.splits - 1) / (KT * P.splits), 0) * KT, range0 = start + split * per;
  const int begin = max(first, range0), end = min(end_all, range0 + per), tiles = end > begin ? (end - range0 + KT - 1) / KT : 0;
  if (end_all > min(P.W.max_kv, P.W.width) || per > P.buf_keys || it.cnt * G > ROWS) {  // more keys than the call was sized for: the whole cluster leaves
    if (tid == 0) atomicOr(P.R.status, JLX_STATUS_BAD_PAGE);
    weights_copy(P, row, 0, P.W.width, everyone, all);
    return;
  }
  const int kept = (n_rows + 1) & ~1;  // scores of a key that are kept
  float* buf = P.W.scratch ? P.W.scratch + (row * P.splits + split) * (size_t)P.buf_keys * ((P.rows + 1) & ~1) : smem_buf;

  // ---- queries: column g of group ng is row 8 ng + g, its entries in the order of the keys' chunks
  uint32_t qf[NG][CH * REGS];
  float sc[NG][2], slope[NG][2], m[NG][2], l[NG][2];
  int pos[NG][2], lo[NG][2];
#pragma unroll
  for (int ng = 0; ng < NG; ++ng) {
    const int qr = min(8 * ng + g, n_rows - 1), t = qr / G;
    const bf16* q = P.R.q + ((size_t)(it.n0 + t) * P.R.Hq + hk * G + qr - t * G) * DH;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int u = 0; u < REGS / 4; ++u) {
        const uint4 v = *reinterpret_cast<const uint4*>(q + (t4 + 4 * c) * 2 * REGS + u * 8);
        qf[ng][c * REGS + u * 4] = v.x; qf[ng][c * REGS + u * 4 + 1] = v.y; qf[ng][c * REGS + u * 4 + 2] = v.z; qf[ng][c * REGS + u * 4 + 3] = v.w;
      }
    int e = 0;
    if (F8) {  // (the row's four threads have its entries)
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < CH * REGS; ++i) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[ng][i]));
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      e = max(min((int)(__float_as_uint(top) >> 23) - 127, 120), -110) - 7;
      const float in = fp8_pow2(-e);
#pragma unroll
      for (int i = 0; i < CH * REGS; ++i) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[ng][i]));
        const __half2 h = __floats2half2_rn(f.x * in, f.y * in);
        qf[ng][i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {  // this thread's scores are those of rows 2 t4 and 2 t4 + 1 of the group
      const int from = min(8 * ng + 2 * t4 + c, n_rows - 1);
      sc[ng][c] = __shfl_sync(0xffffffffu, tok.sc, from);
      if (F8) sc[ng][c] *= fp8_pow2(__shfl_sync(0xffffffffu, e, 4 * (2 * t4 + c)));
      slope[ng][c] = __shfl_sync(0xffffffffu, tok.slope, from);
      pos[ng][c] = __shfl_sync(0xffffffffu, tok.p, from);
      lo[ng][c] = __shfl_sync(0xffffffffu, tok.lo, from);
      m[ng][c] = ROWS_NEG_BIG;
      l[ng][c] = 0.f;
    }
  }
  const int* table = P.R.block_table + (size_t)r * P.R.bt_stride;
  const uint8_t* pages = reinterpret_cast<const uint8_t*>(P.R.pages);

  // ---- scores.  A batch of tiles is on its way while the one before is worked on, and its keys' places are known a batch earlier
  // still: page, key and product would be a chain of two trips to memory otherwise.
  const int full_lo = __reduce_max_sync(0xffffffffu, tok.lo), full_hi = min(__reduce_min_sync(0xffffffffu, tok.p) + 1, end);  // seen by all rows
  const bool bent = P.R.cap_log2 > 0.f || P.R.slopes;
  constexpr int ROW_BYTES = DH * (F8 ? 1 : 2), AT = WHOLE ? 1 : 2;
  // Where a thread's keys lie (WHOLE: the second one 8 rows behind the first).  Keys outside the range are masked, so anything may be read for
  // them (row g); keys without a page are zeros: `lost` has a bit for them.
  struct Places {
    int at[AHEAD][AT];
    uint32_t lost;
  };
  auto find = [&](int t0, Places& L) {
    L.lost = 0u;
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int t = t0 + a * WARPS, place0 = range0 + t * KT;
      if (WHOLE) {
        L.at[a][0] = g;
        if (t < tiles) {
          const int pi = P.page_shift < 0 ? place0 / P.R.page_size : place0 >> P.page_shift, page = pi < P.R.bt_stride ? table[pi] : -1;
          if (rows_page_there(P.R, page)) {
            L.at[a][0] = (page * 2 * P.R.Hkv + hk) * P.R.page_size + (place0 - pi * P.R.page_size) + g;
          } else {
            atomicOr(P.R.status, JLX_STATUS_BAD_PAGE);
            L.lost |= 3u << (2 * a);
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < AT; ++h) {
          const int place = place0 + h * 8 + g;
          L.at[a][h] = 0;
          if (place >= begin && place < end) {
            L.at[a][h] = rows_cache_row(P.R, table, hk, place);
            if (L.at[a][h] < 0) L.lost |= 1u << (2 * a + h);
            L.at[a][h] = max(L.at[a][h], 0);
          }
        }
      }
    }
  };
  struct Batch {
    uint4 k[AHEAD][2][CH];
    float ks[AHEAD][2];
    uint32_t lost;
  };
  auto fetch = [&](const Places& L, Batch& B) {
    B.lost = L.lost;
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* p = pages + (size_t)L.at[a][WHOLE ? 0 : h] * ROW_BYTES + t4 * 16 + (WHOLE ? h * 8 * ROW_BYTES : 0);
        if (F8) B.ks[a][h] = fp8_scale(P.R.scales[L.at[a][WHOLE ? 0 : h] + (WHOLE ? h * 8 : 0)]);
#pragma unroll
        for (int c = 0; c < CH; ++c) B.k[a][h][c] = *reinterpret_cast<const uint4*>(p + c * 64);
      }
  };
  auto score = [&](int t0, const Batch& B) {
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int t = t0 + a * WARPS;
      if (t >= tiles) break;
      float s[NG][4];
#pragma unroll
      for (int ng = 0; ng < NG; ++ng) s[ng][0] = s[ng][1] = s[ng][2] = s[ng][3] = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        uint32_t kf[2][REGS];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w[4] = {B.k[a][h][c].x, B.k[a][h][c].y, B.k[a][h][c].z, B.k[a][h][c].w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (F8) {
              fp8x4_to_half(w[u], kf[h][(2 * u) % REGS], kf[h][(2 * u + 1) % REGS]);
            } else {
              kf[h][u] = w[u];
            }
          }
        }
#pragma unroll
        for (int u = 0; u < REGS; u += 2) {
          const uint32_t f[4] = {kf[0][u], kf[1][u], kf[0][u + 1], kf[1][u + 1]};
#pragma unroll
          for (int ng = 0; ng < NG; ++ng) {
            if (F8) mma_f16(s[ng], f, qf[ng][c * REGS + u], qf[ng][c * REGS + u + 1]);
            else mma_bf16(s[ng], f, qf[ng][c * REGS + u], qf[ng][c * REGS + u + 1]);
          }
        }
      }
      if (__any_sync(0xffffffffu, B.lost >> (2 * a) & 3u)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int ng = 0; ng < NG; ++ng)
            if (B.lost >> (2 * a + h) & 1u) s[ng][2 * h] = s[ng][2 * h + 1] = 0.f;
      }
      const int place0 = range0 + t * KT;
      float* to = buf + (size_t)(t * KT + g) * kept + t4 * 2;
      const bool masked = place0 < max(full_lo, begin) || place0 + KT > full_hi;
#pragma unroll
      for (int ng = 0; ng < NG; ++ng) {
        float v[2][2];  // [key][row]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int c = 0; c < 2; ++c) v[h][c] = s[ng][2 * h + c] * (F8 ? sc[ng][c] * ((B.lost >> (2 * a + h) & 1u) ? 0.f : B.ks[a][h]) : sc[ng][c]);
          if (masked || bent) {
            const int place = place0 + h * 8 + g;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (P.R.cap_log2 > 0.f) v[h][c] = P.R.cap_log2 * weights_tanh(v[h][c]);
              if (P.R.slopes) v[h][c] -= slope[ng][c] * (float)(pos[ng][c] - place);
              if (place < max(lo[ng][c], begin) || place > pos[ng][c] || place >= end) v[h][c] = -INFINITY;
            }
          }
          if (ng * 8 + t4 * 2 < kept) *reinterpret_cast<float2*>(to + h * 8 * kept + ng * 8) = make_float2(v[h][0], v[h][1]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float top = fmaxf(m[ng][c], fmaxf(v[0][c], v[1][c]));
          l[ng][c] = fmaf(l[ng][c], rows_exp2(m[ng][c] - top), rows_exp2(v[0][c] - top) + rows_exp2(v[1][c] - top));
          m[ng][c] = top;
        }
      }
    }
  };
  constexpr int STEP = WARPS * AHEAD;
  Places at;
  Batch even, odd;
  if (tiles > 0) {
    find(warp, at);
    fetch(at, even);
    find(warp + STEP, at);
#pragma unroll 1
    for (int t = warp; t < tiles; t += 2 * STEP) {
      fetch(at, odd);
      find(t + 2 * STEP, at);
      score(t, even);
      fetch(at, even);
      find(t + 3 * STEP, at);
      score(t + STEP, odd);
    }
  }
  // ---- the rows' maxima and sums: of the warp, of the block, of the cluster
  auto join = [](float2 a, float2 b) {
    const float top = fmaxf(a.x, b.x);
    return make_float2(top, (a.x == top ? a.y : a.y * rows_exp2(a.x - top)) + (b.x == top ? b.y : b.y * rows_exp2(b.x - top)));
  };
#pragma unroll
  for (int ng = 0; ng < NG; ++ng)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float2 v = make_float2(m[ng][c], l[ng][c]);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) v = join(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
      if (g == 0) part[warp][ng * 8 + t4 * 2 + c] = v;
    }
  __syncthreads();
  if (tid < ROWS) {
    float2 v = part[0][tid];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) v = join(v, part[w][tid]);
    ml[tid] = v;
  }
  cluster.barrier_arrive();
  // while the others come: what no row sees, and what the first of this thread's keys are added to
  weights_copy(P, row, 0, min(first, P.W.width), everyone, all);
  weights_copy(P, row, max(end_all, 0), P.W.width, everyone, all);
  const float* add = P.W.add ? P.W.add + row * P.W.width : nullptr;
  float* out = P.W.out + row * P.W.width;
  float early[EARLY];
#pragma unroll
  for (int u = 0; u < EARLY; ++u) {
    const int place = range0 + tid + u * THREADS;
    early[u] = add && place >= begin && place < end ? add[place] : 0.f;
  }
  cluster.barrier_wait();
  if (tid < ROWS) {
    float2 v = make_float2(ROWS_NEG_BIG, 0.f);
#pragma unroll
    for (int q0 = 0; q0 < MAX_SPLITS; q0 += 8) {
      if (q0 >= P.splits) break;
      float2 w[8];  // (asked for together: each takes a trip to another multiprocessor)
#pragma unroll
      for (int q = 0; q < 8; ++q) w[q] = q0 + q < P.splits ? *cluster.map_shared_rank(&ml[tid], q0 + q) : make_float2(ROWS_NEG_BIG, 0.f);
#pragma unroll
      for (int q = 0; q < 8; ++q) v = join(v, w[q]);
    }
    const int qr = min(tid, n_rows - 1), head = hk * G + qr - qr / G * G;
    factor[tid] = make_float2(v.x, rows_inverse(P.R, v.x, v.y, head));
  }
  cluster.barrier_arrive();  // (a block's shared memory stays until the others have read it)
  __syncthreads();
  // ---- every key's weights
  float2 f[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) f[i] = factor[i];
  auto weigh = [&](int j, float before) {
    const int place = range0 + j;
    if (place < begin || place >= end) return;
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; i += 2) {
      if (i >= n_rows) break;
      const float2 v = *reinterpret_cast<const float2*>(buf + (size_t)j * kept + i);
      w += rows_exp2(v.x - f[i].x) * f[i].y;
      if (i + 1 < n_rows) w += rows_exp2(v.y - f[i + 1].x) * f[i + 1].y;
    }
    out[place] = before + w;
  };
#pragma unroll
  for (int u = 0; u < EARLY; ++u) weigh(tid + u * THREADS, early[u]);
  for (int j0 = tid + EARLY * THREADS; j0 < tiles * KT; j0 += 4 * THREADS) {
    float before[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int place = range0 + j0 + u * THREADS;
      before[u] = add && place >= begin && place < end ? add[place] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) weigh(j0 + u * THREADS, before[u]);
  }
  cluster.barrier_wait();
}

// -------------------------------------------------------------------------------------------- host
template <int DH, bool F8, int NG, bool WHOLE>
static int launch_weights(const WeightsParams& P, cudaStream_t stream) {
  auto kernel = attention_weights_kernel<DH, F8, NG, WHOLE>;
  const size_t smem = P.W.scratch ? 0 : (size_t)P.buf_keys * ((P.rows + 1) & ~1) * 4;
  if (P.splits > 8) JLX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (smem > 40 * 1024) JLX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(P.splits, P.R.n_requests * P.R.Hkv);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = P.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  JLX_CUDA(cudaLaunchKernelEx(&cfg, kernel, P));
  return 0;
}

template <int DH, bool F8>
static int launch_weights_of(const WeightsParams& P, cudaStream_t stream) {
  const bool whole = P.R.page_size % KT == 0;
  if (P.rows <= 8) return whole ? launch_weights<DH, F8, 1, true>(P, stream) : launch_weights<DH, F8, 1, false>(P, stream);
  return whole ? launch_weights<DH, F8, 2, true>(P, stream) : launch_weights<DH, F8, 2, false>(P, stream);
}

// rows: most query rows of a request and KV head; buf_keys: keys that a range may have.
JLX_API int jlx_attention_weights(const RowsArgs* rows_args, const WeightsArgs* args, int rows, int splits, int buf_keys, void* stream_) {
  WeightsParams P;
  if (int e = rows_params(*rows_args, P.R)) return e;
  P.W = *args;
  P.splits = splits;
  P.buf_keys = buf_keys;
  P.rows = rows;
  P.page_shift = (P.R.page_size & (P.R.page_size - 1)) == 0 ? __builtin_ctz(P.R.page_size) : -1;
  JLX_REQUIRE(splits >= 1 && splits <= MAX_SPLITS && buf_keys > 0 && buf_keys % KT == 0, "attention_weights: %d ranges of %d keys", splits, buf_keys);
  JLX_REQUIRE(P.W.scratch || (size_t)buf_keys * ((rows + 1) & ~1) * 4 <= MAX_HELD, "attention_weights: a range of %d keys needs scratch", buf_keys);
  JLX_REQUIRE((long long)P.R.n_requests * P.R.Hkv <= 65535, "attention_weights: %d requests of %d KV heads are too many for a launch", P.R.n_requests, P.R.Hkv);
  JLX_REQUIRE(rows <= 16, "attention_weights: %d query rows a KV head", rows);
  cudaStream_t stream = (cudaStream_t)stream_;
  if (rows_args->dh == 128) return P.R.scales ? launch_weights_of<128, true>(P, stream) : launch_weights_of<128, false>(P, stream);
  return P.R.scales ? launch_weights_of<64, true>(P, stream) : launch_weights_of<64, false>(P, stream);
}
