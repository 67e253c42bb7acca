// The weights that cached keys receive from few query rows of a request: up to 16 (token, head of the group) rows a KV head, single
// decoded tokens above all (attention_weights.cuh has the formula), over a cache in bfloat16 or in 8 bits, heads of 64 or 128.
//
// A thread-block cluster serves a request and KV head; its blocks cut the keys.  Scores are made transposed, S^T = K Q^T, with
// keys as the 16 rows of a tensor-core tile and query rows as its 8 columns, and straight from memory: the contraction index may
// run in any order that both operands share, and with every fourth 16-byte chunk of a row as a thread's a key's operands of two
// products are one load, nothing passes through shared memory.  The scores stay (in shared memory, or in scratch where a range
// is too long) until the row's maximum and sum are known: of the warps, the block, the cluster.  Then every key's weights
// are added up by one thread, in the rows' order: the same bits every time, no atomics.
//
// 8 bits: codes become bfloat16, which holds every one of them, and a key's power of two multiplies its scores: nothing is rounded.
//
// It is bound by the keys' bytes.
#include <cooperative_groups.h>

#include "attention_weights.cuh"
#include "mma_sync.cuh"

namespace cg = cooperative_groups;

#define THREADS 256
#define WARPS (THREADS / 32)
#define KT 16  // keys of a warp's tile
#define MAX_SPLITS 8

template <int DH, bool F8, int NG>
__global__ void __launch_bounds__(THREADS) attention_weights_kernel(const WeightsParams P) {
  JLX_TL(TL_ATTN_DECODE);
  constexpr int ROWS = 8 * NG, CH = DH * (F8 ? 1 : 2) / 64;  // 16-byte chunks of a key that a thread has
  constexpr int AHEAD = F8 ? 4 : 2;                          // tiles whose loads are in flight together
  constexpr int REGS = F8 ? 8 : 4;                           // registers of bfloat16 pairs that a chunk becomes
  extern __shared__ __align__(16) float smem_buf[];
  __shared__ __align__(16) float ml[2][ROWS], part[WARPS][ROWS], factor[ROWS];
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
  const int first = __reduce_min_sync(0xffffffffu, tok.lo), p_max = __reduce_max_sync(0xffffffffu, tok.p);
  const int end_all = rows_end(P.R, it, p_max), start = first / KT * KT;
  // equal ranges of whole tiles
  const int per = max((end_all - start + KT * P.splits - 1) / (KT * P.splits), 0) * KT, range0 = start + split * per;
  const int begin = max(first, range0), end = min(end_all, range0 + per), tiles = end > begin ? (end - range0 + KT - 1) / KT : 0;
  if (end_all > min(P.W.max_kv, P.W.width) || per > P.buf_keys || it.cnt * G > ROWS) {  // more keys than the call was sized for: the whole cluster leaves
    if (tid == 0) atomicOr(P.R.status, JLX_STATUS_BAD_PAGE);
    weights_copy(P, row, 0, P.W.width, everyone, all);
    return;
  }
  float* buf = P.W.scratch ? P.W.scratch + (row * P.splits + split) * (size_t)P.buf_keys * ROWS : smem_buf;

  // ---- queries: column g of group ng is row 8 ng + g, its entries in the order of the keys' chunks
  uint32_t qf[NG][CH * REGS];
  float sc[NG][2], slope[NG][2], m[NG][2];
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
#pragma unroll
    for (int c = 0; c < 2; ++c) {  // this thread's scores are those of rows 2 t4 and 2 t4 + 1 of the group
      const int from = min(8 * ng + 2 * t4 + c, n_rows - 1);
      sc[ng][c] = __shfl_sync(0xffffffffu, tok.sc, from);
      slope[ng][c] = __shfl_sync(0xffffffffu, tok.slope, from);
      pos[ng][c] = __shfl_sync(0xffffffffu, tok.p, from);
      lo[ng][c] = __shfl_sync(0xffffffffu, tok.lo, from);
      m[ng][c] = ROWS_NEG_BIG;
    }
  }
  const int* table = P.R.block_table + (size_t)r * P.R.bt_stride;
  const uint8_t* pages = reinterpret_cast<const uint8_t*>(P.R.pages);

  // ---- scores
  for (int t0 = warp; t0 < tiles; t0 += WARPS * AHEAD) {
    uint4 k[AHEAD][2][CH];
    float ks[AHEAD][2];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int place = range0 + (t0 + a * WARPS) * KT + h * 8 + g;
        const int at = place >= begin && place < end ? rows_cache_row(P.R, table, hk, place) : -1;
        if (F8) ks[a][h] = at >= 0 ? fp8_scale(P.R.scales[at]) : 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
          k[a][h][c] = at >= 0 ? *reinterpret_cast<const uint4*>(pages + (size_t)at * (DH * (F8 ? 1 : 2)) + (t4 + 4 * c) * 16) : make_uint4(0, 0, 0, 0);
      }
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
          const uint32_t w[4] = {k[a][h][c].x, k[a][h][c].y, k[a][h][c].z, k[a][h][c].w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (F8) {
              kf[h][(2 * u) % REGS] = weights_widen(w[u], 0x9180);
              kf[h][(2 * u + 1) % REGS] = weights_widen(w[u], 0xb3a2);
            } else {
              kf[h][u] = w[u];
            }
          }
        }
#pragma unroll
        for (int u = 0; u < REGS; u += 2) {
          const uint32_t f[4] = {kf[0][u], kf[1][u], kf[0][u + 1], kf[1][u + 1]};
#pragma unroll
          for (int ng = 0; ng < NG; ++ng) mma_bf16(s[ng], f, qf[ng][c * REGS + u], qf[ng][c * REGS + u + 1]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int place = range0 + t * KT + h * 8 + g;
#pragma unroll
        for (int ng = 0; ng < NG; ++ng) {
          float v[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            v[c] = s[ng][2 * h + c] * sc[ng][c];
            if (F8) v[c] *= ks[a][h];
            if (P.R.cap_log2 > 0.f) v[c] = P.R.cap_log2 * weights_tanh(v[c]);
            if (P.R.slopes) v[c] -= slope[ng][c] * (float)(pos[ng][c] - place);
            if (place < lo[ng][c] || place > pos[ng][c] || place < begin || place >= end) v[c] = -INFINITY;
            m[ng][c] = fmaxf(m[ng][c], v[c]);
          }
          *reinterpret_cast<float2*>(buf + (size_t)(place - range0) * ROWS + ng * 8 + t4 * 2) = make_float2(v[0], v[1]);
        }
      }
    }
  }
  // ---- the rows' maxima: of the warp, of the block
#pragma unroll
  for (int ng = 0; ng < NG; ++ng)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) m[ng][c] = fmaxf(m[ng][c], __shfl_xor_sync(0xffffffffu, m[ng][c], o));
      if (g == 0) part[warp][ng * 8 + t4 * 2 + c] = m[ng][c];
    }
  __syncthreads();
  if (tid < ROWS) {
    float v = part[0][tid];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) v = fmaxf(v, part[w][tid]);
    ml[0][tid] = v;
  }
  __syncthreads();
  // ---- exponentials in place, and their sums; a thread has four rows of every (THREADS / (ROWS / 4))-th key
  constexpr int QUADS = ROWS / 4;
  const int quad = tid % QUADS;
  float4 top = reinterpret_cast<const float4*>(ml[0])[quad], sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j = tid / QUADS; j < tiles * KT; j += THREADS / QUADS) {
    float4* at = reinterpret_cast<float4*>(buf + (size_t)j * ROWS) + quad;
    float4 v = *at;
    v.x = rows_exp2(v.x - top.x); v.y = rows_exp2(v.y - top.y); v.z = rows_exp2(v.z - top.z); v.w = rows_exp2(v.w - top.w);
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    *at = v;
  }
#pragma unroll
  for (int o = QUADS; o < 32; o <<= 1) {
    sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o); sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
    sum.z += __shfl_xor_sync(0xffffffffu, sum.z, o); sum.w += __shfl_xor_sync(0xffffffffu, sum.w, o);
  }
  if (lane < QUADS) reinterpret_cast<float4*>(part[warp])[lane] = sum;
  __syncthreads();
  if (tid < ROWS) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += part[w][tid];
    ml[1][tid] = v;
  }
  cluster.sync();
  // ---- of the cluster
  if (tid < ROWS) {
    float mm = ROWS_NEG_BIG, l = 0.f;
    for (int q = 0; q < P.splits; ++q) mm = fmaxf(mm, *cluster.map_shared_rank(&ml[0][tid], q));
    for (int q = 0; q < P.splits; ++q) {
      const float mq = *cluster.map_shared_rank(&ml[0][tid], q);
      l += *cluster.map_shared_rank(&ml[1][tid], q) * (mq == mm ? 1.f : rows_exp2(mq - mm));
    }
    const int t = min(tid, n_rows - 1) / G, head = hk * G + min(tid, n_rows - 1) - t * G;
    const float mine = ml[0][tid];
    factor[tid] = tid < n_rows ? (mine == mm ? 1.f : rows_exp2(mine - mm)) * rows_inverse(P.R, mm, l, head) : 0.f;
  }
  cluster.barrier_arrive();  // (a block's shared memory stays until the others have read it)
  __syncthreads();
  // ---- every key's weights
  float f[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) f[i] = factor[i];
  const float* add = P.W.add ? P.W.add + row * P.W.width : nullptr;
  float* out = P.W.out + row * P.W.width;
  for (int j = tid; j < tiles * KT; j += THREADS) {
    const int place = range0 + j;
    if (place < begin || place >= end) continue;
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(buf + (size_t)j * ROWS + i);
      if (i < n_rows) w += v.x * f[i];
      if (i + 1 < n_rows) w += v.y * f[i + 1];
      if (i + 2 < n_rows) w += v.z * f[i + 2];
      if (i + 3 < n_rows) w += v.w * f[i + 3];
    }
    out[place] = (add ? add[place] : 0.f) + w;
  }
  // what no row sees
  weights_copy(P, row, 0, min(first, P.W.width), everyone, all);
  weights_copy(P, row, max(end_all, 0), P.W.width, everyone, all);
  cluster.barrier_wait();
}

// -------------------------------------------------------------------------------------------- host
template <int DH, bool F8, int NG>
static int launch_weights(const WeightsParams& P, cudaStream_t stream) {
  auto kernel = attention_weights_kernel<DH, F8, NG>;
  const size_t smem = P.W.scratch ? 0 : (size_t)P.buf_keys * 8 * NG * 4;
  if (smem > 48 * 1024) JLX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
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

// rows: most query rows of a request and KV head; buf_keys: keys that a range may have.
JLX_API int jlx_attention_weights(const RowsArgs* rows_args, const WeightsArgs* args, int rows, int splits, int buf_keys, void* stream_) {
  WeightsParams P;
  if (int e = rows_params(*rows_args, P.R)) return e;
  P.W = *args;
  P.splits = splits;
  P.buf_keys = buf_keys;
  JLX_REQUIRE(splits >= 1 && splits <= MAX_SPLITS && buf_keys > 0 && buf_keys % KT == 0, "attention_weights: %d ranges of %d keys", splits, buf_keys);
  JLX_REQUIRE(P.W.scratch || (size_t)buf_keys * (rows <= 8 ? 8 : 16) * 4 <= 200 * 1024, "attention_weights: a range of %d keys needs scratch", buf_keys);
  JLX_REQUIRE((long long)P.R.n_requests * P.R.Hkv <= 65535, "attention_weights: %d requests of %d KV heads are too many for a launch", P.R.n_requests, P.R.Hkv);
  JLX_REQUIRE(rows <= 16, "attention_weights: %d query rows a KV head", rows);
  cudaStream_t stream = (cudaStream_t)stream_;
  const bool f8 = P.R.scales != nullptr;
  const int dh = rows_args->dh;
  if (rows <= 8)
    return dh == 128 ? (f8 ? launch_weights<128, true, 1>(P, stream) : launch_weights<128, false, 1>(P, stream))
                     : (f8 ? launch_weights<64, true, 1>(P, stream) : launch_weights<64, false, 1>(P, stream));
  return dh == 128 ? (f8 ? launch_weights<128, true, 2>(P, stream) : launch_weights<128, false, 2>(P, stream))
                   : (f8 ? launch_weights<64, true, 2>(P, stream) : launch_weights<64, false, 2>(P, stream));
}
