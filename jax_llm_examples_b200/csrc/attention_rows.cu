// Grouped-query attention over the paged cache, held in bfloat16 or in 8 bits (fp8_rows.cuh), of more query rows than
// attention_few.cu takes: short portions and drafted trees (attention_rows.cuh has the mask and the formula), head sizes 64
// and 128.
//
// A block of four warps takes up to 32 or 64 query rows of one item and KV head, and one range of its keys; keys come in
// tiles of 64 by cp.async, row by row through the block table (any page size), STAGES tiles in flight.  With 32 rows
// two warps share 16 rows' keys, with 64 each warp has 16 rows to itself; warps that share rows keep maxima, sums and outputs
// of their own and meet once, at the end.  Ranges of one row (split over the key axis
// when there are few rows) are joined by a second kernel.
//
// 8 bits: codes go to the tensor cores as float16, which holds every one of them; no number of the cache is rounded.  A key's
// power of two multiplies its column of scores.  A value's is added to its key's exponent: with a_j = s_j + e_j the weights
// w_j = 2^(a_j - max a) and the sum  sum w_j 2^-e_j  give  out = sum w_j code_j / sum w_j 2^-e_j,  so that weights stay in
// [0, 1] and float16 rounds each by 2^-11 of it at most, or by 2^-25 where it is below 2^-14: keys whose weight times scale is
// below 2^-25 of the row's largest add to the sum and no longer to the values, of which they are at most as small a part.
// (Scales lie within 2^-60 .. 2^60: no product leaves the 32-bit range.)  Queries are brought to float16 by a power of two per
// row, which makes the largest entry 2^7 .. 2^8: entries above 2^-24 of it are exact, smaller ones off by 2^-32 of it at most.
// Bfloat16 caches: probabilities are rounded to bfloat16 for the product with the values (2^-8 of each at most); sums, maxima
// and outputs are 32-bit in both.
//
// The contraction index of a product may run in any order that both operands share, and this is what makes codes cheap: the 16
// codes that a thread reads at once (16 bytes of a key) serve four steps of the score product, whose query fragments are
// gathered in that order; of the values a transposing load of byte pairs gives two keys' codes of two neighbouring entries,
// which a byte permutation makes operands for two products, over the even and the odd entries.
//
// Masked keys: their scores are replaced, not added to; rows of the cache outside an item's keys are never read (zeros stand
// in); a value that is not finite and that some row of the tile does not see is taken out of the tile and added to the rows
// that do see it at the end (a product would spread 0 * infinity over all rows).  In 8 bits only a row's scale can say NaN.
//
// Pages that hold no whole boxes of 16 rows, and scales that start off a 16-byte boundary, come here; the rest goes to the
// tcgen05 kernel, which is up to 5.9 times as fast.  Measured (B200, pages of 24): 2,048 tokens after 1,500, 40 heads on 8 of 128,
// 8 bits: 1,089 us, 97 TFLOP/s (185 us there); trees of 32 tokens on 8 requests, bfloat16: 448 us (94).  Its mma.sync products and
// the conversion of codes in every warp bound it.
#include "attention_rows.cuh"
#include "mbarrier.cuh"
#include "mma_sync.cuh"

#define KT 64  // keys per tile

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Where 16-byte chunk c of row `row` lies in a tile whose rows have CH chunks: rows that are read together (eight of one chunk,
// or two of four neighbouring chunks) fall on different banks.
template <int CH> __device__ __forceinline__ int chunk_at(int row, int c) {
  if (CH == 4) return row * CH + (c ^ ((row >> 1) & 3));
  return row * CH + (c ^ (((row & 1) << 2) | ((row >> 1) & 3)));
}

template <int DH, bool F8> struct RowsTile {
  static constexpr int ELEM = F8 ? 1 : 2;
  static constexpr int CH = DH * ELEM / 16;      // 16-byte chunks per row
  static constexpr int BYTES = KT * DH * ELEM;   // keys or values of a tile
  static constexpr int STAGES = F8 ? 4 : 3;
  static constexpr int SCALE_BYTES = F8 ? 3 * KT * 4 : 0;  // per stage: the keys' scales, the values' exponents, 2^-exponent
  static constexpr int LD = DH + 4;              // floats between rows of the outputs as the warps leave them
  static constexpr int RING = STAGES * (2 * BYTES + SCALE_BYTES);
  static constexpr int MERGE = 4 * 16 * LD * 4 + 4 * 16 * 8;
  static constexpr int SMEM = RING > MERGE ? RING : MERGE;
};

// WM: groups of 16 rows per block (2, 4); the 4 / WM warps of a group share its keys.
template <int DH, bool F8, int WM>
__global__ void __launch_bounds__(128) attention_rows_kernel(const RowsParams P) {
  JLX_TL(TL_ATTN_DECODE);
  using T = RowsTile<DH, F8>;
  constexpr int CH = T::CH, STAGES = T::STAGES, WK = 4 / WM, NK = KT / WK, NT = NK / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int row_of[2][KT];      // flat cache rows of the keys of the tile to fetch next
  __shared__ int4 row_tok[16 * WM];  // (token, head, position, first key) of the block's rows
  __shared__ int2 row_sc[16 * WM];   // (score factor, slope)
  __shared__ int span[4];            // smallest and largest first key, smallest and largest position of the rows
  __shared__ int any_bad, first_token;  // (the item's first token: kept in a register it made the kernel 8 % slower)
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int split = blockIdx.x % P.splits, item_i = blockIdx.x / P.splits;
  const int tiles_y = gridDim.y / P.Hkv, hk = blockIdx.y / tiles_y, row0 = (blockIdx.y - hk * tiles_y) * 16 * WM;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  RowsItem it;
  if (!rows_item(P, item_i, it)) return;
  const int G = P.Hq / P.Hkv, n_rows = min(it.cnt * G - row0, 16 * WM);
  if (n_rows <= 0) return;

  if (tid < 4) span[tid] = (tid & 1) ? (int)0x80000000 : 0x7fffffff;
  if (tid == 0) {
    any_bad = 0;
    first_token = it.n0;
  }
  __syncthreads();
  if (tid < 16 * WM) {
    const RowsToken k = rows_token(P, it, row0 + min(tid, n_rows - 1), hk);
    row_tok[tid] = make_int4(k.n, k.head, k.p, k.lo);
    row_sc[tid] = make_int2(__float_as_int(k.sc), __float_as_int(k.slope));
    atomicMin(&span[0], k.lo);
    atomicMax(&span[1], k.lo);
    atomicMin(&span[2], k.p);
    atomicMax(&span[3], k.p);
  }
  __syncthreads();
  // the item's keys and this block's range of them
  const int first = P.cu_q ? min(span[0], it.base) : span[0], end_all = rows_end(P, it, span[3]);
  const int full_lo = span[1], full_hi = P.cu_q ? it.base : span[2] + 1;  // keys in between are seen by every row
  // equal ranges of whole tiles (an item's own: a short request's blocks are as short as each other)
  const int start = first / KT * KT, per = max((end_all - start + KT * P.splits - 1) / (KT * P.splits), 0) * KT, range0 = start + split * per;
  const int begin = max(first, range0), end = min(end_all, range0 + per);
  const int n_tiles = end > begin ? (end - range0 + KT - 1) / KT : 0;
  const int* table = P.block_table + (size_t)it.r * P.bt_stride;
  const int v_off = P.Hkv * P.page_size;  // rows between a key and its value

  auto k_tile = [&](int s) { return smem + s * 2 * T::BYTES; };
  auto scales_of = [&](int s) { return reinterpret_cast<float*>(smem + STAGES * 2 * T::BYTES + s * T::SCALE_BYTES); };
  // The cache row of key (tid & 63) of tile t, or -1 outside the range.
  auto find_row = [&](int t) {
    const int place = range0 + t * KT + (tid & 63);
    return t < n_tiles && place >= begin && place < end ? rows_cache_row(P, table, hk, place) : -1;
  };
  // Threads 0-63 know the keys' rows, threads 64-127 the values'.
  auto fetch_scale = [&](int row) { return F8 && row >= 0 ? (int)P.scales[row + (tid >> 6) * v_off] : 0; };
  auto put_scale = [&](int t, int byte) {
    if (!F8) return;
    float* sc = scales_of(t % STAGES);
    if (tid < KT) {
      sc[tid] = fp8_scale(byte);
    } else {
      const bool bad = byte == FP8_BAD;
      const int e = fp8_weight_byte(byte) - 127;
      sc[tid] = bad ? __int_as_float(0x7fc00000) : (float)e;
      sc[tid + KT] = bad ? 1.f : fp8_pow2(max(-60, min(60, -e)));
    }
  };
  auto fetch_tile = [&](int t, const int* rows) {
    if (t < n_tiles) {
      uint8_t* kt = k_tile(t % STAGES);
      const int c = tid % CH;
#pragma unroll
      for (int i = 0; i < KT * CH / 128; ++i) {
        const int j = tid / CH + i * (128 / CH), row = rows[j];
        const uint8_t* src = reinterpret_cast<const uint8_t*>(P.pages) + ((size_t)max(row, 0) * CH + c) * 16;
        const uint32_t dst = smem_u32(kt + chunk_at<CH>(j, c) * 16);
        cp_async16(dst, src, row >= 0);
        cp_async16(dst + T::BYTES, src + (row >= 0 ? (size_t)v_off * CH * 16 : 0), row >= 0);
      }
    }
    cp_async_commit();
  };

  // the first STAGES - 1 tiles
#pragma unroll 1
  for (int t = 0; t < STAGES - 1; ++t) {
    const int row = find_row(t);
    if (tid < KT) row_of[t & 1][tid] = row;
    put_scale(t, fetch_scale(row));
    __syncthreads();
    fetch_tile(t, row_of[t & 1]);
  }
  int next_row = find_row(STAGES - 1);       // of the tile that the first round fetches
  int byte_of_last = 0;                       // scale byte of the tile fetched last round

  // queries, in the order of the scores' contraction
  const int wm = warp / WK, wk = warp % WK;
  const int r0 = wm * 16 + g, r1 = r0 + 8;
  const int4 tok0 = row_tok[r0], tok1 = row_tok[r1];
  float sc0 = __int_as_float(row_sc[r0].x), sc1 = __int_as_float(row_sc[r1].x);
  const float slope0 = __int_as_float(row_sc[r0].y), slope1 = __int_as_float(row_sc[r1].y);
  uint32_t qf[DH / 16][4];
  {
    const bf16* q0 = P.q + ((size_t)tok0.x * P.Hq + tok0.y) * DH;
    const bf16* q1 = P.q + ((size_t)tok1.x * P.Hq + tok1.y) * DH;
    if (F8) {
      uint4 a[DH / 64][2], b[DH / 64][2];
      float top0 = 0.f, top1 = 0.f;
#pragma unroll
      for (int i = 0; i < DH / 64; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          a[i][u] = *reinterpret_cast<const uint4*>(q0 + i * 64 + t4 * 16 + u * 8);
          b[i][u] = *reinterpret_cast<const uint4*>(q1 + i * 64 + t4 * 16 + u * 8);
          const __nv_bfloat162* pa = reinterpret_cast<const __nv_bfloat162*>(&a[i][u]);
          const __nv_bfloat162* pb = reinterpret_cast<const __nv_bfloat162*>(&b[i][u]);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float2 fa = __bfloat1622float2(pa[x]), fb = __bfloat1622float2(pb[x]);
            top0 = fmaxf(top0, fmaxf(fabsf(fa.x), fabsf(fa.y)));
            top1 = fmaxf(top1, fmaxf(fabsf(fb.x), fabsf(fb.y)));
          }
        }
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1) {
        top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, x));
        top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, x));
      }
      // the row's power of two: its largest entry into [2^7, 2^8)
      const int e0 = max(min((int)(__float_as_uint(top0) >> 23) - 127, 120), -110) - 7;
      const int e1 = max(min((int)(__float_as_uint(top1) >> 23) - 127, 120), -110) - 7;
      const float in0 = fp8_pow2(-e0), in1 = fp8_pow2(-e1);
      sc0 *= fp8_pow2(e0);
      sc1 *= fp8_pow2(e1);
#pragma unroll
      for (int i = 0; i < DH / 64; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const __nv_bfloat162* pa = reinterpret_cast<const __nv_bfloat162*>(&a[i][w >> 1]) + (w & 1) * 2;
          const __nv_bfloat162* pb = reinterpret_cast<const __nv_bfloat162*>(&b[i][w >> 1]) + (w & 1) * 2;
          const float2 a0 = __bfloat1622float2(pa[0]), a1 = __bfloat1622float2(pa[1]);
          const float2 b0 = __bfloat1622float2(pb[0]), b1 = __bfloat1622float2(pb[1]);
          qf[i * 4 + w][0] = pack_f16(a0.x * in0, a0.y * in0);
          qf[i * 4 + w][1] = pack_f16(b0.x * in1, b0.y * in1);
          qf[i * 4 + w][2] = pack_f16(a1.x * in0, a1.y * in0);
          qf[i * 4 + w][3] = pack_f16(b1.x * in1, b1.y * in1);
        }
    } else {
#pragma unroll
      for (int s = 0; s < DH / 16; ++s) {
        qf[s][0] = *reinterpret_cast<const uint32_t*>(q0 + s * 16 + t4 * 2);
        qf[s][1] = *reinterpret_cast<const uint32_t*>(q1 + s * 16 + t4 * 2);
        qf[s][2] = *reinterpret_cast<const uint32_t*>(q0 + s * 16 + t4 * 2 + 8);
        qf[s][3] = *reinterpret_cast<const uint32_t*>(q1 + s * 16 + t4 * 2 + 8);
      }
    }
  }
  const bool capped = P.cap_log2 > 0.f, sloped = P.slopes != nullptr;
  float m[2] = {ROWS_NEG_BIG, ROWS_NEG_BIG}, l[2] = {0.f, 0.f};
  float o[DH / 8][4];
#pragma unroll
  for (int i = 0; i < DH / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

#pragma unroll 1
  for (int t = 0; t < n_tiles; ++t) {
    const int place0 = range0 + t * KT;
    const bool masked = place0 < full_lo || place0 + KT > min(full_hi, end) || place0 < begin;
    cp_async_wait<STAGES - 2>();  // tile t has landed
    uint8_t* kt = k_tile(t % STAGES);
    uint8_t* vt = kt + T::BYTES;
    if (!F8 && masked) {
      // a value that is not finite leaves the tile before the product (each thread looks at what it fetched itself)
      const int c = tid % CH;
#pragma unroll
      for (int i = 0; i < KT * CH / 128; ++i) {
        uint4* at = reinterpret_cast<uint4*>(vt + chunk_at<CH>(tid / CH + i * (128 / CH), c) * 16);
        uint32_t w[4] = {at->x, at->y, at->z, at->w};
        bool bad = false;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if ((w[u] & 0x7f80u) == 0x7f80u) { w[u] &= 0xffff0000u; bad = true; }
          if ((w[u] & 0x7f800000u) == 0x7f800000u) { w[u] &= 0xffffu; bad = true; }
        }
        if (bad) {
          *at = make_uint4(w[0], w[1], w[2], w[3]);
          any_bad = 1;
        }
      }
    }
    if (tid < KT) row_of[(t + STAGES - 1) & 1][tid] = next_row;
    if (t > 0) put_scale(t + STAGES - 2, byte_of_last);
    __syncthreads();
    fetch_tile(t + STAGES - 1, row_of[(t + STAGES - 1) & 1]);
    byte_of_last = fetch_scale(next_row);
    next_row = find_row(t + STAGES);

    // ---- scores of this warp's keys
    const int key0 = wk * NK;
    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
    if (F8) {
#pragma unroll
      for (int b = 0; b < DH / 64; ++b)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const uint4 c = *reinterpret_cast<const uint4*>(kt + chunk_at<CH>(key0 + i * 8 + g, b * 4 + t4) * 16);
          uint32_t lo, hi;
          fp8x4_to_half(c.x, lo, hi);
          mma_f16(s[i], qf[b * 4], lo, hi);
          fp8x4_to_half(c.y, lo, hi);
          mma_f16(s[i], qf[b * 4 + 1], lo, hi);
          fp8x4_to_half(c.z, lo, hi);
          mma_f16(s[i], qf[b * 4 + 2], lo, hi);
          fp8x4_to_half(c.w, lo, hi);
          mma_f16(s[i], qf[b * 4 + 3], lo, hi);
        }
    } else {
#pragma unroll
      for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
        for (int np = 0; np < NT / 2; ++np) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4(smem_u32(kt + chunk_at<CH>(key0 + np * 16 + (lane >> 4) * 8 + (lane & 7), ks * 2 + ((lane >> 3) & 1)) * 16), b0, b1, b2, b3);
          mma_bf16(s[np * 2], qf[ks], b0, b1);
          mma_bf16(s[np * 2 + 1], qf[ks], b2, b3);
        }
    }
    // ---- base-2 exponents of the weights, and which of them count
    const float* sck = scales_of(t % STAGES) + key0 + t4 * 2;
    uint32_t seen = 0xffffffffu;
    float mx[2] = {m[0], m[1]};
    if (masked || sloped) seen = 0u;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float2 ks = F8 ? *reinterpret_cast<const float2*>(sck + i * 8) : make_float2(1.f, 1.f);
      const float2 ve = F8 ? *reinterpret_cast<const float2*>(sck + KT + i * 8) : make_float2(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = s[i][e] * (F8 ? (e < 2 ? sc0 : sc1) * ((e & 1) ? ks.y : ks.x) : (e < 2 ? sc0 : sc1));
        if (capped) x = x == x ? P.cap_log2 * cap_tanh(x) : x;
        if (masked || sloped) {
          int key_pos;
          const int4 tok = e < 2 ? tok0 : tok1;
          const int place = place0 + key0 + i * 8 + t4 * 2 + (e & 1);
          const bool sees = place >= begin && place < end && rows_sees(P, it, tok.x, tok.z, tok.w, place, key_pos);
          if (sees) {
            x = fmaf(-(e < 2 ? slope0 : slope1), (float)(tok.z - key_pos), x);
            seen |= 1u << (i * 4 + e);
          }
          x = sees ? x + (F8 ? ((e & 1) ? ve.y : ve.x) : 0.f) : ROWS_NEG_BIG;
        } else if (F8) {
          x += (e & 1) ? ve.y : ve.x;
        }
        s[i][e] = x;
        mx[e >> 1] = fmaxf(mx[e >> 1], x);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
    }
    const float corr[2] = {rows_exp2(m[0] - mx[0]), rows_exp2(m[1] - mx[1])};
    m[0] = mx[0];
    m[1] = mx[1];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float ref[2] = {F8 ? m[0] : m[0] + ROWS_HEADROOM, F8 ? m[1] : m[1] + ROWS_HEADROOM};
      const float2 vi = F8 ? *reinterpret_cast<const float2*>(sck + 2 * KT + i * 8) : make_float2(1.f, 1.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float w = (seen >> (i * 4 + e)) & 1 ? rows_exp2(s[i][e] - ref[e >> 1]) : 0.f;
        s[i][e] = w;
        sum[e >> 1] = F8 ? fmaf(w, (e & 1) ? vi.y : vi.x, sum[e >> 1]) : sum[e >> 1] + w;
      }
    }
    l[0] = fmaf(l[0], corr[0], sum[0]);
    l[1] = fmaf(l[1], corr[1], sum[1]);
    if (!__all_sync(0xffffffffu, corr[0] == 1.f && corr[1] == 1.f)) {
#pragma unroll
      for (int i = 0; i < DH / 8; ++i) {
        o[i][0] *= corr[0]; o[i][1] *= corr[0]; o[i][2] *= corr[1]; o[i][3] *= corr[1];
      }
    }
    // ---- weighted values
#pragma unroll
    for (int kp = 0; kp < NT / 2; ++kp) {
      uint32_t pa[4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          pa[u * 2 + h] = F8 ? pack_f16(s[kp * 2 + u][h * 2], s[kp * 2 + u][h * 2 + 1]) : pack_bf16(s[kp * 2 + u][h * 2], s[kp * 2 + u][h * 2 + 1]);
      const int key = key0 + kp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
      if (F8) {
        // o[2 c] / o[2 c + 1]: the even / odd entries of chunk c (16 entries)
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
          uint32_t r[4];
          ldmatrix_x4_trans(smem_u32(vt + chunk_at<CH>(key, c + (lane >> 4)) * 16), r[0], r[1], r[2], r[3]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t even0, odd0, even1, odd1;
            fp8x4_to_half(__byte_perm(r[2 * u], 0, 0x3120), even0, odd0);
            fp8x4_to_half(__byte_perm(r[2 * u + 1], 0, 0x3120), even1, odd1);
            mma_f16(o[(c + u) * 2], pa, even0, even1);
            mma_f16(o[(c + u) * 2 + 1], pa, odd0, odd1);
          }
        }
      } else {
#pragma unroll
        for (int np = 0; np < DH / 16; ++np) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4_trans(smem_u32(vt + chunk_at<CH>(key, np * 2 + (lane >> 4)) * 16), b0, b1, b2, b3);
          mma_bf16(o[np * 2], pa, b0, b1);
          mma_bf16(o[np * 2 + 1], pa, b2, b3);
        }
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
  }
  __syncthreads();  // the ring is free: the warps leave their rows in it

  float* rows_o = reinterpret_cast<float*>(smem);                       // [4 warps][16][LD]
  float2* rows_ml = reinterpret_cast<float2*>(smem + 4 * 16 * T::LD * 4);  // [4 warps][16]
  {
    float* a = rows_o + (size_t)(warp * 16 + g) * T::LD;
    float* b = a + 8 * T::LD;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) {
      if (F8) {
        *reinterpret_cast<float4*>(a + c * 16 + t4 * 4) = make_float4(o[2 * c][0], o[2 * c + 1][0], o[2 * c][1], o[2 * c + 1][1]);
        *reinterpret_cast<float4*>(b + c * 16 + t4 * 4) = make_float4(o[2 * c][2], o[2 * c + 1][2], o[2 * c][3], o[2 * c + 1][3]);
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          *reinterpret_cast<float2*>(a + c * 16 + u * 8 + t4 * 2) = make_float2(o[2 * c + u][0], o[2 * c + u][1]);
          *reinterpret_cast<float2*>(b + c * 16 + u * 8 + t4 * 2) = make_float2(o[2 * c + u][2], o[2 * c + u][3]);
        }
      }
    }
    if (t4 == 0) {
      rows_ml[warp * 16 + g] = make_float2(F8 ? m[0] : m[0] + ROWS_HEADROOM, l[0]);
      rows_ml[warp * 16 + g + 8] = make_float2(F8 ? m[1] : m[1] + ROWS_HEADROOM, l[1]);
    }
  }
  __syncthreads();
  const int part_shift = P.splits > 1 ? rows_part_shift(P, blockIdx.x / P.splits, first_token) : 0;
  for (int idx = tid; idx < n_rows * (DH / 4); idx += 128) {
    const int row = idx / (DH / 4), d = (idx - row * (DH / 4)) * 4, w0 = (row >> 4) * WK, i = row & 15;
    float mm = ROWS_NEG_BIG, ll = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) mm = fmaxf(mm, rows_ml[(w0 + w) * 16 + i].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float2 ml = rows_ml[(w0 + w) * 16 + i];
      const float f = ml.x == mm ? 1.f : rows_exp2(ml.x - mm);  // (infinite maxima: the others count for nothing)
      const float4 v = *reinterpret_cast<const float4*>(rows_o + (size_t)((w0 + w) * 16 + i) * T::LD + d);
      ll = fmaf(ml.y, f, ll);
      acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
    }
    const int4 tok = row_tok[row];
    if (!F8 && any_bad) {  // the values that were taken out, for the rows that see them
      for (int place = begin; place < end; ++place) {
        int key_pos;
        if (!rows_sees(P, it, tok.x, tok.z, tok.w, place, key_pos)) continue;
        if (place >= full_lo && place / KT * KT >= max(full_lo, begin) && place / KT * KT + KT <= min(full_hi, end)) continue;  // (a tile without masks kept them)
        const int row_c = rows_cache_row(P, table, hk, place);
        if (row_c < 0) continue;
        const bf16* v = reinterpret_cast<const bf16*>(P.pages) + (size_t)(row_c + v_off) * DH + d;
        const float x[4] = {__bfloat162float(v[0]), __bfloat162float(v[1]), __bfloat162float(v[2]), __bfloat162float(v[3])};
        if (!isfinite(x[0])) acc.x += x[0];
        if (!isfinite(x[1])) acc.y += x[1];
        if (!isfinite(x[2])) acc.z += x[2];
        if (!isfinite(x[3])) acc.w += x[3];
      }
    }
    const size_t at = (size_t)(tok.x + part_shift) * P.Hq + tok.y;
    if (P.splits > 1) {
      *reinterpret_cast<float4*>(P.part_o + (at * P.splits + split) * DH + d) = acc;
      if (d == 0) P.part_ml[at * P.splits + split] = make_float2(mm, ll);
    } else {
      const float inv = rows_inverse(P, mm, ll, tok.y);
      uint2 v;
      *reinterpret_cast<__nv_bfloat162*>(&v.x) = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
      *reinterpret_cast<__nv_bfloat162*>(&v.y) = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(P.out + at * DH + d) = v;
    }
  }
}

// -------------------------------------------------------------------------------------------- host
template <int DH, bool F8, int WM>
static int launch_rows(const RowsParams& P, dim3 grid, cudaStream_t stream) {
  constexpr int smem = RowsTile<DH, F8>::SMEM;
  static unsigned long long allowed = 0;  // a bit per device: the attribute belongs to the device's context
  int dev = 0;
  JLX_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(allowed >> dev & 1)) {
    JLX_CUDA(cudaFuncSetAttribute(attention_rows_kernel<DH, F8, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) allowed |= 1ull << dev;
  }
  JLX_CUDA(jlx_launch_pdl(attention_rows_kernel<DH, F8, WM>, grid, dim3(128), smem, stream, P));
  return 0;
}
template <int DH, bool F8>
static int launch_rows_of(const RowsParams& P, int max_count, cudaStream_t stream) {
  const int rows = max_count * (P.Hq / P.Hkv), per_block = rows <= 32 ? 32 : 64;
  const long long gx = (long long)P.n_items * P.splits, gy = (long long)P.Hkv * ((rows + per_block - 1) / per_block);
  JLX_REQUIRE(gx < (1ll << 31) && gy <= 65535, "attention over rows: too many items or rows");
  JLX_REQUIRE(P.splits == 1 || (P.part_o && P.part_ml), "attention over rows: scratch for the ranges is missing");
  const dim3 grid((unsigned)gx, (unsigned)gy);
  if (int rc = per_block == 32 ? launch_rows<DH, F8, 2>(P, grid, stream) : launch_rows<DH, F8, 4>(P, grid, stream)) return rc;
  return P.splits > 1 ? launch_rows_join<DH>(P, max_count, stream) : 0;
}

JLX_API int jlx_attention_rows(const RowsArgs* a, cudaStream_t stream) {
  RowsParams P;
  if (rows_params(*a, P)) return 1;
  if (P.n_items == 0) return 0;
  if (a->dh == 128) return a->scales ? launch_rows_of<128, true>(P, a->max_count, stream) : launch_rows_of<128, false>(P, a->max_count, stream);
  return a->scales ? launch_rows_of<64, true>(P, a->max_count, stream) : launch_rows_of<64, false>(P, a->max_count, stream);
}
