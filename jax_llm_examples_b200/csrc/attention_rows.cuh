// What the three kernels of attention over rows (attention_few.cu, attention_rows.cu, attention_rows_tc.cu) share.
//
// A work item is a stretch of a request's tokens; its query rows are (token, head of the KV head's group) pairs, token by
// token, row r = token * G + head: a tile of rows packs a few tokens' heads, so that one read of a key serves all of them.
//
//   causal: a token at position p sees the cached keys up to its own place p;
//   tree:   the request's tokens of this step are drafted ones, stored behind the `base` cached keys in the order of the step;
//           token i sees the cached keys and the drafted tokens j whose bit masks[i] holds.  A drafted key's position is its
//           token's, a cached key's is its place.
//   Both: and of these the keys at positions from start(p) = max(chunk ? p - p % chunk : 0, window ? p - window + 1 : 0) on.
//
//   s = scale temp(p) q.k (soft-capped: cap tanh(s / cap)) - slope (p - key position);   out = sum w v / (sum w + exp(sink)),
//   w = exp(s - max).  A row that sees nothing gives 0.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "fp8_rows.cuh"
#include "softcap.cuh"

#define ROWS_NEG_BIG (-1.0e30f)
// Over a bfloat16 cache, whose values may be as large as 32 bits go, a row's weights are at most 2^-ROWS_HEADROOM against the
// reference of its exponents: the sum of weighted values stays below the largest of them for 2^24 keys, and overflows no sooner
// than the average does.  (Values below 2^-100 lose digits by it.  Codes of 8 bits need none: they are below 2^69.)
#define ROWS_HEADROOM 24.0f
#define LOG2E 1.4426950408889634f

struct RowsParams {
  const bf16* q;           // [N, Hq, DH]
  const void* pages;       // [P, 2, Hkv, page, DH] bfloat16, or e4m3 codes
  const uint8_t* scales;   // [P, 2, Hkv, page] with codes
  const int* block_table;
  int bt_stride, n_requests, max_count;
  const int* req_of_token;
  const int* positions;
  bf16* out;               // [N, Hq, DH]
  const int* items;        // [n_items][2] = (first token row, count), one request each; null: single tokens
  const int* rows;         // single tokens: their token rows (null: 0 .. n_items - 1)
  int n_items;
  const int* cu_q;         // tree: [R + 1] the requests' first token rows (null: causal)
  const int* q_start;      // tree: [R] keys a request has cached before its drafted tokens
  const int* masks;        // tree: [N, words]
  int words;
  int N, Hq, Hkv, page_size, num_pages;
  float scale_log2;        // the score scale * log2(e); with a cap: the score scale / cap
  float cap_log2;          // cap * log2(e), 0: none
  int chunk, window;
  float attn_scale, floor_scale;
  const float* sink;       // [Hq] or null
  const float* slopes;     // [Hq] or null
  int splits;              // ranges that an item's keys are cut into
  float* part_o;           // [tokens, Hq, splits, DH]: sums of weighted values against the maximum
  float2* part_ml;         // [tokens, Hq, splits]: (maximum, sum of weights)
  int* status;
  // Tokens in the scratch: this many for every item, or (0) the step's N, whichever are fewer.  (Last in the list: in front of the
  // scratch's pointers it made one token behind 30,000 keys, joined from 48 ranges, 30.5 us for 26.)
  int part_items;
};

struct RowsItem {
  int n0, cnt, r, base, drafted;  // base: keys before the drafted tokens (causal: INT_MAX), drafted: their count
};

// The item's tokens, then its request; false: nothing to do (a description that points outside the step raises the status).
// What a kernel needs of the tokens alone (positions, queries) it asks for in between: a block's way to its first tile is a
// chain of dependent loads, of 700 cycles and more each.
__device__ __forceinline__ bool rows_tokens(const RowsParams& P, int i, RowsItem& it) {
  it.n0 = P.items ? P.items[2 * i] : (P.rows ? P.rows[i] : i);
  it.cnt = P.items ? P.items[2 * i + 1] : 1;
  if (it.cnt <= 0) return false;
  if (it.n0 < 0 || it.n0 > P.N - it.cnt || it.cnt > P.max_count) { atomicOr(P.status, JLX_STATUS_BAD_PAGE); return false; }
  return true;
}
// Keys that a request's row of the block table can hold.
__device__ __forceinline__ int rows_capacity(const RowsParams& P) { return (int)min((long long)P.bt_stride * P.page_size, 0x7f000000ll); }
__device__ __forceinline__ bool rows_request(const RowsParams& P, RowsItem& it) {
  it.r = P.req_of_token[it.n0];
  if (it.r < 0 || it.r >= P.n_requests) { atomicOr(P.status, JLX_STATUS_BAD_PAGE); return false; }
  it.base = P.cu_q ? P.q_start[it.r] : 0x7fffffff;
  it.drafted = 0;
  if (P.cu_q) {
    const int first = P.cu_q[it.r], end = P.cu_q[it.r + 1];
    if (first < 0 || end > P.N || it.n0 < first || it.n0 + it.cnt > end || it.base < 0 || it.base > rows_capacity(P) - (end - first)) { atomicOr(P.status, JLX_STATUS_BAD_PAGE); return false; }
    it.drafted = end - first;
  }
  return true;
}
__device__ __forceinline__ bool rows_item(const RowsParams& P, int i, RowsItem& it) { return rows_tokens(P, i, it) && rows_request(P, it); }

__device__ __forceinline__ int rows_first_key(const RowsParams& P, int p) {
  int s = 0;
  if (P.chunk > 0) s = p - p % P.chunk;
  if (P.window > 0) s = max(s, p - P.window + 1);
  return max(s, 0);
}

// The place behind the last key that the item's rows see (the highest of their positions is p_max).
__device__ __forceinline__ int rows_end(const RowsParams& P, const RowsItem& it, int p_max) {
  if (P.cu_q) return it.base + it.drafted;
  if (p_max < rows_capacity(P)) return p_max + 1;
  atomicOr(P.status, JLX_STATUS_BAD_PAGE);
  return rows_capacity(P);
}

// What a query row needs to know of its token.
struct RowsToken {
  int n, p, lo, head;
  float sc, slope;  // score factor and slope in base-2 units (with a cap: the factor of the cap's argument)
};
__device__ __forceinline__ RowsToken rows_token(const RowsParams& P, const RowsItem& it, int row, int hk) {
  const int G = P.Hq / P.Hkv, t = row / G;
  RowsToken k;
  k.n = it.n0 + t;
  k.head = hk * G + (row - t * G);
  k.p = P.positions[k.n];  // (by itself: what comes first waits for nothing else)
  k.lo = rows_first_key(P, k.p);
  k.sc = P.scale_log2;
  if (P.attn_scale != 0.f) k.sc *= 1.f + P.attn_scale * log1pf(floorf(((float)k.p + 1.f) / P.floor_scale));
  k.slope = P.slopes ? P.slopes[k.head] * LOG2E : 0.f;
  return k;
}

// Whether the row's token sees the key at `place`, and the key's position.
__device__ __forceinline__ bool rows_sees(const RowsParams& P, const RowsItem& it, int n, int p, int lo, int place, int& key_pos) {
  key_pos = place;
  if (!P.cu_q) return place >= lo && place <= p;
  if (place < it.base) return place >= lo;
  const int j = place - it.base;
  if (j >= it.drafted || j >= 32 * P.words) return false;
  key_pos = P.positions[P.cu_q[it.r] + j];
  return ((P.masks[(size_t)n * P.words + (j >> 5)] >> (j & 31)) & 1) && key_pos >= lo;
}

// Keys whose page the table does not name (below 0, or beyond the pool) raise the status where some row sees them, and are keys
// and values of zeros in every kernel: rows_cache_row says -1, a TMA box is asked for from page num_pages, behind the cache, where all
// it brings is zeros, and the scales' bytes are 0.
__device__ __forceinline__ bool rows_page_there(const RowsParams& P, int page) { return page >= 0 && page < P.num_pages; }

// The flat row of the key at `place` in the cache (values: Hkv * page_size further), or -1.
__device__ __forceinline__ int rows_cache_row(const RowsParams& P, const int* table, int hk, int place) {
  const int pi = place / P.page_size;
  const int page = pi < P.bt_stride ? table[pi] : -1;
  if (!rows_page_there(P, page)) { atomicOr(P.status, JLX_STATUS_BAD_PAGE); return -1; }
  return (page * 2 * P.Hkv + hk) * P.page_size + (place - pi * P.page_size);
}

__device__ __forceinline__ float rows_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a row's weighted sum is divided by, inverted: l against the maximum m, the sink's term with them.
__device__ __forceinline__ float rows_inverse(const RowsParams& P, float m, float l, int head) {
  if (P.sink) l += exp2f(P.sink[head] * LOG2E - m);  // (a row that sees nothing has m = NEG_BIG: the term is infinite, the row 0)
  return l == 0.f ? 0.f : 1.f / l;
}

// What is added to a token row of an item, whose tokens begin at n0, for its token in the scratch (of fewer tokens than the step).
__device__ __forceinline__ int rows_part_shift(const RowsParams& P, int item, int n0) { return P.part_items ? item * P.part_items - n0 : 0; }

// Joins the ranges of a row from scratch: a warp per row, DH / 32 entries a lane.
template <int DH>
__global__ void __launch_bounds__(256) attention_rows_join_kernel(const RowsParams P) {
  JLX_TL(TL_ATTN_COMBINE);
  pdl_launch_dependents_if_small();
  pdl_wait();
  RowsItem it;
  if (!rows_item(P, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (row >= it.cnt * P.Hq) return;
  const int head = row % P.Hq;
  const size_t at = (size_t)it.n0 * P.Hq + row, kept = (size_t)(it.n0 + rows_part_shift(P, blockIdx.x, it.n0)) * P.Hq + row;
  const float2* ml = P.part_ml + kept * P.splits;
  float m = ROWS_NEG_BIG;
  for (int s = lane; s < P.splits; s += 32) m = fmaxf(m, ml[s].x);
  m = warp_max(m);
  constexpr int E = DH / 32;
  float acc[E], l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.f;
  const float* po = P.part_o + kept * P.splits * DH + lane * E;
#pragma unroll 4
  for (int s = 0; s < P.splits; ++s) {
    const float2 x = ml[s];
    const float f = x.x == m ? 1.f : rows_exp2(x.x - m);
    l = fmaf(x.y, f, l);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = fmaf(po[(size_t)s * DH + i], f, acc[i]);
  }
  const float inv = rows_inverse(P, m, l, head);
#pragma unroll
  for (int i = 0; i < E; i += 2)
    *reinterpret_cast<__nv_bfloat162*>(P.out + at * DH + lane * E + i) = __floats2bfloat162_rn(acc[i] * inv, acc[i + 1] * inv);
}

// -------------------------------------------------------------------------------------------- host
// What the callers hand over (_ROWS_ARGS in kernels/api.py).
struct RowsArgs {
  const void *q, *pages, *scales, *block_table, *req_of_token, *positions, *out, *items, *rows, *cu_q, *q_start, *masks, *sink, *slopes, *part_o, *part_ml, *status;
  int bt_stride, n_requests, n_items, max_count, words, N, Hq, Hkv, dh, page_size, num_pages, chunk, window, splits, row_block, part_items;
  float scale, softcap, attn_scale, floor_scale;
};

static int rows_params(const RowsArgs& a, RowsParams& P) {
  JLX_REQUIRE(a.Hkv > 0 && a.Hq > 0 && a.Hq % a.Hkv == 0 && (a.dh == 64 || a.dh == 128), "attention over rows: %d query heads on %d of %d entries (64 or 128) are not supported", a.Hq, a.Hkv, a.dh);
  JLX_REQUIRE(a.N > 0 && a.n_items >= 0 && a.max_count > 0 && a.page_size > 0 && a.num_pages > 0 && a.bt_stride > 0 && a.n_requests > 0, "attention over rows: bad sizes");
  JLX_REQUIRE(((long long)a.num_pages + 1) * 2 * a.Hkv * a.page_size < (1ll << 31), "attention over rows: cache too large for 32-bit rows");
  JLX_REQUIRE((((uintptr_t)a.q | (uintptr_t)a.pages | (uintptr_t)a.out) & 15) == 0, "attention over rows: q, pages and out must be 16-byte aligned");
  JLX_REQUIRE(a.attn_scale == 0.f || a.floor_scale > 0.f, "attention: floor_scale must be positive");
  JLX_REQUIRE(a.softcap >= 0.f && a.chunk >= 0 && a.window >= 0, "attention: the score cap, chunk and window must not be negative (0: none)");
  JLX_REQUIRE(a.splits >= 1 && a.splits <= 4096, "attention over rows: %d ranges", a.splits);
  JLX_REQUIRE((((uintptr_t)a.part_o & 15) | ((uintptr_t)a.part_ml & 7)) == 0, "attention over rows: scratch for the ranges is not aligned");
  JLX_REQUIRE(a.part_items == 0 || a.part_items >= a.max_count, "attention over rows: the scratch holds %d tokens an item, of %d", a.part_items, a.max_count);
  JLX_REQUIRE(!a.cu_q == !a.masks && !a.cu_q == !a.q_start && (!a.cu_q || (a.items && a.words > 0)), "attention over rows: a tree needs its offsets, cached lengths, masks and items");
  JLX_REQUIRE((long long)a.max_count * a.Hq < (1ll << 30), "attention over rows: an item has too many rows");
  P.q = (const bf16*)a.q; P.pages = a.pages; P.scales = (const uint8_t*)a.scales; P.block_table = (const int*)a.block_table; P.bt_stride = a.bt_stride;
  P.n_requests = a.n_requests; P.max_count = a.max_count; P.req_of_token = (const int*)a.req_of_token; P.positions = (const int*)a.positions; P.out = (bf16*)a.out;
  P.items = (const int*)a.items; P.rows = (const int*)a.rows; P.n_items = a.n_items; P.cu_q = (const int*)a.cu_q; P.q_start = (const int*)a.q_start;
  P.masks = (const int*)a.masks; P.words = a.words; P.N = a.N; P.Hq = a.Hq; P.Hkv = a.Hkv; P.page_size = a.page_size; P.num_pages = a.num_pages;
  P.scale_log2 = a.softcap > 0.f ? a.scale / a.softcap : a.scale * LOG2E;
  P.cap_log2 = a.softcap > 0.f ? a.softcap * LOG2E : 0.f;
  P.chunk = a.chunk; P.window = a.window; P.attn_scale = a.attn_scale; P.floor_scale = a.floor_scale;
  P.sink = (const float*)a.sink; P.slopes = (const float*)a.slopes; P.splits = a.splits;
  P.part_items = a.part_items; P.part_o = (float*)a.part_o; P.part_ml = (float2*)a.part_ml; P.status = (int*)a.status;
  return 0;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The cache as rows of keys and values, in boxes of box_rows rows of up to 128 bytes, swizzled.
static int rows_map(const RowsParams& P, int dh, bool f8, int box_rows, CUtensorMap* map) {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = (EncodeTiledFn)p;
  }
  JLX_REQUIRE(fn != nullptr, "attention over rows: the driver does not offer cuTensorMapEncodeTiled");
  const int elem = f8 ? 1 : 2, inner = dh * elem < 128 ? dh : 128 / elem;
  const cuuint64_t dims[2] = {(cuuint64_t)dh, (cuuint64_t)P.num_pages * 2 * P.Hkv * P.page_size}, strides[1] = {(cuuint64_t)dh * elem};
  const cuuint32_t box[2] = {(cuuint32_t)inner, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  const CUresult r = fn(map, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(P.pages), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, inner * elem == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  JLX_REQUIRE(r == CUDA_SUCCESS, "attention over rows: the cache's tensor map failed (%d)", (int)r);
  return 0;
}

template <int DH>
static int launch_rows_join(const RowsParams& P, int max_count, cudaStream_t stream) {
  const long long jy = ((long long)max_count * P.Hq + 7) / 8;
  JLX_REQUIRE(jy <= 65535, "attention over rows: an item has too many rows to join");
  JLX_CUDA(jlx_launch_pdl(attention_rows_join_kernel<DH>, dim3(P.n_items, (unsigned)jy), dim3(256), 0, stream, P));
  return 0;
}
