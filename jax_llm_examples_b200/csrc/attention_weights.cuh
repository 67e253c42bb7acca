// What the kernels of the weights that cached keys receive share (attention_weights.cu, attention_weights_tc.cu).
//
//   out[r, h, j] = add[r, h, j] + sum over the request's query rows (token n of cu[r] .. cu[r + 1], head g of KV head h's group)
//   that see key j of  w = exp(s - lse),   lse = log(sum exp(s) (+ exp(sink))),   mask and s as in attention_rows.cuh (causal).
//
// Values are not read: what a cached key is worth keeping for is the weight it has had.
#pragma once
#include "attention_rows.cuh"

struct WeightsArgs {  // _WEIGHTS_ARGS in kernels/api.py
  const int* cu;       // [R + 1] the requests' first token rows
  const float* add;    // [R, Hkv, width] or null: zeros
  float* out;          // [R, Hkv, width]
  float* scratch;      // see the kernels
  int width, max_kv;   // max_kv: keys of the longest request
};

struct WeightsParams {
  RowsParams R;        // (its items, rows, cu_q, masks and parts are not used; max_count is the most tokens of a request)
  WeightsArgs W;
  int splits, buf_keys, rows, page_shift;  // rows: the most of a request and KV head; page_shift: the page size's logarithm, -1 if it is no power of two
};

// Request r's tokens; false: it has none, or they lie outside the step (the status says so).
__device__ __forceinline__ bool weights_request(const WeightsParams& P, int r, RowsItem& it) {
  it.r = r;
  it.n0 = P.W.cu[r];
  it.cnt = P.W.cu[r + 1] - it.n0;
  it.base = 0x7fffffff;
  it.drafted = 0;
  if (it.cnt == 0) return false;
  if (it.cnt < 0 || it.n0 < 0 || it.n0 > P.R.N - it.cnt || it.cnt > P.R.max_count) { atomicOr(P.R.status, JLX_STATUS_BAD_PAGE); return false; }
  return true;
}

// out = add at the places [from, to) of a row of both, `who` of `of` threads.
__device__ __forceinline__ void weights_copy(const WeightsParams& P, size_t row, int from, int to, int who, int of) {
  const float* add = P.W.add ? P.W.add + row * P.W.width : nullptr;
  float* out = P.W.out + row * P.W.width;
  if (add == out) return;
  for (int j = from + who; j < to; j += of) out[j] = add ? add[j] : 0.f;
}

// Two codes, each with its sign in the byte above, -> two bfloat16 numbers times 2^-120: a code's seven bits are a bfloat16 number's
// exponent and mantissa but for that factor, which a product in bfloat16 takes out exactly.
__device__ __forceinline__ uint32_t weights_widen(uint32_t x, uint32_t select) {
  uint32_t y;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(y) : "r"(x), "r"(select));
  y = (y << 4) & 0x87f087f0u;
  const uint32_t f = 0x7b807b80u;  // 2^120
  const __nv_bfloat162 z = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&y), *reinterpret_cast<const __nv_bfloat162*>(&f));
  return *reinterpret_cast<const uint32_t*>(&z);
}

// tanh for capped scores, whose weights go out in 32 bits (the other attention kernels round theirs to 16 and take softcap.cuh's):
// |x| <= 1: x p(x^2), p of degree 7 with the smallest largest relative error against tanh(x) / x on [0, 1] (fitted by iteratively
// reweighted least squares in a Chebyshev basis: 4.2e-9, 1.1e-7 with its roundings); beyond as there.
__device__ __forceinline__ float weights_tanh(float x) {
  const float u = x * x;
  float p = fmaf(-0.00035334538551978767f, u, 0.0022822292521595955f);
  p = fmaf(p, u, -0.007917444221675396f);
  p = fmaf(p, u, 0.021464819088578224f);
  p = fmaf(p, u, -0.05387091264128685f);
  p = fmaf(p, u, 0.1333215981721878f);
  p = fmaf(p, u, -0.33333277702331543f);
  p = fmaf(p, u, 1.f);
  return fabsf(x) <= 1.f ? p * x : cap_tanh_large(x);
}
