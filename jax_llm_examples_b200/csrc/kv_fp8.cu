// The paged cache in 8 bits: quantising rows as they are written, and reading them back (fp8_rows.cuh has the format).
//
// Cache of one layer: pages[page][0 = K, 1 = V][kv head][slot in page][dh] of e4m3 codes, scales[page][0 / 1][kv head][slot]
// of scale bytes.  Token n of request r is held at its place: page block_table[r][place / page_size], slot place % page_size.
//
// A row of dh entries belongs to `lanes` neighbouring threads of a warp (the power of two that covers dh / 8), eight entries
// each: 16 bytes of bfloat16 (or 2 x 16 of float32) in, 8 bytes of codes out; the row's largest magnitude and the norm's sum
// of squares meet by shuffles, so a row is read once and nothing passes through shared memory but a token's angles.
// Both directions move bytes and little else: what bounds them is the memory, and for a decode step's few rows the launch.
#include "fp8_rows.cuh"

struct KvFp8Params {
  uint8_t* pages;
  uint8_t* scales;
  const int* block_table;
  int bt_stride, n_requests;
  const int* req_of_token;
  const int* places;
  int N, Hkv, dh, page_size, num_pages, lanes;
  int* status;
};

// The flat index of token n's key row of head 0 (rows of page_size slots per head; values Hkv * page_size further), or -1.
__device__ __forceinline__ long long kv_fp8_row(const KvFp8Params& P, int n) {
  const int place = P.places[n], r = P.req_of_token[n];
  if (place < 0 || r < 0 || r >= P.n_requests) return -1;
  const int pi = place / P.page_size;
  if (pi >= P.bt_stride) return -1;
  const int page = P.block_table[(size_t)r * P.bt_stride + pi];
  if (page < 0 || page >= P.num_pages) return -1;
  return (long long)page * 2 * P.Hkv * P.page_size + (place - pi * P.page_size);
}

template <typename T> __device__ __forceinline__ void load8(const T* p, bool wide, float* f);
template <> __device__ __forceinline__ void load8<float>(const float* p, bool wide, float* f) {
  if (wide) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = p[i];
  }
}
template <> __device__ __forceinline__ void load8<bf16>(const bf16* p, bool wide, float* f) {
  if (wide) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __bfloat1622float2(h[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __bfloat162float(p[i]);
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, bool wide, const float* f);
template <> __device__ __forceinline__ void store8<float>(float* p, bool wide, const float* f) {
  if (wide) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = f[i];
  }
}
template <> __device__ __forceinline__ void store8<bf16>(bf16* p, bool wide, const float* f) {
  if (wide) {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(f[i]);
  }
}

// Eight entries of a row -> codes at `row` (flat), the scale byte by the row's first thread.  Every lane of the warp calls it;
// `mine`: the lane holds entries, `keep`: the row is written.
__device__ __forceinline__ void kv_fp8_write(const KvFp8Params& P, long long row, int part, bool mine, bool keep, const float* f) {
  float amax = 0.f;
  if (mine) {
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fabsf(f[i]) <= FP8_LIMIT ? fmaxf(amax, fabsf(f[i])) : INFINITY;  // (a NaN is not <=)
  }
  for (int o = P.lanes >> 1; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, amax, o);
    amax = fmaxf(amax, other);
  }
  if (!mine || !keep) return;
  const bool bad = amax > FP8_LIMIT;
  const int e = bad ? 0 : fp8_row_exp(amax);
  const float s = fp8_pow2(-e);
  uint2 c = make_uint2(0u, 0u);
  if (!bad) {
    c.x = fp8x4_from_float(f[0] * s, f[1] * s, f[2] * s, f[3] * s);
    c.y = fp8x4_from_float(f[4] * s, f[5] * s, f[6] * s, f[7] * s);
  }
  *reinterpret_cast<uint2*>(P.pages + row * P.dh + part * 8) = c;
  if (part == 0) P.scales[row] = (uint8_t)(bad ? FP8_BAD : e + 127);
}

// k, v: [N, Hkv, dh] (encoded already).  One block per token and stretch of rows.
template <typename T>
__global__ void __launch_bounds__(256) kv_store_fp8_kernel(const T* __restrict__ k, const T* __restrict__ v, const KvFp8Params P, int wide) {
  JLX_TL(TL_KV_STORE);
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int n = blockIdx.x, part = threadIdx.x % P.lanes, step = blockDim.x / P.lanes;
  const long long row0 = kv_fp8_row(P, n);
  if (row0 < 0) {
    if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(P.status, JLX_STATUS_BAD_PAGE);
    return;
  }
  const int rows = 2 * P.Hkv;
  // (whole warps stay in the loop: the shuffles need every lane)
  for (int h0 = blockIdx.y * step; h0 < rows; h0 += gridDim.y * step) {
    const int h = h0 + threadIdx.x / P.lanes;
    const bool mine = h < rows && part * 8 < P.dh;
    float f[8];
    if (mine) load8<T>((h < P.Hkv ? k + ((size_t)n * P.Hkv + h) * P.dh : v + ((size_t)n * P.Hkv + h - P.Hkv) * P.dh) + part * 8, wide, f);
    kv_fp8_write(P, row0 + (long long)h * P.page_size, part, mine, true, f);
  }
}

// qkv: projected rows [N, (Hq + 2 Hkv) dh], or `splits` float32 partials of them, added in order.  q and k turn in neighbouring
// pairs (2j, 2j + 1) by positions[n] * inv_freq[j] (null: not at all) and are divided by sqrt(mean(x^2) + eps) after it
// (l2norm); q goes to q_out, k and v into the cache, quantised from their 32-bit values.
//
// The angle is the product position * inv_freq carried with its rounding error: far positions lose nothing that the frequency
// itself has (the product alone is off by up to position * 2^-25 radians, 4e-3 at position 131072).
template <typename TI>
__global__ void __launch_bounds__(256)
rope_kv_store_fp8_kernel(const TI* __restrict__ qkv, int splits, long long split_stride, bf16* __restrict__ q_out, const KvFp8Params P,
                         const int* __restrict__ positions, const float* __restrict__ inv_freq, int l2norm, float eps, int Hq, int wide) {
  JLX_TL(TL_ROPE);
  extern __shared__ float2 turn[];  // [dh / 2]: cosine and sine of this token's angles
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int n = blockIdx.x, part = threadIdx.x % P.lanes, step = blockDim.x / P.lanes;
  const int rows = Hq + 2 * P.Hkv;
  const TI* src = qkv + (size_t)n * rows * P.dh + part * 8;
  const long long row0 = kv_fp8_row(P, n);
  if (row0 < 0 && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(P.status, JLX_STATUS_BAD_PAGE);
  if (inv_freq) {
    const float p = (float)positions[n];
    for (int j = threadIdx.x; j < P.dh >> 1; j += blockDim.x) {
      const float a = p * inv_freq[j], rest = fmaf(p, inv_freq[j], -a);
      float s, c;
      sincosf(a, &s, &c);
      turn[j] = make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
    }
    __syncthreads();
  }
  for (int h0 = blockIdx.y * step; h0 < rows; h0 += gridDim.y * step) {
    const int h = h0 + threadIdx.x / P.lanes;
    const bool mine = h < rows && part * 8 < P.dh, is_v = h >= Hq + P.Hkv;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (mine) {
      load8<TI>(src + (size_t)h * P.dh, wide, f);
      for (int z = 1; z < splits; z += 4) {  // partials four at a time: their loads are in flight together
        float g[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (z + u < splits) load8<TI>(src + (size_t)h * P.dh + (size_t)(z + u) * split_stride, wide, g[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (z + u < splits)
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] += g[u][i];
      }
    }
    float ss = 0.f;
    if (mine && !is_v) {
      if (inv_freq) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float2 t = turn[part * 4 + u];
          const float a = f[2 * u], b = f[2 * u + 1];
          f[2 * u] = a * t.x - b * t.y;
          f[2 * u + 1] = b * t.x + a * t.y;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
    }
    if (l2norm) {
      for (int o = P.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (!is_v) {
        const float inv = 1.f / sqrtf(ss / (float)P.dh + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= inv;
      }
    }
    kv_fp8_write(P, row0 + (long long)(h - Hq) * P.page_size, part, mine, h >= Hq && row0 >= 0, f);
    if (mine && h < Hq) store8<bf16>(q_out + ((size_t)n * Hq + h) * P.dh + part * 8, wide, f);
  }
}

// The rows at the listed places back as numbers: k, v [N, Hkv, dh] (zeros where a place has no page).
template <typename T>
__global__ void __launch_bounds__(256) kv_load_fp8_kernel(const KvFp8Params P, T* __restrict__ k, T* __restrict__ v, int wide) {
  JLX_TL(TL_OTHER);
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int n = blockIdx.x, part = threadIdx.x % P.lanes, step = blockDim.x / P.lanes;
  if (part * 8 >= P.dh) return;
  const long long row0 = kv_fp8_row(P, n);
  if (row0 < 0 && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(P.status, JLX_STATUS_BAD_PAGE);
  for (int h = blockIdx.y * step + threadIdx.x / P.lanes; h < 2 * P.Hkv; h += gridDim.y * step) {
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row0 >= 0) {
      const long long row = row0 + (long long)h * P.page_size;
      const uint2 c = *reinterpret_cast<const uint2*>(P.pages + row * P.dh + part * 8);
      const float s = fp8_scale(P.scales[row]);
      uint32_t w[4];
      fp8x4_to_half(c.x, w[0], w[1]);
      fp8x4_to_half(c.y, w[2], w[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = t.x * s;
        f[2 * i + 1] = t.y * s;
      }
    }
    store8<T>((h < P.Hkv ? k + ((size_t)n * P.Hkv + h) * P.dh : v + ((size_t)n * P.Hkv + h - P.Hkv) * P.dh) + part * 8, wide, f);
  }
}

// Rows that a block takes per turn, and how many blocks share a token: a turn each while the step is small.
static int kv_fp8_grid_y(int N, int rows, int lanes) {
  const int step = 256 / lanes, turns = (rows + step - 1) / step;
  return N >= 1024 ? 1 : turns;
}

static int kv_fp8_check(const char* what, const KvFp8Params& P) {
  JLX_REQUIRE(P.N >= 0 && P.Hkv > 0 && P.page_size > 0 && P.num_pages > 0 && P.bt_stride > 0 && P.n_requests > 0, "%s: bad sizes", what);
  JLX_REQUIRE(P.dh >= 8 && P.dh <= 256 && P.dh % 8 == 0, "%s: head size %d (a multiple of 8 up to 256)", what, P.dh);
  JLX_REQUIRE(((uintptr_t)P.pages & 7) == 0, "%s: the pages must start on an 8-byte boundary", what);
  JLX_REQUIRE(P.Hkv <= 65535 / 2, "%s: too many heads", what);
  return 0;
}

static int lanes_of(int dh) {
  int l = 1;
  while (l * 8 < dh) l *= 2;
  return l;
}

// `cache`: what kernels/api.py fills in, but for the lanes.
JLX_API int jlx_kv_store_fp8(const KvFp8Params* cache, const void* k, const void* v, int dtype, cudaStream_t stream) {
  KvFp8Params P = *cache;
  if (kv_fp8_check("kv_store_fp8", P)) return 1;
  if (P.N == 0) return 0;
  P.lanes = lanes_of(P.dh);
  const int wide = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
  JLX_DISPATCH_DTYPE(dtype, T, {
    JLX_CUDA(jlx_launch_pdl(kv_store_fp8_kernel<T>, dim3(P.N, kv_fp8_grid_y(P.N, 2 * P.Hkv, P.lanes)), dim3(256), 0, stream, (const T*)k, (const T*)v, P, wide));
  });
  return 0;
}

struct RopeFp8Args {
  const void* qkv;
  void* q_out;
  const int* positions;
  const float* inv_freq;
  long long split_stride;
  int in_dtype, splits, Hq, l2norm;
  float eps;
};

JLX_API int jlx_rope_kv_store_fp8(const KvFp8Params* cache, const RopeFp8Args* a, cudaStream_t stream) {
  KvFp8Params P = *cache;
  if (kv_fp8_check("rope_kv_store_fp8", P)) return 1;
  JLX_REQUIRE(a->Hq > 0 && a->Hq <= 65535, "rope_kv_store_fp8: bad head count %d", a->Hq);
  JLX_REQUIRE(a->splits >= 1 && (a->splits == 1 || a->in_dtype == JLX_F32), "rope_kv_store_fp8: split-K partials are float32");
  if (P.N == 0) return 0;
  P.lanes = lanes_of(P.dh);
  const int wide = (((uintptr_t)a->qkv | (uintptr_t)a->q_out) & 15) == 0 && a->split_stride % 4 == 0;
  const size_t smem = (size_t)P.dh / 2 * sizeof(float2);
  JLX_DISPATCH_DTYPE(a->in_dtype, TI, {
    JLX_CUDA(jlx_launch_pdl(rope_kv_store_fp8_kernel<TI>, dim3(P.N, kv_fp8_grid_y(P.N, a->Hq + 2 * P.Hkv, P.lanes)), dim3(256), smem, stream, (const TI*)a->qkv,
                            a->splits, a->split_stride, (bf16*)a->q_out, P, a->positions, a->inv_freq, a->l2norm, a->eps, a->Hq, wide));
  });
  return 0;
}

JLX_API int jlx_kv_load_fp8(const KvFp8Params* cache, void* k, void* v, int dtype, cudaStream_t stream) {
  KvFp8Params P = *cache;
  if (kv_fp8_check("kv_load_fp8", P)) return 1;
  if (P.N == 0) return 0;
  P.lanes = lanes_of(P.dh);
  const int wide = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
  JLX_DISPATCH_DTYPE(dtype, T, {
    JLX_CUDA(jlx_launch_pdl(kv_load_fp8_kernel<T>, dim3(P.N, kv_fp8_grid_y(P.N, 2 * P.Hkv, P.lanes)), dim3(256), 0, stream, P, (T*)k, (T*)v, wide));
  });
  return 0;
}
