// The paged cache in 8 bits: quantising rows as they are written, and reading them back (fp8_rows.cuh has the format).
//
// Cache of one layer: pages[page][0 = K, 1 = V][kv head][slot in page][dh] of e4m3 codes, scales[page][0 / 1][kv head][slot]
// of scale bytes.  Token n of request r is held at its place: page block_table[r][place / page_size], slot place % page_size.
//
// A row of dh entries belongs to `lanes` neighbouring threads of a warp (the power of two that covers dh / 8), eight entries
// each: 16 bytes of bfloat16 (or 2 x 16 of float32) in, 8 bytes of codes out; the row's largest magnitude and the norm's sum
// of squares meet by shuffles, so a row is read once and nothing passes through shared memory but a token's angles.
// What bounds them: for a prompt's rows behind rotation and norm the issue slots (240 instructions a warp and two rows, 76 % of the
// rate: 4,096 tokens of 40 + 2 x 8 heads of 128 take 29 us, 3.7 TB/s; half the angles' loads kept in registers, packed arithmetic or
// six blocks a multiprocessor are slower: registers and the warps they cost); for plain writing and reading back the memory (7 us
// for the same tokens back); for a decode step's few rows the launch.
#include "fp8_rows.cuh"

struct KvFp8Params {
  uint8_t* pages;
  uint8_t* scales;
  const int* block_table;
  int bt_stride, n_requests;
  const int* req_of_token;
  const int* places;
  int N, Hkv, dh, page_size, num_pages, lanes;  // lanes, lanes_log2: the launcher's
  int* status;
  int lanes_log2;
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
  // magnitudes compare as whole numbers, and a NaN's is above infinity's
  uint32_t top = 0u;
  if (mine) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < P.lanes) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (!mine || !keep) return;
  const bool bad = top > __float_as_uint(FP8_LIMIT);
  const int e = bad ? 0 : fp8_row_exp(__uint_as_float(top));
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
  const int n = blockIdx.x, part = threadIdx.x & (P.lanes - 1), step = 256 >> P.lanes_log2;
  const long long row0 = kv_fp8_row(P, n);
  if (row0 < 0) {
    if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(P.status, JLX_STATUS_BAD_PAGE);
    return;
  }
  const int rows = 2 * P.Hkv;
  // (whole warps stay in the loop: the shuffles need every lane)
  for (int h0 = blockIdx.y * step; h0 < rows; h0 += gridDim.y * step) {
    const int h = h0 + (threadIdx.x >> P.lanes_log2);
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
//
// A block takes a token's rows TURNS at a time: their loads are issued together, the first ones before the angles are made, so
// that a prompt portion's blocks wait for memory once, not once per row and angle.  (TURNS 1 for partials, whose own loads are
// many, and for a decode step, whose rows lie in a block each.)
template <typename TI> struct Raw8 { float4 a, b; };
template <> struct Raw8<bf16> { uint4 a; };
template <typename TI> __device__ __forceinline__ void fetch8(const TI* p, bool wide, Raw8<TI>& r);
template <> __device__ __forceinline__ void fetch8<float>(const float* p, bool wide, Raw8<float>& r) {
  if (wide) {
    r.a = reinterpret_cast<const float4*>(p)[0];
    r.b = reinterpret_cast<const float4*>(p)[1];
  } else {
    r.a = make_float4(p[0], p[1], p[2], p[3]);
    r.b = make_float4(p[4], p[5], p[6], p[7]);
  }
}
template <> __device__ __forceinline__ void fetch8<bf16>(const bf16* p, bool wide, Raw8<bf16>& r) {
  if (wide) {
    r.a = *reinterpret_cast<const uint4*>(p);
  } else {
    uint32_t w[4];
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
    r.a = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float* f) {
  f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w; f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
}
__device__ __forceinline__ void unpack8(const Raw8<bf16>& r, float* f) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r.a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

template <typename TI, int TURNS>
__global__ void __launch_bounds__(256)
rope_kv_store_fp8_kernel(const TI* __restrict__ qkv, int splits, long long split_stride, bf16* __restrict__ q_out, const KvFp8Params P,
                         const int* __restrict__ positions, const float* __restrict__ inv_freq, int l2norm, float eps, int Hq, int wide) {
  JLX_TL(TL_ROPE);
  extern __shared__ float2 turn[];  // [dh / 2]: cosine and sine of this token's angles
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int n = blockIdx.x, part = threadIdx.x & (P.lanes - 1), step = 256 >> P.lanes_log2;
  const int rows = Hq + 2 * P.Hkv, mine_h = (threadIdx.x >> P.lanes_log2);
  const bool entries = part * 8 < P.dh;
  const TI* src = qkv + (size_t)n * rows * P.dh + part * 8;
  Raw8<TI> raw[TURNS];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
      const int h = h0 + t * step + mine_h;
      if (h < rows && entries) fetch8<TI>(src + (size_t)h * P.dh, wide, raw[t]);
    }
  };
  fetch(blockIdx.y * TURNS * step);
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
  const float per_entry = 1.f / (float)P.dh;
  // (whole warps stay in the loop: the shuffles need every lane)
  for (int h0 = blockIdx.y * TURNS * step; h0 < rows; h0 += gridDim.y * TURNS * step) {
    if (h0 != blockIdx.y * TURNS * step) fetch(h0);
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
      const int h = h0 + t * step + mine_h;
      if (h0 + t * step >= rows) break;
      const bool mine = h < rows && entries, is_v = h >= Hq + P.Hkv;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (mine) {
        unpack8(raw[t], f);
        if (TURNS == 1) {
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
      }
      float ss = 0.f;
      if (mine && !is_v) {
        if (inv_freq) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float2 w = turn[part * 4 + u];
            const float a = f[2 * u], b = f[2 * u + 1];
            f[2 * u] = a * w.x - b * w.y;
            f[2 * u + 1] = b * w.x + a * w.y;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
      }
      if (l2norm) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          if (o < P.lanes) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (!is_v) {
          // (a Newton step on the reciprocal root, which is off by two units otherwise: fewer entries cross a rounding border)
          const float mean = fmaf(ss, per_entry, eps), root = rsqrtf(mean), step = fmaf(-mean * root, root, 1.f);
          const float inv = fabsf(step) < 1.f ? fmaf(0.5f * root, step, root) : root;  // (not of an infinite sum)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] *= inv;
        }
      }
      if (__any_sync(0xffffffffu, h >= Hq)) kv_fp8_write(P, row0 + (long long)(h - Hq) * P.page_size, part, mine, h >= Hq && row0 >= 0, f);
      if (mine && h < Hq) store8<bf16>(q_out + ((size_t)n * Hq + h) * P.dh + part * 8, wide, f);
    }
  }
}

// The rows at the listed places back as numbers: k, v [N, Hkv, dh] (zeros where a place has no page).  A block takes TOKENS
// tokens: the chain from a place to its codes (request, page, row) is walked for all of them at once.
template <typename T, int TOKENS>
__global__ void __launch_bounds__(256) kv_load_fp8_kernel(const KvFp8Params P, T* __restrict__ k, T* __restrict__ v, int wide) {
  JLX_TL(TL_OTHER);
  pdl_launch_dependents_if_small();
  pdl_wait();
  const int n0 = blockIdx.x * TOKENS, part = threadIdx.x & (P.lanes - 1), step = 256 >> P.lanes_log2;
  if (part * 8 >= P.dh) return;
  long long row0[TOKENS];
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    row0[t] = n0 + t < P.N ? kv_fp8_row(P, n0 + t) : -1;
    if (row0[t] < 0 && n0 + t < P.N && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(P.status, JLX_STATUS_BAD_PAGE);
  }
  for (int h = blockIdx.y * step + (threadIdx.x >> P.lanes_log2); h < 2 * P.Hkv; h += gridDim.y * step) {
    uint2 c[TOKENS];
    int b[TOKENS];
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      const long long row = row0[t] + (long long)h * P.page_size;
      c[t] = row0[t] >= 0 ? *reinterpret_cast<const uint2*>(P.pages + row * P.dh + part * 8) : make_uint2(0u, 0u);
      b[t] = row0[t] >= 0 ? P.scales[row] : 127;
    }
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      if (n0 + t >= P.N) break;
      const float s = fp8_scale(b[t]);
      float f[8];
      uint32_t w[4];
      fp8x4_to_half(c[t].x, w[0], w[1]);
      fp8x4_to_half(c[t].y, w[2], w[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = x.x * s;
        f[2 * i + 1] = x.y * s;
      }
      const size_t n = n0 + t;
      store8<T>((h < P.Hkv ? k + (n * P.Hkv + h) * P.dh : v + (n * P.Hkv + h - P.Hkv) * P.dh) + part * 8, wide, f);
    }
  }
}

// Rows that a block takes per turn, and how many blocks share a token: a turn each while the step is small.
static int kv_fp8_grid_y(int N, int rows, int lanes) {
  const int step = 256 / lanes, turns = (rows + step - 1) / step;
  return N >= 256 ? 1 : turns;
}

static int kv_fp8_check(const char* what, const KvFp8Params& P) {
  JLX_REQUIRE(P.N >= 0 && P.Hkv > 0 && P.page_size > 0 && P.num_pages > 0 && P.bt_stride > 0 && P.n_requests > 0, "%s: bad sizes", what);
  JLX_REQUIRE(P.dh >= 8 && P.dh <= 256 && P.dh % 8 == 0, "%s: head size %d (a multiple of 8 up to 256)", what, P.dh);
  JLX_REQUIRE(((uintptr_t)P.pages & 7) == 0, "%s: the pages must start on an 8-byte boundary", what);
  JLX_REQUIRE(P.Hkv <= 65535 / 2, "%s: too many heads", what);
  return 0;
}

static int lanes_of(int dh, int* log2) {
  *log2 = 0;
  while ((8 << *log2) < dh) ++*log2;
  return 1 << *log2;
}

// `cache`: what kernels/api.py fills in, but for the lanes.
JLX_API int jlx_kv_store_fp8(const KvFp8Params* cache, const void* k, const void* v, int dtype, cudaStream_t stream) {
  KvFp8Params P = *cache;
  if (kv_fp8_check("kv_store_fp8", P)) return 1;
  if (P.N == 0) return 0;
  P.lanes = lanes_of(P.dh, &P.lanes_log2);
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
  P.lanes = lanes_of(P.dh, &P.lanes_log2);
  const int wide = (((uintptr_t)a->qkv | (uintptr_t)a->q_out) & 15) == 0 && a->split_stride % 4 == 0;
  const size_t smem = (size_t)P.dh / 2 * sizeof(float2);
  const int gy = kv_fp8_grid_y(P.N, a->Hq + 2 * P.Hkv, P.lanes);
  JLX_DISPATCH_DTYPE(a->in_dtype, TI, {
    auto kernel = gy == 1 && a->splits == 1 ? rope_kv_store_fp8_kernel<TI, 4> : rope_kv_store_fp8_kernel<TI, 1>;
    JLX_CUDA(jlx_launch_pdl(kernel, dim3(P.N, gy), dim3(256), smem, stream, (const TI*)a->qkv, a->splits, a->split_stride, (bf16*)a->q_out, P, a->positions,
                            a->inv_freq, a->l2norm, a->eps, a->Hq, wide));
  });
  return 0;
}

JLX_API int jlx_kv_load_fp8(const KvFp8Params* cache, void* k, void* v, int dtype, cudaStream_t stream) {
  KvFp8Params P = *cache;
  if (kv_fp8_check("kv_load_fp8", P)) return 1;
  if (P.N == 0) return 0;
  P.lanes = lanes_of(P.dh, &P.lanes_log2);
  const int wide = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
  JLX_DISPATCH_DTYPE(dtype, T, {
    const int gy = kv_fp8_grid_y(P.N, 2 * P.Hkv, P.lanes);
    if (P.N >= 1024) JLX_CUDA(jlx_launch_pdl(kv_load_fp8_kernel<T, 4>, dim3((P.N + 3) / 4, gy), dim3(256), 0, stream, P, (T*)k, (T*)v, wide));
    else JLX_CUDA(jlx_launch_pdl(kv_load_fp8_kernel<T, 1>, dim3(P.N, gy), dim3(256), 0, stream, P, (T*)k, (T*)v, wide));
  });
  return 0;
}
