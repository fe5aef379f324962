// Activations kept in 8 bits: e4m3 codes with one power-of-two exponent for every 32 consecutive elements.
//
// See blocks8.cuh for the rule.
//
//   blocks_cast_kernel         x -> codes and exponents; with GELU also y = gelu(x) from the same read of x
//   blocks_uncast_kernel       codes and exponents -> values; with GELU dx = dy * gelu'(value), the values never written
#include "blocks8.cuh"

namespace {

constexpr int kThreads = 256;
using namespace blocks8;
constexpr int kUnroll = 2;    // vectors of a thread in flight
static inline bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

// 32 elements of any alignment, one per lane
template <typename T, bool GELU>
__device__ __forceinline__ void cast_block_by_lane(const T* x, T* y, uint8_t* codes, uint8_t* exps, int64_t n, int64_t blk) {
  const int lane = threadIdx.x & 31;
  const int64_t i = blk * kBlock + lane;
  const float v = i < n ? to_f32<T>(x[i]) : 0.0f;
  const int k = block_shift(__reduce_max_sync(0xffffffffu, finite_bits(v)));
  if (i < n) {
    codes[i] = f32_to_fp8<FMT_E4M3>(mul_keep(inf_to_nan(v), __uint_as_float((uint32_t)(k + 127) << 23)));
    if (GELU) y[i] = from_f32<T>(gelu_f(v));
  }
  if (lane == 0) exps[blk] = (uint8_t)(127 - k);
}

// A 32-byte vector of T: V elements, as 32-bit words of one or two.
template <typename T>
struct Vec {
  static constexpr int V = 32 / sizeof(T), L = kBlock / V;    // elements of a vector, lanes of a block
};
struct alignas(32) Bytes32 { uint32_t w[8]; };
__device__ __forceinline__ Bytes32 ld32(const void* p) {
  Bytes32 r;
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
               : "l"(p));
  return r;
}
__device__ __forceinline__ void st32(void* p, const Bytes32& r) {
  asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]), "r"(r.w[4]),
               "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7]), "l"(p)
               : "memory");
}
// The two elements of a word of 16-bit T
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&t);
}
template <typename T>
__device__ __forceinline__ void unpack(const Bytes32& raw, float (&v)[Vec<T>::V]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(raw.w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = unpack2(raw.w[j], T());
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ Bytes32 pack(const float (&v)[Vec<T>::V]) {
  Bytes32 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (sizeof(T) == 4) o.w[j] = __float_as_uint(v[j]);
    else                          o.w[j] = pack2(v[2 * j], v[2 * j + 1], T());
  }
  return o;
}
// Largest |x| of a vector as bits of fp32, from packed integer maxima (|x| as bits is monotone, with infinities and NaN on top)
template <typename T>
__device__ __forceinline__ uint32_t vector_amax(const Bytes32& raw) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (sizeof(T) == 4) m = max(m, raw.w[j] & 0x7fffffffu);
    else                m = __vmaxu2(m, raw.w[j] & 0x7fff7fffu);
  }
  if constexpr (sizeof(T) == 4) {
    return m;
  } else {
    m = max(m >> 16, m & 0xffffu);
    return __float_as_uint(unpack2(m, T()).x);
  }
}

// Bound by memory.  VEC: every pointer aligned for whole vectors of 32 bytes, so that a thread stores 16 codes at once and a warp 16 exponents;
// two vectors a thread and step are in flight, L lanes find the maximum of a block with log2(L) shuffles.  8192 x 16384 bf16, L2 flushed:
// 72 us (5.7 TB/s), with GeLU 120 us (5.6 TB/s); 16-byte vectors 84 and 128 us, one in flight 78 and 122 us, maxima of unpacked elements
// 110 and 154 us.  A copy of 537 MB runs at 6.1 TB/s.  A warp that sees an infinity or a NaN (its maxima are on top of all numbers) goes over its elements again.
template <typename T, bool GELU, bool VEC>
__global__ void __launch_bounds__(kThreads) blocks_cast_kernel(const T* __restrict__ x, T* __restrict__ y, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ exps, int64_t n) {
  const int64_t full = VEC ? n / kBlock : 0;    // blocks taken by vectors
  if constexpr (VEC) {
    constexpr int V = Vec<T>::V, L = Vec<T>::L, U = kUnroll;
    const int64_t nv = full * L;
    for (int64_t i0 = (int64_t)blockIdx.x * (kThreads * U) + threadIdx.x; i0 - threadIdx.x < nv; i0 += (int64_t)gridDim.x * (kThreads * U)) {
      Bytes32 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = i0 + u * kThreads < nv ? ld32(x + (i0 + u * kThreads) * V) : Bytes32{};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + u * kThreads;
        float v[V];
        unpack<T>(raw[u], v);
        uint32_t a = vector_amax<T>(raw[u]);
        float w[V];    // what is coded
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = v[j];
        if (__any_sync(0xffffffffu, a >= 0x7f800000u)) {
          a = 0;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            a = max(a, finite_bits(v[j]));
            w[j] = inf_to_nan(v[j]);
          }
        }
#pragma unroll
        for (int o = 1; o < L; o <<= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
        if (i >= nv) continue;
        const int k = block_shift(a);
        const float s = __uint_as_float((uint32_t)(k + 127) << 23);
        uint32_t c[V / 4];
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const uint32_t lo = f32x2_to_fp8x2<FMT_E4M3>(mul_keep(w[j], s), mul_keep(w[j + 1], s));
          const uint32_t hi = f32x2_to_fp8x2<FMT_E4M3>(mul_keep(w[j + 2], s), mul_keep(w[j + 3], s));
          c[j / 4] = lo | hi << 16;
        }
        if constexpr (V == 16) reinterpret_cast<uint4*>(codes)[i] = make_uint4(c[0], c[1], c[2], c[3]);
        else                   reinterpret_cast<uint2*>(codes)[i] = make_uint2(c[0], c[1]);
        if (threadIdx.x % L == 0) exps[i / L] = (uint8_t)(127 - k);
        if (GELU) {
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = gelu_f(v[j]);
          st32(y + i * V, pack<T>(v));
        }
      }
    }
  }
  const int64_t tid = (int64_t)blockIdx.x * kThreads + threadIdx.x, threads = (int64_t)gridDim.x * kThreads;
  const int64_t blocks = (n + kBlock - 1) / kBlock;
  for (int64_t b = full + tid / 32; b < blocks; b += threads / 32) cast_block_by_lane<T, GELU>(x, y, codes, exps, n, b);
}

template <typename T, bool GELU>
__device__ __forceinline__ T uncast_one(float v, T dy) {
  if (GELU) return from_f32<T>(to_f32<T>(dy) * gelu_grad_f(v));
  return from_f32<T>(in_range<T>(v));
}

// Bound by memory: two vectors a thread and step in flight.  8192 x 16384 bf16, L2 flushed: 75 us (5.4 TB/s), with the GeLU slope 123 us
// (5.5 TB/s); one vector in flight 74 and 143 us.
template <typename T, bool GELU, bool VEC>
__global__ void __launch_bounds__(kThreads) blocks_uncast_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                                                                 const T* __restrict__ dy, T* __restrict__ out, int64_t n) {
  constexpr int V = Vec<T>::V, L = Vec<T>::L, U = kUnroll;
  const int64_t nv = VEC ? n / V : 0;
  if constexpr (VEC) {
    for (int64_t i0 = (int64_t)blockIdx.x * (kThreads * U) + threadIdx.x; i0 < nv; i0 += (int64_t)gridDim.x * (kThreads * U)) {
      uint32_t c[U][V / 4], byte[U];
      Bytes32 g[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + u * kThreads;
        if (i >= nv) continue;
        if constexpr (V == 16) {
          const uint4 r = reinterpret_cast<const uint4*>(codes)[i];
          c[u][0] = r.x;
          c[u][1] = r.y;
          c[u][2] = r.z;
          c[u][3] = r.w;
        } else {
          const uint2 r = reinterpret_cast<const uint2*>(codes)[i];
          c[u][0] = r.x;
          c[u][1] = r.y;
        }
        byte[u] = exps[i / L];
        if (GELU) g[u] = ld32(dy + i * V);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + u * kThreads;
        if (i >= nv) continue;
        const float unit = block_unit(byte[u]);
        float v[V], d[V];
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c[u][j / 4] >> (8 * (j & 2))), __NV_E4M3);
          const float2 f = __half22float2(__half2(h));
          v[j] = mul_keep(f.x, unit);
          v[j + 1] = mul_keep(f.y, unit);
        }
        if (GELU) {
          unpack<T>(g[u], d);
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = d[j] * gelu_grad_f(v[j]);
        } else if (may_overflow<T>(byte[u])) {
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = in_range<T>(v[j]);
        }
        st32(out + i * V, pack<T>(v));
      }
    }
  }
  const int64_t tid = (int64_t)blockIdx.x * kThreads + threadIdx.x, threads = (int64_t)gridDim.x * kThreads;
  for (int64_t i = nv * V + tid; i < n; i += threads)
    out[i] = uncast_one<T, GELU>(mul_keep(fp8_to_f32<FMT_E4M3>(codes[i]), block_unit(exps[i / kBlock])), GELU ? dy[i] : T());
}

}    // namespace

// x -> codes [n], exps [ceil(n / 32)] and, where y is given, y = gelu(x) (tanh form) in the type of x.
MSAMP_API int msamp_blocks_cast(const void* x, void* y, void* codes, void* exps, int64_t n, int dtype, void* stream_) {
  if (n <= 0) return MSAMP_OK;
  MSAMP_REQUIRE(x && codes && exps, "blocks_cast: null pointer");
  cudaStream_t stream = (cudaStream_t)stream_;
  const bool vec = aligned32(x) && aligned32(codes) && (!y || aligned32(y));
  MSAMP_DISPATCH_HP(dtype, T, {
    const int grid = msamp_grid_for(vec ? (n * (int64_t)sizeof(T) + 32 * kUnroll - 1) / (32 * kUnroll) : n, kThreads, 8);
    if (vec && y)  blocks_cast_kernel<T, true, true><<<grid, kThreads, 0, stream>>>((const T*)x, (T*)y, (uint8_t*)codes, (uint8_t*)exps, n);
    else if (vec)  blocks_cast_kernel<T, false, true><<<grid, kThreads, 0, stream>>>((const T*)x, nullptr, (uint8_t*)codes, (uint8_t*)exps, n);
    else if (y)    blocks_cast_kernel<T, true, false><<<grid, kThreads, 0, stream>>>((const T*)x, (T*)y, (uint8_t*)codes, (uint8_t*)exps, n);
    else           blocks_cast_kernel<T, false, false><<<grid, kThreads, 0, stream>>>((const T*)x, nullptr, (uint8_t*)codes, (uint8_t*)exps, n);
  });
  return msamp_check_launch("msamp_blocks_cast");
}

// codes, exps -> out = values, or out = dy * gelu'(values) where dy is given; dtype is that of dy and out.
MSAMP_API int msamp_blocks_uncast(const void* codes, const void* exps, const void* dy, void* out, int64_t n, int dtype, void* stream_) {
  if (n <= 0) return MSAMP_OK;
  MSAMP_REQUIRE(codes && exps && out, "blocks_uncast: null pointer");
  cudaStream_t stream = (cudaStream_t)stream_;
  const bool vec = aligned32(codes) && aligned32(out) && (!dy || aligned32(dy));
  MSAMP_DISPATCH_HP(dtype, T, {
    const int grid = msamp_grid_for(vec ? (n * (int64_t)sizeof(T) + 32 * kUnroll - 1) / (32 * kUnroll) : n, kThreads, 8);
    const uint8_t *c = (const uint8_t*)codes, *e = (const uint8_t*)exps;
    if (vec && dy) blocks_uncast_kernel<T, true, true><<<grid, kThreads, 0, stream>>>(c, e, (const T*)dy, (T*)out, n);
    else if (vec)  blocks_uncast_kernel<T, false, true><<<grid, kThreads, 0, stream>>>(c, e, nullptr, (T*)out, n);
    else if (dy)   blocks_uncast_kernel<T, true, false><<<grid, kThreads, 0, stream>>>(c, e, (const T*)dy, (T*)out, n);
    else           blocks_uncast_kernel<T, false, false><<<grid, kThreads, 0, stream>>>(c, e, nullptr, (T*)out, n);
  });
  return msamp_check_launch("msamp_blocks_uncast");
}
