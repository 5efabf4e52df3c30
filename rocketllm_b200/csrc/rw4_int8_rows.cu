// 8-bit rows for the W8A8 path: every kernel here turns one row of K values into K signed 8-bit
// codes and one fp32 scale, or back.
//
//   rw4_int8_quantize    y = x, or y = silu(gate) * x for the MLP product
//   rw4_int8_rmsnorm     h = round(x + residual), y = h * rsqrt(mean(h^2) + eps) * w, h stored
//   rw4_int8_dequantize  code * scale
//
// and for y:  a = max |y|,  scale = a / 127,  code = rint(y * (127 / a)), ties to even.  y stays in
// fp32 from the inputs to the code: one rounding, to 8 bits (a module-by-module model rounds the
// normed row and the product to bf16 first, which costs accuracy and saves nothing here).
//   - a row whose scale would be subnormal (a < 2^-119) is stored as scale 0 and codes 0: below it
//     127 / a overflows fp32;
//   - a row that holds a NaN or an infinity (in y) is stored as scale NaN and codes 0, so that
//     what reads the row is NaN instead of a finite number.  The maximum is taken over the bit
//     patterns of |y| as unsigned numbers, where NaN > infinity > every number, so that no
//     comparison drops a NaN.
//
// Memory-bound: each input is read once, in 16-byte loads, into registers, where the row stays
// through the reductions (sum of squares, maximum) until its codes are written.  A CTA of up to 512
// threads holds 8 * NV values a thread; rows beyond 16384 values are split over a thread-block
// cluster (up to 8 CTAs: K <= 131072) that joins the sums through distributed shared memory, so no
// row is read twice.  Rows whose address, stride or length is not a multiple of 8 values take
// scalar loads in the same layout.
#include <cooperative_groups.h>

#include <climits>
#include <cstdlib>

#include "rw4_common.cuh"

namespace cg = cooperative_groups;

namespace {

using rw4::fail;

constexpr int kMaxThreads = 512;
constexpr int kVec = 8;                       // values a thread takes at a time
constexpr int64_t kMaxK = 131072;             // 8 CTAs x 512 threads x 4 vectors of 8
constexpr uint32_t kTinyBits = 0x04000000u;   // 2^-119
constexpr uint32_t kInfBits = 0x7f800000u;

enum Mode { kPlain = 0, kGated = 1, kNorm = 2, kNormRes = 3 };

struct RowArgs {
  const void* x;
  const void* second;    // gate (kGated) or residual (kNormRes)
  const void* weight;    // kNorm / kNormRes
  void* hidden;          // kNormRes: the new residual stream
  int8_t* codes;
  float* scale;
  int64_t x_ld, second_ld;
  int K;
  float eps;
  int vec;               // 16-byte loads and 8-byte code stores are aligned
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// Data read once: not kept in L1.  (A plain load, not the read-only path: `hidden` may be the
// residual itself, which each thread reads before it writes.)
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ void unpack(const uint4& u, float (&v)[8], __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[8], __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Values i .. i+7 of a row of K (0 past its end).
template <typename T>
__device__ __forceinline__ void load8(const T* row, int i, int K, bool vec, float (&v)[8]) {
  if (vec && i + kVec <= K) {
    if constexpr (sizeof(T) == 4) {
      const uint4 a = load_once(row + i), b = load_once(row + i + 4);
      v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y);
      v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
      v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y);
      v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
    } else {
      unpack(load_once(row + i), v, T());
    }
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) v[j] = i + j < K ? to_f(row[i + j]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* row, int i, int K, bool vec, const float (&v)[8]) {
  if (vec && i + kVec <= K) {
    __align__(16) T t[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) t[j] = from_f<T>(v[j]);
#pragma unroll
    for (int j = 0; j < kVec * (int)sizeof(T) / 16; ++j)
      reinterpret_cast<uint4*>(row + i)[j] = reinterpret_cast<const uint4*>(t)[j];
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (i + j < K) row[i + j] = from_f<T>(v[j]);
  }
}

__device__ __forceinline__ uint32_t code8(float v) {
  int q;
  asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(q) : "f"(v));
  return (uint32_t)q & 0xffu;
}

// Start of a kernel under programmatic dependent launch: the previous grid's writes are waited
// for, then the next grid may be scheduled (it waits in the same way).
__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// The block's sum in a fixed order (the result does not change from run to run).
__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  v = (threadIdx.x & 31) < nw ? part[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* part) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  v = (threadIdx.x & 31) < nw ? part[threadIdx.x & 31] : 0u;
  return __reduce_max_sync(0xffffffffu, v);
}

template <typename T, int MODE, int NV, bool CLUSTER>
__global__ void __launch_bounds__(kMaxThreads) rows_kernel(const RowArgs a) {
  __shared__ float fpart[16];
  __shared__ uint32_t upart[16];
  __shared__ float fjoin;
  __shared__ uint32_t ujoin;
  int rank = 0, parts = 1;
  if constexpr (CLUSTER) {
    rank = static_cast<int>(cg::this_cluster().block_rank());
    parts = static_cast<int>(cg::this_cluster().num_blocks());
  }
  const int64_t row = CLUSTER ? blockIdx.x / parts : blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const T* second = static_cast<const T*>(a.second) + row * a.second_ld;
  const T* weight = static_cast<const T*>(a.weight);
  const bool vec = a.vec;
  // this thread's vectors: base, base + step, ...  (consecutive threads, consecutive vectors)
  const int step = blockDim.x * parts * kVec;
  const int base = (rank * blockDim.x + threadIdx.x) * kVec;

  pdl_enter();
  float y[NV][kVec];
  float w[MODE >= kNorm ? NV : 1][kVec];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int i = base + n * step;
    if (i < a.K) {
      load8(x, i, a.K, vec, y[n]);
      if constexpr (MODE >= kNorm) load8(weight, i, a.K, vec, w[n]);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) y[n][j] = 0.f;
    }
  }
  if constexpr (MODE == kGated || MODE == kNormRes) {
    float s[NV][kVec];
#pragma unroll
    for (int n = 0; n < NV; ++n)
      if (base + n * step < a.K) load8(second, base + n * step, a.K, vec, s[n]);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = base + n * step;
      if (i >= a.K) continue;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if constexpr (MODE == kGated)
          // positions past K hold 0 in both, and silu(0) * 0 = 0
          y[n][j] *= __fdividef(s[n][j], 1.f + __expf(-s[n][j]));
        else
          y[n][j] = to_f(from_f<T>(y[n][j] + s[n][j]));
      }
      if constexpr (MODE == kNormRes)
        store8(static_cast<T*>(a.hidden) + row * a.K, i, a.K, vec, y[n]);
    }
  }
  if constexpr (MODE >= kNorm) {
    float ss = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int j = 0; j < kVec; ++j) ss = fmaf(y[n][j], y[n][j], ss);
    ss = block_sum(ss, fpart);
    if constexpr (CLUSTER) {
      if (threadIdx.x == 0) fjoin = ss;
      cg::this_cluster().sync();
      ss = 0.f;
      for (int r = 0; r < parts; ++r) ss += *cg::this_cluster().map_shared_rank(&fjoin, r);
    }
    const float rs = rsqrtf(ss / static_cast<float>(a.K) + a.eps);
#pragma unroll
    for (int n = 0; n < NV; ++n)
      if (base + n * step < a.K)
#pragma unroll
        for (int j = 0; j < kVec; ++j) y[n][j] = y[n][j] * rs * w[n][j];
  }
  uint32_t top = 0;
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      // in a normed row, 0 * inf past K must not become a NaN of the row
      const bool in = MODE < kNorm || base + n * step + j < a.K;
      top = max(top, in ? __float_as_uint(y[n][j]) & 0x7fffffffu : 0u);
    }
  top = block_max(top, upart);
  if constexpr (CLUSTER) {
    if (threadIdx.x == 0) ujoin = top;
    cg::this_cluster().sync();
    for (int r = 0; r < parts; ++r) top = max(top, *cg::this_cluster().map_shared_rank(&ujoin, r));
  }
  const bool bad = top >= kInfBits;
  const float amax = __uint_as_float(top);
  float inv = 0.f, scale = 0.f;
  if (bad) {
    scale = __uint_as_float(0x7fc00000u);
  } else if (top >= kTinyBits) {
    scale = __fdiv_rn(amax, 127.f);
    inv = __fdiv_rn(127.f, amax);
  }
  if (threadIdx.x == 0 && rank == 0) a.scale[row] = scale;
  int8_t* codes = a.codes + row * a.K;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int i = base + n * step;
    if (i >= a.K) continue;
    uint32_t lo = 0, hi = 0;
    if (!bad) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo |= code8(y[n][j] * inv) << (8 * j);
        hi |= code8(y[n][j + 4] * inv) << (8 * j);
      }
    }
    if (vec && i + kVec <= a.K) {
      *reinterpret_cast<uint2*>(codes + i) = make_uint2(lo, hi);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j < a.K) codes[i + j] = static_cast<int8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
  }
  if constexpr (CLUSTER) cg::this_cluster().sync();  // every CTA has read the others' sums
}

template <typename T, int MODE, int NV, bool CLUSTER>
int launch_rows(const RowArgs& a, int64_t M, int parts, int threads, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(M * parts));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 2 : 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, rows_kernel<T, MODE, NV, CLUSTER>, a);
  if (err != cudaSuccess) return rw4::cuda_status(err, "rw4 int8 rows launch");
  return rw4::launch_status("rw4 int8 rows launch");
}

template <typename T, int MODE>
int run_rows(const RowArgs& a, int64_t M, cudaStream_t stream) {
  const int nvec = (a.K + kVec - 1) / kVec;
  auto threads_for = [](int vecs, int nv) { return (((vecs + nv - 1) / nv) + 31) / 32 * 32; };
  if (nvec <= kMaxThreads)
    return launch_rows<T, MODE, 1, false>(a, M, 1, threads_for(nvec, 1), stream);
  if (nvec <= 2 * kMaxThreads)
    return launch_rows<T, MODE, 2, false>(a, M, 1, threads_for(nvec, 2), stream);
  if (nvec <= 4 * kMaxThreads)
    return launch_rows<T, MODE, 4, false>(a, M, 1, threads_for(nvec, 4), stream);
  int parts = 2;
  while (parts < 8 && nvec > parts * 4 * kMaxThreads) parts *= 2;
  return launch_rows<T, MODE, 4, true>(a, M, parts, threads_for((nvec + parts - 1) / parts, 4),
                                       stream);
}

template <int MODE>
int run_rows_dtype(const RowArgs& a, int32_t dtype, int64_t M, cudaStream_t stream) {
  if (dtype == RW4_F32) return run_rows<float, MODE>(a, M, stream);
  if (dtype == RW4_F16) return run_rows<__half, MODE>(a, M, stream);
  return run_rows<__nv_bfloat16, MODE>(a, M, stream);
}

int elem_size(int32_t dtype) { return dtype == RW4_F32 ? 4 : 2; }

bool vec_ok(const void* p, int64_t ld, int es) {
  return rw4::aligned(p, 16) && (ld * es) % 16 == 0;
}

// The checks that every row entry point shares.
int check_rows(const char* who, int32_t dtype, int64_t M, int64_t K) {
  if (dtype != RW4_F32 && dtype != RW4_BF16 && dtype != RW4_F16)
    return fail(RW4_EINVAL, "%s: dtype %d (0 f32, 1 bf16, 2 f16)", who, dtype);
  if (M < 0 || M > INT_MAX / 8) return fail(RW4_EINVAL, "%s: %lld rows", who, (long long)M);
  if (K < 1 || K > kMaxK)
    return fail(RW4_EINVAL, "%s: rows of %lld values (1 to %lld)", who, (long long)K,
                (long long)kMaxK);
  return RW4_OK;
}

// ---- codes -> values ---------------------------------------------------------------------------

constexpr int kDeqVec = 16;  // codes a thread: one 16-byte load, two (bf16 / fp16) or four stores

template <typename T>
__global__ void __launch_bounds__(256)
    dequant_rows_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scale,
                        int64_t M, int K, int vec, T* __restrict__ out) {
  pdl_enter();
  const int i = (blockIdx.x * blockDim.x + threadIdx.x) * kDeqVec;
  if (i >= K) return;
  for (int64_t row = blockIdx.y; row < M; row += gridDim.y) {
    const int8_t* c = codes + row * K + i;
    T* o = out + row * K + i;
    const float s = __ldg(scale + row);
    if (vec && i + kDeqVec <= K) {
      const uint4 u = load_once(c);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      __align__(16) T t[kDeqVec];
#pragma unroll
      for (int j = 0; j < kDeqVec; ++j) {
        const int q = static_cast<int8_t>(w[j / 4] >> (8 * (j % 4)));
        t[j] = from_f<T>(static_cast<float>(q) * s);
      }
#pragma unroll
      for (int j = 0; j < kDeqVec * (int)sizeof(T) / 16; ++j)
        reinterpret_cast<uint4*>(o)[j] = reinterpret_cast<const uint4*>(t)[j];
    } else {
      for (int j = 0; j < kDeqVec && i + j < K; ++j) o[j] = from_f<T>(static_cast<float>(c[j]) * s);
    }
  }
}

template <typename T>
int launch_dequant(const int8_t* codes, const float* scale, int64_t M, int K, int vec, T* out,
                   cudaStream_t stream) {
  const int nvec = (K + kDeqVec - 1) / kDeqVec;
  const int threads = nvec >= 256 ? 256 : (nvec + 31) / 32 * 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((nvec + threads - 1) / threads, static_cast<unsigned>(M < 65535 ? M : 65535));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err =
      cudaLaunchKernelEx(&cfg, dequant_rows_kernel<T>, codes, scale, M, K, vec, out);
  if (err != cudaSuccess) return rw4::cuda_status(err, "rw4 int8 dequantize launch");
  return rw4::launch_status("rw4 int8 dequantize launch");
}

}  // namespace

extern "C" int rw4_int8_quantize(const void* x, int64_t x_stride, const void* gate,
                                 int64_t gate_stride, int32_t dtype, int64_t M, int64_t K,
                                 int8_t* codes, float* scale, void* stream) {
  int st = check_rows("int8_quantize", dtype, M, K);
  if (st != RW4_OK) return st;
  if (M == 0) return RW4_OK;
  if (!x || !codes || !scale) return fail(RW4_EINVAL, "int8_quantize: null pointer");
  const int es = elem_size(dtype);
  if (!rw4::aligned(x, es) || !rw4::aligned(gate, es) || !rw4::aligned(scale, 4))
    return fail(RW4_EINVAL, "int8_quantize: a pointer is not aligned to its type");
  if (M > 1 && (x_stride < 0 || (gate && gate_stride < 0)))
    return fail(RW4_EINVAL, "int8_quantize: negative row stride");
  RowArgs a = {};
  a.x = x;
  a.second = gate;
  a.codes = codes;
  a.scale = scale;
  a.x_ld = M > 1 ? x_stride : K;
  a.second_ld = M > 1 ? gate_stride : K;
  a.K = static_cast<int>(K);
  a.vec = K % kVec == 0 && vec_ok(x, M > 1 ? x_stride : 0, es) &&
          (!gate || vec_ok(gate, M > 1 ? gate_stride : 0, es)) && rw4::aligned(codes, 8);
  cudaStream_t s = rw4::as_stream(stream);
  return gate ? run_rows_dtype<kGated>(a, dtype, M, s) : run_rows_dtype<kPlain>(a, dtype, M, s);
}

extern "C" int rw4_int8_rmsnorm(const void* x, int64_t x_stride, const void* residual,
                                int64_t residual_stride, const void* weight, int32_t dtype,
                                int64_t M, int64_t K, float eps, void* hidden, int8_t* codes,
                                float* scale, void* stream) {
  int st = check_rows("int8_rmsnorm", dtype, M, K);
  if (st != RW4_OK) return st;
  if (!(eps >= 0.f)) return fail(RW4_EINVAL, "int8_rmsnorm: eps %g", eps);
  if (M == 0) return RW4_OK;
  if (!x || !weight || !codes || !scale) return fail(RW4_EINVAL, "int8_rmsnorm: null pointer");
  if (!residual != !hidden)
    return fail(RW4_EINVAL, "int8_rmsnorm: residual and hidden come together");
  const int es = elem_size(dtype);
  if (!rw4::aligned(x, es) || !rw4::aligned(residual, es) || !rw4::aligned(weight, es) ||
      !rw4::aligned(hidden, es) || !rw4::aligned(scale, 4))
    return fail(RW4_EINVAL, "int8_rmsnorm: a pointer is not aligned to its type");
  if (M > 1 && (x_stride < 0 || (residual && residual_stride < 0)))
    return fail(RW4_EINVAL, "int8_rmsnorm: negative row stride");
  RowArgs a = {};
  a.x = x;
  a.second = residual;
  a.weight = weight;
  a.hidden = hidden;
  a.codes = codes;
  a.scale = scale;
  a.x_ld = M > 1 ? x_stride : K;
  a.second_ld = M > 1 ? residual_stride : K;
  a.K = static_cast<int>(K);
  a.eps = eps;
  a.vec = K % kVec == 0 && vec_ok(x, M > 1 ? x_stride : 0, es) && rw4::aligned(weight, 16) &&
          (!residual || (vec_ok(residual, M > 1 ? residual_stride : 0, es) &&
                         rw4::aligned(hidden, 16))) &&
          rw4::aligned(codes, 8);
  cudaStream_t s = rw4::as_stream(stream);
  return residual ? run_rows_dtype<kNormRes>(a, dtype, M, s) : run_rows_dtype<kNorm>(a, dtype, M, s);
}

extern "C" int rw4_int8_dequantize(const int8_t* codes, const float* scale, int64_t M, int64_t K,
                                   void* out, int32_t out_dtype, void* stream) {
  int st = check_rows("int8_dequantize", out_dtype, M, K);
  if (st != RW4_OK) return st;
  if (M == 0) return RW4_OK;
  if (!codes || !scale || !out) return fail(RW4_EINVAL, "int8_dequantize: null pointer");
  if (!rw4::aligned(out, elem_size(out_dtype)) || !rw4::aligned(scale, 4))
    return fail(RW4_EINVAL, "int8_dequantize: a pointer is not aligned to its type");
  const int k = static_cast<int>(K);
  const int vec = K % kDeqVec == 0 && rw4::aligned(codes, 16) && rw4::aligned(out, 16);
  cudaStream_t s = rw4::as_stream(stream);
  if (out_dtype == RW4_F32)
    return launch_dequant(codes, scale, M, k, vec, static_cast<float*>(out), s);
  if (out_dtype == RW4_F16)
    return launch_dequant(codes, scale, M, k, vec, static_cast<__half*>(out), s);
  return launch_dequant(codes, scale, M, k, vec, static_cast<__nv_bfloat16*>(out), s);
}
