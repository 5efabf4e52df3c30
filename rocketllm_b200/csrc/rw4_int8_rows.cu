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
// through the reductions (sum of squares, maximum) until its codes are written.  A thread holds NV
// vectors of 8 values; a row belongs to one warp (up to 1024 values), to a CTA of up to 512 threads
// (up to 16384), or to a thread-block cluster of up to 8 CTAs that joins its sums through
// distributed shared memory (up to 131056): no row is read twice.
//
// Rows of any length and alignment: the vectors of a row start where its codes reach an 8-byte
// boundary, so its first and last vectors may be partial (read and written value by value).  An
// input whose vectors then do not start on 16 bytes (the row stride is its own, a norm's weight has
// none) is read as the two or three aligned 16-byte granules around each vector, shifted together.
#include <cooperative_groups.h>

#include <climits>
#include <cstdlib>

#include "rw4_common.cuh"

namespace cg = cooperative_groups;

namespace {

using rw4::fail;

constexpr int kMaxThreads = 512;
constexpr int kVec = 8;                       // values a thread takes at a time
// the widest row of rw4_int8_linear; 8 CTAs x 512 threads x 4 vectors of 8 hold it at any alignment
constexpr int64_t kMaxK = 131056;
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
  int64_t x_ld, second_ld, M;
  int K;
  float eps;
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

// Sums in a fixed order (the result does not change from run to run).
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float block_sum(float v, float* part) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  return warp_sum((threadIdx.x & 31) < nw ? part[threadIdx.x & 31] : 0.f);
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* part) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  v = (threadIdx.x & 31) < nw ? part[threadIdx.x & 31] : 0u;
  return __reduce_max_sync(0xffffffffu, v);
}

__device__ __forceinline__ uint4 load_cached(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Eight values of a row as their inputs' type holds them (16 or 32 bytes of registers).
template <typename T>
struct Held {
  static constexpr int kQuads = sizeof(T) / 2;
  uint4 u[kQuads];
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    } else {
      unpack(u[0], v, T());
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    __align__(16) T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = from_f<T>(v[j]);
#pragma unroll
    for (int j = 0; j < kQuads; ++j) u[j] = reinterpret_cast<const uint4*>(t)[j];
  }
  // Values i .. i+7 of a row of K (0 outside it).  `shift`: bytes past a 16-byte boundary at
  // which every vector of this row starts; kKeep: the row is read again (kept in L1).
  template <bool kKeep>
  __device__ __forceinline__ void load(const T* row, int i, int K, int shift) {
    if (shift == 0 && i >= 0 && i + kVec <= K) {
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
        u[j] = kKeep ? load_cached(reinterpret_cast<const uint4*>(row + i) + j)
                     : load_once(reinterpret_cast<const uint4*>(row + i) + j);
    } else if (i >= kVec && i + 2 * kVec <= K) {
      // the granules around the vector lie inside the row; neighbouring threads share them (L1)
      const uint4* g = reinterpret_cast<const uint4*>(
          reinterpret_cast<const uint8_t*>(row + i) - shift);
      uint32_t w[4 * kQuads + 4];
#pragma unroll
      for (int j = 0; j <= kQuads; ++j) {
        const uint4 q = load_cached(g + j);
        w[4 * j] = q.x, w[4 * j + 1] = q.y, w[4 * j + 2] = q.z, w[4 * j + 3] = q.w;
      }
      if (shift & 8) {
#pragma unroll
        for (int j = 0; j < 4 * kQuads + 2; ++j) w[j] = w[j + 2];
      }
      if (shift & 4) {
#pragma unroll
        for (int j = 0; j < 4 * kQuads + 1; ++j) w[j] = w[j + 1];
      }
      if (sizeof(T) == 2 && (shift & 2)) {
#pragma unroll
        for (int j = 0; j < 4 * kQuads; ++j) w[j] = __byte_perm(w[j], w[j + 1], 0x5432);
      }
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
        u[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    } else {
      float v[8];
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[j] = i + j >= 0 && i + j < K ? to_f(row[i + j]) : 0.f;
      set(v);
    }
  }
  // `aligned`: every vector of this row starts on 16 bytes
  __device__ __forceinline__ void store(T* row, int i, int K, bool aligned) const {
    if (aligned && i >= 0 && i + kVec <= K) {
#pragma unroll
      for (int j = 0; j < kQuads; ++j) reinterpret_cast<uint4*>(row + i)[j] = u[j];
    } else {
      float v[8];
      get(v);
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j >= 0 && i + j < K) row[i + j] = from_f<T>(v[j]);
    }
  }
};

template <typename T>
__device__ __forceinline__ int shift_of(const T* p) {
  return static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
}

// max of the bit patterns of |v|
__device__ __forceinline__ uint32_t top_of(const float (&v)[8], uint32_t top) {
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  return top;
}

// who holds a row
enum Kind { kWarp = 0, kBlock = 1, kCluster = 2 };

template <typename T, int MODE, int NV, int KIND>
__global__ void __launch_bounds__(kMaxThreads, 2) rows_kernel(const RowArgs a) {
  __shared__ float fpart[16];
  __shared__ uint32_t upart[16];
  __shared__ float fjoin;
  __shared__ uint32_t ujoin;
  int rank = 0, parts = 1;
  if constexpr (KIND == kCluster) {
    rank = static_cast<int>(cg::this_cluster().block_rank());
    parts = static_cast<int>(cg::this_cluster().num_blocks());
  }
  const int64_t row = KIND == kWarp
                          ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)
                          : blockIdx.x / parts;
  if (KIND == kWarp && row >= a.M) return;
  const int K = a.K;
  int8_t* codes = a.codes + row * K;
  // this thread's vectors: base, base + step, ...  (consecutive threads, consecutive vectors),
  // from the 8-byte boundary at or before the row's first code
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(codes) & 7);
  const int step = (KIND == kWarp ? 32 : static_cast<int>(blockDim.x) * parts) * kVec;
  const int base = (KIND == kWarp ? static_cast<int>(threadIdx.x & 31)
                                  : rank * static_cast<int>(blockDim.x) +
                                        static_cast<int>(threadIdx.x)) * kVec - lead;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const T* second = static_cast<const T*>(a.second) + row * a.second_ld;
  const T* weight = static_cast<const T*>(a.weight);
  const int x_shift = shift_of(x - lead);

  pdl_enter();
  Held<T> h[NV];   // x, or the new residual stream
#pragma unroll
  for (int n = 0; n < NV; ++n)
    if (base + n * step < K) h[n].template load<false>(x, base + n * step, K, x_shift);
  // a norm's weight, which all rows share: early where registers allow
  constexpr bool kEarly = MODE >= kNorm && NV * sizeof(T) <= 4;
  Held<T> wt[kEarly ? NV : 1];
  const int w_shift = shift_of(weight - lead);
  if constexpr (kEarly) {
#pragma unroll
    for (int n = 0; n < NV; ++n)
      if (base + n * step < K) wt[n].template load<true>(weight, base + n * step, K, w_shift);
  }
  float y[NV][kVec];
  if constexpr (MODE == kGated || MODE == kNormRes) {
    const int s_shift = shift_of(second - lead);
    Held<T> s[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n)
      if (base + n * step < K) s[n].template load<false>(second, base + n * step, K, s_shift);
    T* hidden = static_cast<T*>(a.hidden) + row * K;
    const bool hidden_aligned = shift_of(hidden - lead) == 0;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = base + n * step;
      if (i >= K) continue;
      float v[8], g[8];
      h[n].get(v);
      s[n].get(g);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if constexpr (MODE == kGated)
          // positions outside the row hold 0 in both, and silu(0) * 0 = 0
          y[n][j] = v[j] * __fdividef(g[j], 1.f + __expf(-g[j]));
        else
          v[j] += g[j];
      }
      if constexpr (MODE == kNormRes) {
        h[n].set(v);
        h[n].store(hidden, i, K, hidden_aligned);
      }
    }
  }
  if constexpr (MODE >= kNorm) {
    float ss = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      if (base + n * step >= K) continue;
      float v[8];
      h[n].get(v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) ss = fmaf(v[j], v[j], ss);
    }
    ss = KIND == kWarp ? warp_sum(ss) : block_sum(ss, fpart);
    if constexpr (KIND == kCluster) {
      if (threadIdx.x == 0) fjoin = ss;
      cg::this_cluster().sync();
      ss = 0.f;
      for (int r = 0; r < parts; ++r) ss += *cg::this_cluster().map_shared_rank(&fjoin, r);
    }
    const float rs = rsqrtf(ss / static_cast<float>(K) + a.eps);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = base + n * step;
      if (i >= K) continue;
      float w[8];
      h[n].get(y[n]);
      if constexpr (kEarly) {
        wt[n].get(w);
      } else {
        wt[0].template load<true>(weight, i, K, w_shift);
        wt[0].get(w);
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        // outside the row: 0, not 0 * infinity
        y[n][j] = i + j >= 0 && i + j < K ? y[n][j] * rs * w[j] : 0.f;
    }
  } else if constexpr (MODE == kPlain) {
#pragma unroll
    for (int n = 0; n < NV; ++n) h[n].get(y[n]);
  }
  uint32_t top = 0;
#pragma unroll
  for (int n = 0; n < NV; ++n)
    if (base + n * step < K) top = top_of(y[n], top);
  top = KIND == kWarp ? __reduce_max_sync(0xffffffffu, top) : block_max(top, upart);
  if constexpr (KIND == kCluster) {
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
  if (rank == 0 && (KIND == kWarp ? threadIdx.x & 31 : threadIdx.x) == 0) a.scale[row] = scale;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int i = base + n * step;
    if (i >= K) continue;
    uint32_t lo = 0, hi = 0;
    if (!bad) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo |= code8(y[n][j] * inv) << (8 * j);
        hi |= code8(y[n][j + 4] * inv) << (8 * j);
      }
    }
    if (i >= 0 && i + kVec <= K) {
      *reinterpret_cast<uint2*>(codes + i) = make_uint2(lo, hi);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j >= 0 && i + j < K)
          codes[i + j] = static_cast<int8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
  }
  if constexpr (KIND == kCluster) cg::this_cluster().sync();  // all have read the others' sums
}

template <typename T, int MODE, int NV, int KIND>
int launch_rows(const RowArgs& a, int64_t blocks, int parts, int threads, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
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
  cfg.numAttrs = KIND == kCluster ? 2 : 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, rows_kernel<T, MODE, NV, KIND>, a);
  if (err != cudaSuccess) return rw4::cuda_status(err, "rw4 int8 rows launch");
  return rw4::launch_status("rw4 int8 rows launch");
}

template <typename T, int MODE>
int run_rows(const RowArgs& a, cudaStream_t stream) {
  // a row's vectors, with one more where it can start inside one
  const bool whole = a.K % kVec == 0 && rw4::aligned(a.codes, kVec);
  const int nvec = whole ? a.K / kVec : (a.K + 2 * (kVec - 1)) / kVec;
  if (nvec <= 128) {   // one warp a row, four rows a CTA
    const int64_t blocks = (a.M + 3) / 4;
    if (nvec <= 32) return launch_rows<T, MODE, 1, kWarp>(a, blocks, 1, 128, stream);
    if (nvec <= 64) return launch_rows<T, MODE, 2, kWarp>(a, blocks, 1, 128, stream);
    return launch_rows<T, MODE, 4, kWarp>(a, blocks, 1, 128, stream);
  }
  auto threads_for = [](int vecs, int nv) { return (((vecs + nv - 1) / nv) + 31) / 32 * 32; };
  static const int forced = getenv("RW4_ROWS_NV") ? atoi(getenv("RW4_ROWS_NV")) : 0;
  if (forced == 2 && nvec <= 2 * kMaxThreads)
    return launch_rows<T, MODE, 2, kBlock>(a, a.M, 1, threads_for(nvec, 2), stream);
  if (forced == 4 && nvec <= 4 * kMaxThreads)
    return launch_rows<T, MODE, 4, kBlock>(a, a.M, 1, threads_for(nvec, 4), stream);
  if (nvec <= kMaxThreads)
    return launch_rows<T, MODE, 1, kBlock>(a, a.M, 1, threads_for(nvec, 1), stream);
  if (nvec <= 2 * kMaxThreads)
    return launch_rows<T, MODE, 2, kBlock>(a, a.M, 1, threads_for(nvec, 2), stream);
  if (nvec <= 4 * kMaxThreads)
    return launch_rows<T, MODE, 4, kBlock>(a, a.M, 1, threads_for(nvec, 4), stream);
  static const int fnv = getenv("RW4_ROWS_CNV") ? atoi(getenv("RW4_ROWS_CNV")) : 4;
  int parts = 2;
  while (parts < 8 && nvec > parts * fnv * kMaxThreads) parts *= 2;
  if (fnv == 2 && nvec <= parts * 2 * kMaxThreads)
    return launch_rows<T, MODE, 2, kCluster>(a, a.M * parts, parts,
                                             threads_for((nvec + parts - 1) / parts, 2), stream);
  return launch_rows<T, MODE, 4, kCluster>(a, a.M * parts, parts,
                                           threads_for((nvec + parts - 1) / parts, 4), stream);
}

template <int MODE>
int run_rows_dtype(const RowArgs& a, int32_t dtype, cudaStream_t stream) {
  if (dtype == RW4_F32) return run_rows<float, MODE>(a, stream);
  if (dtype == RW4_F16) return run_rows<__half, MODE>(a, stream);
  return run_rows<__nv_bfloat16, MODE>(a, stream);
}

int elem_size(int32_t dtype) { return dtype == RW4_F32 ? 4 : 2; }

// The checks that every row entry point shares.
int check_rows(const char* who, int32_t dtype, int64_t M, int64_t K) {
  if (dtype != RW4_F32 && dtype != RW4_BF16 && dtype != RW4_F16)
    return fail(RW4_EINVAL, "%s: dtype %d (0 f32, 1 bf16, 2 f16)", who, dtype);
  if (M < 0 || M > INT_MAX / 8) return fail(RW4_EINVAL, "%s: %lld rows", who, (long long)M);
  if (K < 1 || K > kMaxK)
    return fail(RW4_EINVAL, "%s: rows of %lld values (1 to %lld)", who, (long long)K,
                (long long)kMaxK);
  if (M * K > (1ll << 40))   // (blocks are counted in 31 bits)
    return fail(RW4_EINVAL, "%s: %lld rows of %lld values", who, (long long)M, (long long)K);
  return RW4_OK;
}

// ---- codes -> values ---------------------------------------------------------------------------

constexpr int kDeqVec = 16;  // codes a thread: one 16-byte load, two (bf16 / fp16) or four stores

// The M x K codes as one run of M * K values (rows of any length: a vector may cross into the next
// row).  I: the type that counts them (a 64-bit division costs more than the rest of a vector).
template <typename T, typename I>
__global__ void __launch_bounds__(256)
    dequant_rows_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scale, I n, I K,
                        int vec, T* __restrict__ out) {
  pdl_enter();
  const I at = (static_cast<I>(blockIdx.x) * blockDim.x + threadIdx.x) * kDeqVec;
  if (at >= n) return;
  I row = at / K, left = K - (at - row * K);   // values left in the row, this one included
  float s = __ldg(scale + row);
  if (vec && n - at >= kDeqVec) {
    const uint4 u = load_once(codes + at);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    __align__(16) T t[kDeqVec];
    if (left >= kDeqVec) {
#pragma unroll
      for (int j = 0; j < kDeqVec; ++j)
        t[j] = from_f<T>(static_cast<float>(static_cast<int8_t>(w[j / 4] >> (8 * (j % 4)))) * s);
    } else {
#pragma unroll
      for (int j = 0; j < kDeqVec; ++j) {
        if (left == 0) {
          s = __ldg(scale + ++row);
          left = K;
        }
        --left;
        t[j] = from_f<T>(static_cast<float>(static_cast<int8_t>(w[j / 4] >> (8 * (j % 4)))) * s);
      }
    }
#pragma unroll
    for (int j = 0; j < kDeqVec * (int)sizeof(T) / 16; ++j)
      reinterpret_cast<uint4*>(out + at)[j] = reinterpret_cast<const uint4*>(t)[j];
  } else {
    for (I j = at; j < n && j < at + kDeqVec; ++j) {
      if (left == 0) {
        s = __ldg(scale + ++row);
        left = K;
      }
      --left;
      out[j] = from_f<T>(static_cast<float>(codes[j]) * s);
    }
  }
}

template <typename T>
int launch_dequant(const int8_t* codes, const float* scale, int64_t M, int64_t K, T* out,
                   cudaStream_t stream) {
  const int64_t n = M * K, threads = (n + kDeqVec - 1) / kDeqVec;
  const int vec = rw4::aligned(codes, 16) && rw4::aligned(out, 16);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((threads + 255) / 256));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // 32 bits count the values where the last thread's start does not pass them either
  const cudaError_t err =
      n < (1ll << 32) - 256 * kDeqVec
          ? cudaLaunchKernelEx(&cfg, dequant_rows_kernel<T, uint32_t>, codes, scale,
                               static_cast<uint32_t>(n), static_cast<uint32_t>(K), vec, out)
          : cudaLaunchKernelEx(&cfg, dequant_rows_kernel<T, uint64_t>, codes, scale,
                               static_cast<uint64_t>(n), static_cast<uint64_t>(K), vec, out);
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
  a.M = M;
  a.K = static_cast<int>(K);
  cudaStream_t s = rw4::as_stream(stream);
  return gate ? run_rows_dtype<kGated>(a, dtype, s) : run_rows_dtype<kPlain>(a, dtype, s);
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
  a.M = M;
  a.K = static_cast<int>(K);
  a.eps = eps;
  cudaStream_t s = rw4::as_stream(stream);
  return residual ? run_rows_dtype<kNormRes>(a, dtype, s) : run_rows_dtype<kNorm>(a, dtype, s);
}

extern "C" int rw4_int8_dequantize(const int8_t* codes, const float* scale, int64_t M, int64_t K,
                                   void* out, int32_t out_dtype, void* stream) {
  int st = check_rows("int8_dequantize", out_dtype, M, K);
  if (st != RW4_OK) return st;
  if (M == 0) return RW4_OK;
  if (!codes || !scale || !out) return fail(RW4_EINVAL, "int8_dequantize: null pointer");
  if (!rw4::aligned(out, elem_size(out_dtype)) || !rw4::aligned(scale, 4))
    return fail(RW4_EINVAL, "int8_dequantize: a pointer is not aligned to its type");
  cudaStream_t s = rw4::as_stream(stream);
  if (out_dtype == RW4_F32)
    return launch_dequant(codes, scale, M, K, static_cast<float*>(out), s);
  if (out_dtype == RW4_F16)
    return launch_dequant(codes, scale, M, K, static_cast<__half*>(out), s);
  return launch_dequant(codes, scale, M, K, static_cast<__nv_bfloat16*>(out), s);
}
