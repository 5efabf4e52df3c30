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
//   - In a norm, rsqrt(..) is one factor r of the whole row: code = rint(h w * (127 / max |h w|)) and
//     scale = r * max |h w| / 127, so the sum of squares and the maximum are taken in one pass and
//     joined across the row in one exchange, and no value is multiplied by r.  Rows whose squares or
//     products leave fp32 that way, though y does not, are taken again with h scaled (scaled_norm).
//   - A row whose scale would be subnormal (a below 2^-119) is stored as scale 0 and codes 0: below
//     it 127 / a overflows fp32.
//   - A row that holds a NaN or an infinity is stored as scale NaN and codes 0, so that what reads
//     the row is NaN instead of a finite number.  The maximum is the NaN-propagating one.
//   - Rounding to a code is the addition of 1.5 * 2^23 to the scaled value: the sum's low byte is the
//     code in two's complement, rounded to even.  (The conversion instruction runs at a quarter of
//     the rate, on the unit that also serves silu's exponential and reciprocal: with it swiglu
//     8192 x 8192 took 69 us, without it 56.)  The product is rounded to fp32 first: 16-bit rows
//     hold many values at an exact half of a code, 127 / a is rounded, and a fused multiply-add
//     would let that rounding's sign take the half up or down (one draw of 1001 x 5632 normal bf16
//     values has 18.7 thousand such ties: 3.8 thousand go to the odd code fused, 0.9 thousand so).
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

#include <atomic>
#include <climits>

#include "rw4_tma.cuh"

namespace cg = cooperative_groups;

namespace {

using namespace rw4;

constexpr int kMaxThreads = 512;
constexpr int kWarpThreads = 128;             // of a CTA whose warps hold a row each
constexpr int kVec = 8;                       // values a thread takes at a time
// the widest row of rw4_int8_linear; 8 CTAs x 512 threads x 4 vectors of 8 hold it at any alignment
constexpr int64_t kMaxK = 131056;
constexpr float kTiny = 1.504632769052528e-36f;   // 2^-119

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

// Start of a kernel under programmatic dependent launch: the previous grid's writes are waited
// for, then the next grid may be scheduled (it waits in the same way).
__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// max(top, |a|, |b|), a NaN if any is
__device__ __forceinline__ float top3(float top, float a, float b) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(top), "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float top_of(const float (&v)[8], float top) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) top = top3(top, v[j], v[j + 1]);
  return top;
}

// What the values of a row are reduced to.
struct RowSums {
  float top;   // max |y| (a norm's: max |h w|)
  float ss;    // a norm's sum of squares
};

// Over a warp, in a fixed order (the result does not change from run to run).  Bit patterns of
// magnitudes compare as unsigned numbers, a NaN above infinity.
template <int MODE>
__device__ __forceinline__ RowSums warp_sums(RowSums v) {
  v.top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v.top)));
  if (MODE >= kNorm) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v.ss += __shfl_xor_sync(0xffffffffu, v.ss, o);
  }
  return v;
}

// Over a CTA; `part` holds one entry a warp.  Two calls in a row take different `part`s (a fast
// warp's next entry must not replace one that a slow warp still reads).
template <int MODE>
__device__ __forceinline__ RowSums block_sums(RowSums v, RowSums* part) {
  v = warp_sums<MODE>(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sums<MODE>(lane < (blockDim.x >> 5) ? part[lane] : RowSums{0.f, 0.f});
}

__device__ __forceinline__ uint4 load_cached(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
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
  // the eight values that start `shift` bytes into kQuads + 1 granules
  __device__ __forceinline__ void take(uint32_t (&w)[4 * kQuads + 4], int shift) {
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
      take(w, shift);
    } else {
      float v[8];
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[j] = i + j >= 0 && i + j < K ? to_f(row[i + j]) : 0.f;
      set(v);
    }
  }
  __device__ __forceinline__ void load_shared(const T* p) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j) u[j] = reinterpret_cast<const uint4*>(p)[j];
  }
  // from shared memory, `shift` bytes past a 16-byte boundary
  __device__ __forceinline__ void load_shared_at(uint32_t addr, int shift) {
    if (shift == 0) {
#pragma unroll
      for (int j = 0; j < kQuads; ++j) u[j] = lds128(addr + 16 * j);
    } else {
      uint32_t w[4 * kQuads + 4];
#pragma unroll
      for (int j = 0; j <= kQuads; ++j) {
        const uint4 q = lds128(addr - shift + 16 * j);
        w[4 * j] = q.x, w[4 * j + 1] = q.y, w[4 * j + 2] = q.z, w[4 * j + 3] = q.w;
      }
      take(w, shift);
    }
  }
  // value by value
  __device__ __forceinline__ void load_values(const T* row, int i, int K) {
    float v[8];
#pragma unroll
    for (int j = 0; j < kVec; ++j) v[j] = i + j >= 0 && i + j < K ? to_f(row[i + j]) : 0.f;
    set(v);
  }
  // keep the values of positions i .. i+7 that lie in a row of K
  __device__ __forceinline__ void clip(int i, int K) {
    float v[8];
    get(v);
#pragma unroll
    for (int j = 0; j < kVec; ++j) v[j] = i + j >= 0 && i + j < K ? v[j] : 0.f;
    set(v);
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

struct RowScale {
  float scale, inv;
  bool bad;
};

// What a norm's root is taken of.
__device__ __forceinline__ float norm_mean(const RowSums& v, int K, float eps) {
  return v.ss / static_cast<float>(K) + eps;
}

// A row's scale, and the factor to its codes.  `bad`: the row is stored as scale NaN and codes 0,
// because it holds a NaN or an infinity or, in a norm, because its squares or its products h w are
// not finite or so small that codes would be taken from subnormal numbers; scaled_norm then takes
// it again.  (A mean from 2^-60 on keeps the factor below 2^30: products that vanish stand for values
// below 2^-119.)
template <int MODE>
__device__ __forceinline__ RowScale row_scale(const RowSums& v, int K, float eps) {
  float a = v.top;
  RowScale r = {0.f, 0.f, false};
  if constexpr (MODE >= kNorm) {
    const float mean = norm_mean(v, K, eps);
    a *= rsqrtf(mean);
    r.bad = !(mean < INFINITY) || mean < 0x1p-60f || (v.top < kTiny && v.top > 0.f);
  }
  r.bad |= !(a < INFINITY);
  if (r.bad) {
    r.scale = __uint_as_float(0x7fc00000u);
  } else if (a >= kTiny) {
    r.scale = __fdiv_rn(a, 127.f);
    r.inv = __fdiv_rn(127.f, v.top);
  }
  return r;
}

// Two values times `inv`, rounded to fp32, then to whole numbers in the low bytes.  (The additions of
// a pair are one operation on packed registers: one by one they cost the quantizer of 2048 x 28672
// values 28.6 us against 27.5.  The products are not packed: ptxas fuses a packed product and sum.)
__device__ __forceinline__ void round_pair(float a, float b, float inv, uint32_t& ca, uint32_t& cb) {
  asm("{\n .reg .b64 v, f;\n mov.b64 v, {%2, %3};\n mov.b64 f, {%4, %4};\n"
      " add.rn.f32x2 v, v, f;\n mov.b64 {%0, %1}, v;\n}\n"
      : "=r"(ca), "=r"(cb)
      : "f"(__fmul_rn(a, inv)), "f"(__fmul_rn(b, inv)), "f"(12582912.f));
}

// One code.
__device__ __forceinline__ int8_t code_of(float y, const RowScale& r) {
  return r.bad ? 0 : static_cast<int8_t>(__float_as_uint(__fadd_rn(__fmul_rn(y, r.inv), 12582912.f)));
}

// The codes of values i .. i+7 of a row of K (i on an 8-byte boundary of the codes).
__device__ __forceinline__ void store_codes(int8_t* codes, int i, int K, const float (&y)[8],
                                            const RowScale& r) {
  uint32_t lo = 0, hi = 0;
  if (!r.bad) {
    uint32_t c[8];   // the code in the low byte
#pragma unroll
    for (int j = 0; j < 8; j += 2) round_pair(y[j], y[j + 1], r.inv, c[j], c[j + 1]);
    lo = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    hi = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
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

// silu(g) * v = g / (1 + exp(-g)) * v, from h = exp(-|g| / 2) = 2^(-|g| log2(e) / 2): below zero
// silu(g) is g h^2 / (1 + h^2), so no power exceeds 1, the denominator lies in [1, 2], and with an h
// for each factor nothing underflows whose product does not (exp(-g) itself leaves fp32 at -88.7).
// The exponent is rounded to fp32, so the product is off by |g| 2^-24 relative (beside a few steps):
// 2^-20 at 16, 2^-17.5 at -88, which only rows without any other gate show.  Carrying the rounded-off
// part along cost swiglu 2048 x 28672 56.5 us against 53.5 here, expf and an approximate division
// 62.5, expf and an exact one 79.
__device__ __forceinline__ float gated(float v, float g) {
  float h, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(fabsf(g) * -0.72134752f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(h, h, 1.f)));
  const float s = g < 0.f ? h : 1.f;
  return (v * s) * ((g * s) * r);
}

// Eight values of a row: y (a norm's: h w) and, in a norm, their squares added to ss; `h` becomes
// the new residual stream.  Positions outside the row hold 0 everywhere and stay 0.
template <typename T, int MODE>
__device__ __forceinline__ void combine(Held<T>& h, const Held<T>& second, const Held<T>& weight,
                                        float (&y)[8], float& ss) {
  float t[8];
  h.get(y);
  if constexpr (MODE == kGated || MODE == kNormRes) {
    second.get(t);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = MODE == kGated ? gated(y[j], t[j]) : y[j] + t[j];
  }
  if constexpr (MODE == kNormRes) {
    h.set(y);
    h.get(y);
  }
  if constexpr (MODE >= kNorm) {
    weight.get(t);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = fmaf(y[j], y[j], ss);
      y[j] *= t[j];
    }
  }
}

// who holds a row
enum Kind { kWarp = 0, kBlock = 1, kCluster = 2 };

// The sums of all that hold a row, once more (`part` and `join` may still be read for the last).
template <int KIND>
__device__ __forceinline__ RowSums row_sums_again(RowSums v, RowSums* part, RowSums* join) {
  if constexpr (KIND == kWarp) return warp_sums<kNorm>(v);
  if constexpr (KIND == kBlock) __syncthreads();
  if constexpr (KIND == kCluster) cg::this_cluster().sync();
  v = block_sums<kNorm>(v, part);
  if constexpr (KIND == kCluster) {
    if (threadIdx.x == 0) *join = v;
    cg::this_cluster().sync();
    const int lane = threadIdx.x & 31;
    v = warp_sums<kNorm>(lane < static_cast<int>(cg::this_cluster().num_blocks())
                             ? *cg::this_cluster().map_shared_rank(join, lane)
                             : RowSums{0.f, 0.f});
  }
  return v;
}

// A norm's row, stored as a NaN one, by its definition, with h times a power of two that keeps its
// squares inside fp32: y = (h f) rsqrt(mean (h f)^2 + eps f^2) w.  The row is read again (`h`: x, or
// the hidden row, whose values each thread wrote itself) for the mean, the squares, the maximum and
// the codes: such rows are rare, and the others' registers and time are not spent on them.  (It comes
// after the first codes and scale: in their place it cost norm 1001 x 5632 6.7 us against 5.6, and
// 515 x 2048 in fp32, 2.7 us without it, takes 3.0 either way.)
// f = 2^84 for a mean below 2^-60 keeps 131056 squares under 2^125, 2^-84 from 2^60 on those of any
// finite h.
template <typename T, int KIND>
__device__ __forceinline__ void scaled_norm(const T* h, const T* weight, int8_t* codes, float* scale,
                                            int K, int base, int step, float eps, RowSums* part,
                                            RowSums* join, bool first) {
  auto sum_of = [&](float f) {
    RowSums v = {0.f, 0.f};
#pragma unroll 1
    for (int i0 = base; i0 < K; i0 += step)
#pragma unroll 1
      for (int i = max(i0, 0); i < min(i0 + kVec, K); ++i)
        v.ss = fmaf(to_f(h[i]) * f, to_f(h[i]) * f, v.ss);
    return norm_mean(row_sums_again<KIND>(v, part, join), K, eps * f * f);
  };
  const float mean = sum_of(1.f);
  const float f = mean < 0x1p-60f ? 0x1p84f : mean < 0x1p60f ? 1.f : 0x1p-84f;
  const float r = rsqrtf(sum_of(f));
  auto normed = [&](int i) { return to_f(h[i]) * f * r * to_f(weight[i]); };
  RowSums v = {0.f, 0.f};
#pragma unroll 1
  for (int i0 = base; i0 < K; i0 += step)
#pragma unroll 1
    for (int i = max(i0, 0); i < min(i0 + kVec, K); ++i) v.top = top3(v.top, normed(i), 0.f);
  const RowScale r8 = row_scale<kPlain>(row_sums_again<KIND>(v, part, join), K, 0.f);
  if (r8.bad) return;
  if (first) *scale = r8.scale;
#pragma unroll 1
  for (int i0 = base; i0 < K; i0 += step)
#pragma unroll 1
    for (int i = max(i0, 0); i < min(i0 + kVec, K); ++i) codes[i] = code_of(normed(i), r8);
}

template <typename T, int MODE, int NV, int KIND>
__global__ void __launch_bounds__(KIND == kWarp ? kWarpThreads : kMaxThreads,
                                  KIND == kWarp ? 4 : sizeof(T) == 4 && NV == 4 ? 1 : 2)
    rows_kernel(const RowArgs a) {
  __shared__ RowSums part[16];
  __shared__ RowSums join;
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

  constexpr bool kTwo = MODE == kGated || MODE == kNormRes;
  const int s_shift = kTwo ? shift_of(second - lead) : 0;
  const int w_shift = MODE >= kNorm ? shift_of(weight - lead) : 0;
  T* hidden = static_cast<T*>(a.hidden) + row * K;
  const bool hidden_aligned = MODE == kNormRes && shift_of(hidden - lead) == 0;

  pdl_enter();
  Held<T> h[NV], s[kTwo ? NV : 1], w[MODE >= kNorm ? NV : 1];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int i = base + n * step;
    if (i >= K) continue;
    h[n].template load<false>(x, i, K, x_shift);
    if constexpr (kTwo) s[n].template load<false>(second, i, K, s_shift);
    if constexpr (MODE >= kNorm) w[n].template load<true>(weight, i, K, w_shift);
  }
  float y[NV][kVec];
  RowSums sums = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int i = base + n * step;
    if (i >= K) continue;
    combine<T, MODE>(h[n], s[kTwo ? n : 0], w[MODE >= kNorm ? n : 0], y[n], sums.ss);
    if constexpr (MODE == kNormRes) h[n].store(hidden, i, K, hidden_aligned);
    sums.top = top_of(y[n], sums.top);
  }
  sums = KIND == kWarp ? warp_sums<MODE>(sums) : block_sums<MODE>(sums, part);
  if constexpr (KIND == kCluster) {
    if (threadIdx.x == 0) join = sums;
    cg::this_cluster().sync();
    const int lane = threadIdx.x & 31;
    sums = warp_sums<MODE>(lane < parts ? *cg::this_cluster().map_shared_rank(&join, lane)
                                        : RowSums{0.f, 0.f});
  }
  const bool writes_scale =
      rank == 0 && (KIND == kWarp ? threadIdx.x & 31 : threadIdx.x) == 0;
  const RowScale r8 = row_scale<MODE>(sums, K, a.eps);
  if (writes_scale) a.scale[row] = r8.scale;
#pragma unroll
  for (int n = 0; n < NV; ++n)
    if (base + n * step < K) store_codes(codes, base + n * step, K, y[n], r8);
  if constexpr (MODE >= kNorm)
    if (r8.bad)   // (the same for all that hold the row)
      scaled_norm<T, KIND>(MODE == kNormRes ? hidden : x, weight, codes, a.scale + row, K, base,
                           step, a.eps, part, &join, writes_scale);
  if constexpr (KIND == kCluster) cg::this_cluster().sync();  // all have read the others' sums
}

// ---- many rows: a ring of rows in shared memory ---------------------------------------------------

constexpr int kRingNV = 4;
constexpr int kRingStages = 2;       // at most
constexpr int kRingThreads = 1024;   // at most (64 registers a thread)

// L2 drops these lines first: the inputs are not read again, the codes written beside them are.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], "
      "%2, [%3], %4;" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}

// A CTA takes rows blockIdx.x, + gridDim.x, ...; bulk copies fill the stages ahead, a row is read
// from its stage into registers once and the stage refilled at once, so the next rows stream in
// under the reductions and stores of this one.  (With a CTA per row each CTA's loads, reductions
// and stores follow one another, and 40 to 70% of the bandwidth is what is left.)  A norm's weight
// stays in shared memory.  Rows here are whole 16-byte units at 16-byte addresses.
template <typename T, int MODE>
__global__ void __launch_bounds__(kRingThreads, 1)
    ring_kernel(const RowArgs a, int stages, unsigned int* status) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kRingStages + 1];
  __shared__ RowSums part[2][32];
  __shared__ volatile int aborted;
  constexpr bool kTwo = MODE == kGated || MODE == kNormRes;
  constexpr int NV = kRingNV;
  const int K = a.K;
  const uint32_t row_bytes = static_cast<uint32_t>(K) * sizeof(T);
  const uint32_t stage_bytes = kTwo ? 2 * row_bytes : row_bytes;
  uint8_t* ring = smem + (MODE >= kNorm ? row_bytes : 0);
  const uint32_t bar0 = smem_addr(bars), wbar = bar0 + 8 * kRingStages;
  const int64_t mine = (a.M - blockIdx.x + gridDim.x - 1) / gridDim.x;   // rows of this CTA
  if (threadIdx.x == 0) {
    aborted = 0;
    for (int s = 0; s <= kRingStages; ++s) mbar_init(bar0 + 8 * s, 1);
    fence_barrier_init();
  }
  __syncthreads();
  pdl_enter();
  const uint64_t once = policy_evict_first();
  auto issue = [&](int64_t j) {   // thread 0
    const int64_t row = blockIdx.x + j * gridDim.x;
    const int s = static_cast<int>(j % stages);
    const uint32_t dst = smem_addr(ring) + s * stage_bytes, bar = bar0 + 8 * s;
    mbar_arrive_expect_tx(bar, stage_bytes);
    bulk_load(dst, static_cast<const T*>(a.x) + row * a.x_ld, row_bytes, bar, once);
    if (kTwo)
      bulk_load(dst + row_bytes, static_cast<const T*>(a.second) + row * a.second_ld, row_bytes,
                bar, once);
  };
  if (threadIdx.x == 0) {
    if (MODE >= kNorm) {
      mbar_arrive_expect_tx(wbar, row_bytes);
      bulk_load(smem_addr(smem), a.weight, row_bytes, wbar, policy_evict_last());
    }
    for (int64_t j = 0; j < stages && j < mine; ++j) issue(j);
  }
  if (MODE >= kNorm && !mbar_wait(wbar, 0, status)) aborted = 1;
  const int base = threadIdx.x * kVec, step = blockDim.x * kVec;
  bool again = false;   // a norm's row is to be taken again (the same for the whole CTA)
  int s = 0;
  uint32_t phase = 0;
  for (int64_t j = 0; j < mine; ++j) {
    const int64_t row = blockIdx.x + j * gridDim.x;
    // (after a wait that ran out the rest of the loop only keeps the barriers in step)
    if (!aborted && !mbar_wait(bar0 + 8 * s, phase, status)) aborted = 1;
    const T* xs = reinterpret_cast<const T*>(ring + s * stage_bytes);
    float y[NV][kVec];
    RowSums sums = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = base + n * step;
      if (i >= K) continue;
      Held<T> h, g, w;
      h.load_shared(xs + i);
      if constexpr (kTwo) g.load_shared(xs + K + i);
      if constexpr (MODE >= kNorm) w.load_shared(reinterpret_cast<const T*>(smem) + i);
      combine<T, MODE>(h, g, w, y[n], sums.ss);
      if constexpr (MODE == kNormRes)
        if (!aborted) h.store(static_cast<T*>(a.hidden) + row * K, i, K, true);
      sums.top = top_of(y[n], sums.top);
    }
    // the stage's values are in registers: order these reads before the copy that refills it
    fence_proxy_async_smem();
    sums = block_sums<MODE>(sums, part[j & 1]);
    if (threadIdx.x == 0 && j + stages < mine && !aborted) issue(j + stages);
    const RowScale r8 = row_scale<MODE>(sums, K, a.eps);
    if (MODE >= kNorm) again |= r8.bad;
    if (!aborted) {
      if (threadIdx.x == 0) a.scale[row] = r8.scale;
#pragma unroll
      for (int n = 0; n < NV; ++n)
        if (base + n * step < K) store_codes(a.codes + row * K, base + n * step, K, y[n], r8);
    }
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
  if constexpr (MODE >= kNorm) {
    if (again) {
      __syncthreads();   // thread 0's scales, and a last word on `aborted`
      for (int64_t row = blockIdx.x; row < a.M && !aborted; row += gridDim.x)
        if (isnan(*static_cast<volatile float*>(a.scale + row)))
          scaled_norm<T, kBlock>(MODE == kNormRes ? static_cast<const T*>(a.hidden) + row * K
                                                  : static_cast<const T*>(a.x) + row * a.x_ld,
                                 static_cast<const T*>(a.weight), a.codes + row * K, a.scale + row,
                                 K, base, step, a.eps, part[0], nullptr, threadIdx.x == 0);
    }
  }
  if (aborted) {
    // leave the copies in flight time to land before the shared memory goes
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 2000000ull) __nanosleep(1000);
  }
}

// The quantizer's ring for rows of any length, alignment and stride, and for rows longer than a CTA
// holds: the parts CTAs of a cluster take a piece of every row each, of vp vectors, and exchange
// their sums once a row.  A piece is copied as the 16-byte granules that it touches, and its vectors
// are shifted out of them.  Those granules lie inside the tensor except at its two ends: in its
// first and last row (any row, where rows overlap) a granule that reaches past the first or last
// value is not copied, and the vectors that need it are read value by value.  (2877 x 11660:
// quantize 29.1 us with a CTA a row, 25.0 here, swiglu 59.6 and 41.6; 496 x 21731 fp32: 18.5 and
// 13.5, 56 and 30.  A norm, whose weight has to be shifted too, lost: 57.8 and 72.8.)
struct Piece {
  const uint8_t* from;   // first granule copied
  uint32_t bytes;        // of the granules copied
  uint32_t skip;         // where they go: bytes past the first granule touched (0 or 16)
  bool no_lo, no_hi;     // the first / last granule touched is not copied
};

template <typename T>
__device__ __forceinline__ Piece piece_of(const T* base, int64_t ld, int64_t M, int K, int64_t row,
                                          int e0, int e1) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(base);
  const uintptr_t hi = lo + ((M - 1) * ld + K) * sizeof(T);
  const uintptr_t a = lo + (row * ld + e0) * sizeof(T), e = lo + (row * ld + e1) * sizeof(T);
  uintptr_t g0 = a & ~uintptr_t(15), g1 = (e + 15) & ~uintptr_t(15);
  Piece p;
  p.no_lo = g0 < lo;
  p.no_hi = g1 > hi;
  p.skip = p.no_lo ? 16 : 0;
  if (p.no_lo) g0 += 16;
  if (p.no_hi) g1 -= 16;
  p.from = reinterpret_cast<const uint8_t*>(g0);
  p.bytes = g1 > g0 ? static_cast<uint32_t>(g1 - g0) : 0;
  return p;
}

constexpr int kRingPad = 64;   // shared memory before and after a piece that vectors may read

template <typename T, int MODE, bool SPLIT>
__global__ void __launch_bounds__(kRingThreads, 1)
    ring_any_kernel(const RowArgs a, int parts, int vp, int piece_bytes, int stages,
                    unsigned int* status) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kRingStages];
  __shared__ RowSums part[2][32];
  __shared__ RowSums join[2];
  __shared__ volatile int aborted;
  static_assert(MODE == kPlain || MODE == kGated);
  constexpr bool kTwo = MODE == kGated;
  constexpr int NV = kRingNV, es = sizeof(T);
  const int K = a.K;
  const int rank = SPLIT ? blockIdx.x % parts : 0;
  const int64_t first = SPLIT ? blockIdx.x / parts : blockIdx.x;
  const int64_t stride = SPLIT ? gridDim.x / parts : gridDim.x;
  const int64_t mine = (a.M - first + stride - 1) / stride;
  const uint32_t stage_bytes = kTwo ? 2 * piece_bytes : piece_bytes;
  const uint32_t ring = smem_addr(smem), bar0 = smem_addr(bars);
  const T* x = static_cast<const T*>(a.x);
  const T* second = static_cast<const T*>(a.second);
  const int piece0 = rank * vp * kVec, piece1 = piece0 + vp * kVec;   // this CTA's, before the lead
  // the last bits of an address p + (row * ld + i) * size: products need no more than theirs
  auto low = [](const void* p, int64_t row, int64_t ld, int i, int size, int mask) {
    return static_cast<int>((static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) +
                             (static_cast<uint32_t>(row) * static_cast<uint32_t>(ld) +
                              static_cast<uint32_t>(i)) * static_cast<uint32_t>(size)) & mask);
  };
  // rows that overlap can all lie at an end of the tensor
  const bool overlap = a.x_ld < K || (kTwo && a.second_ld < K);
  if (threadIdx.x == 0) {
    aborted = 0;
    for (int s = 0; s < kRingStages; ++s) mbar_init(bar0 + 8 * s, 1);
    fence_barrier_init();
  }
  __syncthreads();
  pdl_enter();
  const uint64_t once = policy_evict_first();
  auto issue = [&](int64_t j) {   // thread 0
    const int64_t row = first + j * stride;
    const int s = static_cast<int>(j % stages), lead = low(a.codes, row, K, 0, 1, 7);
    const int e0 = max(0, piece0 - lead), e1 = min(K, piece1 - lead);
    const uint32_t dst = ring + s * stage_bytes + kRingPad, bar = bar0 + 8 * s;
    const Piece p = piece_of(x, a.x_ld, a.M, K, row, e0, e1);
    Piece q = {};
    if (kTwo) q = piece_of(second, a.second_ld, a.M, K, row, e0, e1);
    mbar_arrive_expect_tx(bar, p.bytes + q.bytes);
    if (p.bytes) bulk_load(dst + p.skip, p.from, p.bytes, bar, once);
    if (q.bytes) bulk_load(dst + piece_bytes + q.skip, q.from, q.bytes, bar, once);
  };
  if (threadIdx.x == 0)
    for (int64_t j = 0; j < stages && j < mine; ++j) issue(j);
  const int tbase = piece0 + static_cast<int>(threadIdx.x) * kVec, step = blockDim.x * kVec;
  int s = 0;
  uint32_t phase = 0;
  for (int64_t j = 0; j < mine; ++j) {
    const int64_t row = first + j * stride;
    const int lead = low(a.codes, row, K, 0, 1, 7);
    const int e0 = max(0, piece0 - lead), e1 = min(K, piece1 - lead), end = piece1 - lead;
    const int base = tbase - lead;
    // shared addresses of value 0 of the row, and what every vector is past a boundary
    const uint32_t at = ring + s * stage_bytes + kRingPad - e0 * es;
    const uint32_t xz = at + low(x, row, a.x_ld, e0, es, 15);
    const uint32_t sz = at + piece_bytes + (kTwo ? low(second, row, a.second_ld, e0, es, 15) : 0);
    const int x_shift = (xz + base * es) & 15, s_shift = (sz + base * es) & 15;
    Piece p = {}, q = {};
    if (row == 0 || row == a.M - 1 || overlap) {
      p = piece_of(x, a.x_ld, a.M, K, row, e0, e1);
      if (kTwo) q = piece_of(second, a.second_ld, a.M, K, row, e0, e1);
    }
    // (after a wait that ran out the rest of the loop only keeps the barriers in step)
    if (!aborted && !mbar_wait(bar0 + 8 * s, phase, status)) aborted = 1;
    float y[NV][kVec];
    RowSums sums = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = base + n * step;
      if (i >= K || i >= end) continue;
      Held<T> h, g;
      h.load_shared_at(xz + i * es, x_shift);
      if constexpr (kTwo) g.load_shared_at(sz + i * es, s_shift);
      if (i < e0 + kVec || i + 2 * kVec > e1) {   // the piece's ends
        if ((p.no_lo && i < e0 + kVec) || (p.no_hi && i + 2 * kVec > e1)) {
          h.load_values(x + row * a.x_ld, i, K);
        } else {
          h.clip(i, K);
        }
        if constexpr (kTwo) {
          if ((q.no_lo && i < e0 + kVec) || (q.no_hi && i + 2 * kVec > e1)) {
            g.load_values(second + row * a.second_ld, i, K);
          } else {
            g.clip(i, K);
          }
        }
      }
      combine<T, MODE>(h, g, g, y[n], sums.ss);
      sums.top = top_of(y[n], sums.top);
    }
    // the stage's values are in registers: order these reads before the copy that refills it
    fence_proxy_async_smem();
    sums = block_sums<MODE>(sums, part[j & 1]);
    if (threadIdx.x == 0 && j + stages < mine && !aborted) issue(j + stages);
    if constexpr (SPLIT) {
      // (two slots in turn, as for the warps' sums)
      if (threadIdx.x == 0) join[j & 1] = sums;
      cg::this_cluster().sync();
      const int lane = threadIdx.x & 31;
      sums = warp_sums<MODE>(lane < parts ? *cg::this_cluster().map_shared_rank(&join[j & 1], lane)
                                          : RowSums{0.f, 0.f});
    }
    const RowScale r8 = row_scale<MODE>(sums, K, a.eps);
    if (!aborted) {
      if (threadIdx.x == 0 && rank == 0) a.scale[row] = r8.scale;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int i = base + n * step;
        if (i < K && i < end) store_codes(a.codes + row * K, i, K, y[n], r8);
      }
    }
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
  if (aborted) {
    // leave the copies in flight time to land before the shared memory goes
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 2000000ull) __nanosleep(1000);
  }
  if constexpr (SPLIT) cg::this_cluster().sync();   // the others have read this CTA's last sums
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

struct RingShape {
  int parts, vp, threads, piece, stages, grid, smem;
};

// How a ring takes rows of nvec vectors; false where it does not: short rows (a warp each), or
// fewer than two rows for every CTA (then a CTA per row is faster: 1001 x 5632, norm 5.6 us against
// 7.3).  pad: bytes around a piece in shared memory (0: whole rows, as they are).
template <typename T, int MODE>
bool ring_shape(const RowArgs& a, int nvec, int pad, RingShape& r) {
  if (nvec <= 128) return false;
  for (r.parts = 1; r.parts <= (pad ? 8 : 1); r.parts *= 2) {
    r.vp = (nvec + r.parts - 1) / r.parts;
    r.threads = ((r.vp + kRingNV - 1) / kRingNV + 31) / 32 * 32;
    if (r.threads > kRingThreads) continue;
    const int values = pad ? r.vp * kVec + kVec : a.K;
    r.piece = (values * static_cast<int>(sizeof(T)) + 15) / 16 * 16 + 2 * pad;
    const int stage = MODE == kGated || MODE == kNormRes ? 2 * r.piece : r.piece;
    const int fixed = MODE >= kNorm ? r.piece : 0;
    int per_sm = kRingThreads / r.threads;   // 64 registers a thread
    if (per_sm > 16) per_sm = 16;
    auto fits = [&](int n) { return 227 * 1024 / (fixed + n * stage + 2048); };
    // two stages as long as two CTAs an SM hold them (or the one that its threads allow): below
    // that a second CTA hides more than a second stage (swiglu 2048 x 14336: 31.5 us with two CTAs
    // of one stage, 34.0 with one of two; norm with residual 8192 x 8192: 77 us with two CTAs of two
    // stages, 79 with four of one)
    r.stages = fits(2) >= (per_sm < 2 ? per_sm : 2) ? 2 : 1;
    const int f = fits(r.stages);
    if (f < 1) continue;
    if (per_sm > f) per_sm = f;
    r.smem = fixed + r.stages * stage;
    r.grid = sm_count() * per_sm / r.parts * r.parts;
    return a.M >= 2 * static_cast<int64_t>(r.grid) / r.parts;
  }
  return false;
}

// Whole 16-byte rows at 16-byte addresses.
template <typename T>
bool whole_rows(const RowArgs& a) {
  auto whole = [](const void* p, int64_t ld) {
    return aligned(p, 16) && ld * static_cast<int>(sizeof(T)) % 16 == 0;
  };
  return a.K % kVec == 0 && whole(a.x, a.x_ld) && whole(a.second, a.second_ld) &&
         aligned(a.weight, 16) && aligned(a.hidden, 16) && aligned(a.codes, kVec);
}

template <typename... KArgs, typename... Args>
int launch_ring(void (*kern)(KArgs...), std::atomic<uint64_t>& done, const RingShape& r,
                cudaStream_t stream, Args... args) {
  unsigned int* status = device_status_ptr();
  if (!status) return fail(RW4_ECUDA, "int8 rows: device status word unavailable");
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !((done.load() >> dev) & 1)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024) !=
        cudaSuccess)
      return fail(RW4_ECUDA, "int8 rows: cannot set the kernel's shared memory size");
    if (dev < 64) done.fetch_or(1ull << dev);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(r.grid);
  cfg.blockDim = dim3(r.threads);
  cfg.dynamicSmemBytes = r.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = r.parts;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = r.parts > 1 ? 2 : 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, args..., status);
  if (err != cudaSuccess) return cuda_status(err, "rw4 int8 rows launch");
  return launch_status("rw4 int8 rows launch");
}

template <typename T, int MODE>
int run_rows(const RowArgs& a, cudaStream_t stream) {
  // a row's vectors, with one more where it can start inside one
  const bool whole = a.K % kVec == 0 && aligned(a.codes, kVec);
  const int nvec = whole ? a.K / kVec : (a.K + 2 * (kVec - 1)) / kVec;
  RingShape r;
  static std::atomic<uint64_t> done[3];
  if (whole_rows<T>(a) && ring_shape<T, MODE>(a, nvec, 0, r))
    return launch_ring(ring_kernel<T, MODE>, done[0], r, stream, a, r.stages);
  if constexpr (MODE == kPlain || MODE == kGated) {
    // (long rows of two aligned inputs: 512 x 53248 44.4 us with a cluster a row, 48.3 in this ring)
    if (nvec > 1024 && (MODE == kPlain || !whole_rows<T>(a)) &&
        ring_shape<T, MODE>(a, nvec, kRingPad, r)) {
      if (r.parts == 1)
        return launch_ring(ring_any_kernel<T, MODE, false>, done[1], r, stream, a, 1, r.vp, r.piece,
                           r.stages);
      return launch_ring(ring_any_kernel<T, MODE, true>, done[2], r, stream, a, r.parts, r.vp,
                         r.piece, r.stages);
    }
  }
  if (nvec <= 128) {   // one warp a row, four rows a CTA
    const int64_t blocks = (a.M + kWarpThreads / 32 - 1) / (kWarpThreads / 32);
    if (nvec <= 32) return launch_rows<T, MODE, 1, kWarp>(a, blocks, 1, kWarpThreads, stream);
    if (nvec <= 64) return launch_rows<T, MODE, 2, kWarp>(a, blocks, 1, kWarpThreads, stream);
    return launch_rows<T, MODE, 4, kWarp>(a, blocks, 1, kWarpThreads, stream);
  }
  auto threads_for = [](int vecs, int nv) { return (((vecs + nv - 1) / nv) + 31) / 32 * 32; };
  // Few long rows: a cluster a row, one vector a thread, where that is faster than one CTA with
  // more (one row: swiglu of 28672 values 2.7 us against 4.6, of 14336 2.6 against 3.3; quantize of
  // 14336 2.4 against 1.9).
  int parts = 1;
  while (parts < 8 && nvec > parts * kMaxThreads) parts *= 2;
  if (nvec * (MODE == kPlain ? 1 : 2) > 4 * kMaxThreads && nvec <= parts * kMaxThreads &&
      a.M * parts <= sm_count())
    return launch_rows<T, MODE, 1, kCluster>(a, a.M * parts, parts,
                                             threads_for((nvec + parts - 1) / parts, 1), stream);
  // With a CTA or less on every SM threads hide latency, beyond it registers do (norm with residual
  // of 4096 values: 150 rows 2.3 us with one vector a thread, 2.4 with two; 600 rows 6.2 and 5.5).
  if (nvec <= kMaxThreads && (a.M <= sm_count() || nvec <= 3 * kMaxThreads / 8 ||
                              (nvec <= kMaxThreads / 2 && a.M <= 8 * sm_count())))
    return launch_rows<T, MODE, 1, kBlock>(a, a.M, 1, threads_for(nvec, 1), stream);
  if (nvec <= 2 * kMaxThreads)
    return launch_rows<T, MODE, 2, kBlock>(a, a.M, 1, threads_for(nvec, 2), stream);
  if (nvec <= 4 * kMaxThreads)
    return launch_rows<T, MODE, 4, kBlock>(a, a.M, 1, threads_for(nvec, 4), stream);
  parts = 2;
  while (parts < 8 && nvec > parts * 4 * kMaxThreads) parts *= 2;
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

// Whether the M x K codes or their scales at these addresses meet each other or rows of input (or the
// new hidden rows): what another thread has yet to read could be written.
bool outputs_meet(const RowArgs& a, int es) {
  const int64_t codes = a.M * a.K, scale = 4 * a.M;
  auto meet = [&](const void* p, int64_t ld) {
    return rw4::meets(a.codes, codes, p, a.K * es, a.M, ld * es) ||
           rw4::meets(a.scale, scale, p, a.K * es, a.M, ld * es);
  };
  return rw4::meets(a.codes, codes, a.scale, scale) || meet(a.x, a.x_ld) ||
         meet(a.second, a.second_ld) || meet(a.hidden, a.K) ||
         rw4::meets(a.codes, codes, a.weight, a.K * es) ||
         rw4::meets(a.scale, scale, a.weight, a.K * es);
}

// Whether the hidden rows meet rows of input without being those very rows.
bool hidden_meets(const RowArgs& a, int es) {
  auto meet = [&](const void* p, int64_t ld) {
    return !(p == a.hidden && ld == a.K) &&
           rw4::meets(a.hidden, a.M * a.K * es, p, a.K * es, a.M, ld * es);
  };
  return meet(a.x, a.x_ld) || meet(a.second, a.second_ld) ||
         rw4::meets(a.hidden, a.M * a.K * es, a.weight, a.K * es);
}

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
  if (outputs_meet(a, es))
    return fail(RW4_EINVAL, "int8_quantize: codes or scale overlap an input or each other");
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
  if (outputs_meet(a, es))
    return fail(RW4_EINVAL, "int8_rmsnorm: codes or scale overlap another operand or each other");
  if (hidden_meets(a, es))
    return fail(RW4_EINVAL, "int8_rmsnorm: hidden overlaps an input without being x or residual "
                "itself");
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
  const int64_t bytes = M * K * elem_size(out_dtype);
  if (rw4::meets(out, bytes, codes, M * K) || rw4::meets(out, bytes, scale, 4 * M))
    return fail(RW4_EINVAL, "int8_dequantize: out overlaps an input");
  cudaStream_t s = rw4::as_stream(stream);
  if (out_dtype == RW4_F32)
    return launch_dequant(codes, scale, M, K, static_cast<float*>(out), s);
  if (out_dtype == RW4_F16)
    return launch_dequant(codes, scale, M, K, static_cast<__half*>(out), s);
  return launch_dequant(codes, scale, M, K, static_cast<__nv_bfloat16*>(out), s);
}
