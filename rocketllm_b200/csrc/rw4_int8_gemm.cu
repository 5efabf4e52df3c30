// 8-bit matrix product of the W8A8 path on the 5th-generation tensor cores (sm_100a):
//
//   out[m, n] = round(scale[m] * weight_scale[n] * sum_k codes[m, k] * weight[n, k]
//                     + bias[n] + residual[m, n])
//
// codes and weight are signed 8-bit rows (K innermost).  The sum is exact: tcgen05.mma kind::i8
// accumulates in 32-bit integers in TMEM, and K <= 131056 keeps any sum of products of 8-bit codes
// (at most 2^14 each) inside them.  So the result does not depend on tiles or splits; scales, bias
// and residual are applied to it in fp32 and rounded once to the output's type.
//
// Both kernels put the weight rows on the M side of the MMA (the accumulator's 128 TMEM lanes) and
// tokens on its N side (its columns): one token is then one column, and a call of any number of
// tokens from one on reads no more weight bytes than there are.  Operand tiles are 128 bytes of K
// wide (one 128-byte swizzle atom: four MMAs of K = 32), loaded by TMA through an mbarrier ring; the
// ends of K, of the weight rows and of the tokens are zero-filled by TMA and never stored.
//
//   split kernel   one CTA for 128 weight rows x BN tokens (BN = 16 .. 128), K split over the CTAs
//                  of a cluster when there are fewer tiles than SMs; the integer partial sums meet
//                  in distributed shared memory (no workspace, no atomics).
//   pair kernel    two CTAs (cta_group::2) share one 256 x 256 tile: each holds 128 weight rows and
//                  half of the tokens' operand, so a byte of shared memory feeds twice the MMAs.
//                  Persistent over tiles; the accumulator is double-buffered in TMEM so that the
//                  epilogue of one tile runs under the MMAs of the next.
//
// Every TMA load is a plain per-CTA load.  Every mbarrier wait is bounded (rw4_tma.cuh).
#include <atomic>

#include "rw4_tcgen05.cuh"

namespace {

using namespace rw4;

constexpr int BK = 128;                  // bytes (= codes) of K per stage
constexpr int BMW = 128;                 // weight rows per CTA
constexpr int kWBytes = BMW * BK;        // 16 KB
constexpr int64_t kMaxK = 131056;

// Instruction descriptor, kind::i8: D s32 (2 << 4), A and B signed 8-bit (1 << 7, 1 << 10), both
// K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

struct Epilogue {
  const float* scale;         // [M]
  const float* weight_scale;  // [N]
  const void* bias;           // [N] or null
  const void* residual;       // [M, N] or null
  void* out;                  // [M, N]
};

template <typename T>
__device__ __forceinline__ float ep_f(T v);
template <>
__device__ __forceinline__ float ep_f(float v) { return v; }
template <>
__device__ __forceinline__ float ep_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float ep_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T ep_t(float v);
template <>
__device__ __forceinline__ float ep_t(float v) { return v; }
template <>
__device__ __forceinline__ __half ep_t(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 ep_t(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 16 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void pdl_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// The address, in the cluster's shared window, of `addr` in the CTA of rank `rank`.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

// Copy within the cluster, from this CTA's shared memory to another's, whose barrier counts it.
__device__ __forceinline__ void bulk_send(uint32_t dst, uint32_t src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, "
      "[%3];" ::"r"(dst),
      "r"(src), "r"(bytes), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void st_shared(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__device__ __forceinline__ void ld_shared8(uint32_t addr, int (&v)[8]) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(addr + 16)
               : "memory");
}

__device__ __forceinline__ int ld_shared(uint32_t addr) {
  int v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Eight adjacent values in whole 16-byte units.
template <typename T>
struct Eight {
  static constexpr int kQuads = sizeof(T) / 2;
  uint4 u[kQuads];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j) u[j] = reinterpret_cast<const uint4*>(p)[j];
  }
};

// A token's scale on its way to sum * scale * weight_scale + bias: to the sum, or, where it is so large
// that their product could overflow, to the weight's scale, with which it cannot underflow there.
// (The scales' product alone leaves the normal numbers while the result does not.  Chosen for every
// output instead it cost 3 to 9% of a call.)
struct TokenScale {
  float sum, weight;
  __device__ __forceinline__ explicit TokenScale(float s) {
    const bool large = !(fabsf(s) < 0x1p64f);
    sum = large ? 1.f : s;
    weight = large ? s : 1.f;
  }
  __device__ __forceinline__ float apply(int acc, float ws, float bias) const {
    return fmaf(static_cast<float>(acc) * sum, weight * ws, bias);
  }
};

// Eight adjacent outputs from their exact sums and (res) residuals.
template <typename T>
__device__ __forceinline__ void store8(const int (&sum)[8], float sx, const float (&ws)[8],
                                       const float (&bias)[8], bool res, const Eight<T>& r, T* out) {
  const T* rv = reinterpret_cast<const T*>(r.u);
  const TokenScale s(sx);
  __align__(16) T y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float f = s.apply(sum[j], ws[j], bias[j]);
    if (res) f += ep_f(rv[j]);
    y[j] = ep_t<T>(f);
  }
#pragma unroll
  for (int j = 0; j < Eight<T>::kQuads; ++j)
    reinterpret_cast<uint4*>(out)[j] = reinterpret_cast<const uint4*>(y)[j];
}

// Whether every output row is whole 16-byte units.  Where it is, a thread stores eight adjacent
// outputs at a time; else adjacent threads store adjacent outputs (eight single stores of a thread,
// 16 bytes apart from its neighbour's, took 254 us for 4086 x 5072 x 8212 against 151).
inline bool wide_rows(const Epilogue& e, int64_t N) {
  return N % 8 == 0 && ((reinterpret_cast<uintptr_t>(e.out) |
                         reinterpret_cast<uintptr_t>(e.residual)) & 15) == 0;
}

// ---------------------------------------------------------------------------------------------
// split kernel
// ---------------------------------------------------------------------------------------------

template <int BN>
struct SplitCfg {
  static constexpr int kXBytes = BN * BK;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  // up to 64 tokens two CTAs share an SM (one's prologue and epilogue under the other's loads)
  static constexpr int kCtasPerSm = BN <= 64 ? 2 : 1;
  static constexpr int kStages = BN == 16 ? 5 : BN == 32 ? 4 : BN == 64 ? 3 : 5;
  // K splits: the partial sums to send lie over the stages, those received beside them
  static constexpr int kPartBytes = BN * BMW * 4;
  static constexpr int kOffPart = kStages * kStageBytes;
  static constexpr int kOffBars = kOffPart + kPartBytes;
  static constexpr int kOffTmem = kOffBars + (2 * kStages + 2) * 8;
  static constexpr int kSmem = kOffTmem + 8 + 1024;
  static constexpr uint32_t kTmemCols = BN < 32 ? 32 : BN;
  static constexpr int kEpiWarps = BN <= 64 ? 4 : 8;   // four, or four for each half of the columns
  static constexpr int kThreads = 64 + 32 * kEpiWarps; // TMA, MMA, epilogue
  static constexpr int kCols = BN / (kEpiWarps / 4);   // columns of an epilogue warp
  static_assert(kPartBytes <= kStages * kStageBytes, "the sums fit over the stages");
  static_assert((kSmem + 1024) * kCtasPerSm <= 228 * 1024, "shared memory budget");
};

// k-blocks of the weight that a CTA prefetches into L2 before its turn (norm, products and quantizer
// of a layer of width 8192 in one graph, one token: 151.8 us a layer without, 149.2 with 3, 151.8 with
// 10, 157.6 with 20)
constexpr int kPrefetch = 3;

template <int BN, typename T, bool WIDE, bool RES>
__global__ void __launch_bounds__(SplitCfg<BN>::kThreads)
    int8_split_kernel(const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_x, const Epilogue e, int M, int N,
                      int nkb, int m_tiles, int log_splits, unsigned int* status) {
  using C = SplitCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  __shared__ int aborted;
  __shared__ float sx[BN];                      // the tokens' scales
  const int splits = 1 << log_splits;
  const int rank = blockIdx.x & (splits - 1);   // in the cluster: its CTAs are adjacent
  const int tile = blockIdx.x >> log_splits;
  const int m0 = (tile % m_tiles) * BN;   // tokens fastest: a weight tile is read once
  const int n0 = (tile / m_tiles) * BMW;
  const int kb0 = (int)((int64_t)nkb * rank >> log_splits);
  const int kb1 = (int)((int64_t)nkb * (rank + 1) >> log_splits);

  const uint32_t sb = smem_addr(smem);
  const uint32_t full0 = sb + C::kOffBars;
  const uint32_t empty0 = full0 + 8 * C::kStages;
  const uint32_t accum = empty0 + 8 * C::kStages;
  const uint32_t parts = accum + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffTmem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cols = min(BN, M - m0);
  // columns of the tile that CTA r of the cluster sums and stores: r, r + splits, ...
  auto share = [&](int r) { return (cols - r + splits - 1) >> log_splits; };
  constexpr uint32_t kColBytes = BMW * 4;

  if (threadIdx.x == 0) {
    aborted = 0;
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(accum, 1);
    mbar_init(parts, 1);
    fence_barrier_init();
    if (splits > 1 && share(rank) > 0)
      mbar_arrive_expect_tx(parts, splits * share(rank) * kColBytes);
  }
  if (warp == 1) tmem_alloc(smem_addr(tmem_slot), C::kTmemCols);
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
    // the weight's first tiles into L2 while the kernel before this one runs (nothing is read that
    // it could still write: L2 holds what is written)
    for (int kb = kb0; kb < min(kb1, kb0 + kPrefetch); ++kb) tma_prefetch_2d(&tm_w, kb * BK, n0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (splits > 1) cluster_arrive();   // this CTA's shared memory and barriers are there
  pdl_wait();
  pdl_launch();

  const int q = warp & 3;                 // TMEM lane quarter
  const bool epi = warp >= 2;
  // outputs: this thread takes 8 adjacent weight rows of a token (wide), or rows 32 apart
  const int et = threadIdx.x - 64;
  const int n_first = n0 + (WIDE ? 8 * (et & 15) : lane), n_step = WIDE ? 1 : 32;
  float ws[8], bias[8];
  if (warp == 0) {
    if (lane == 0) {
      int issued = kb0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, s = i % C::kStages;
        if (!mbar_wait(empty0 + 8 * s, ((i / C::kStages) & 1) ^ 1, status)) {
          aborted = 1;
          break;
        }
        const uint32_t dst = sb + s * C::kStageBytes;
        mbar_arrive_expect_tx(full0 + 8 * s, C::kStageBytes);
        tma_load_2d(dst, &tm_w, kb * BK, n0, full0 + 8 * s);
        tma_load_2d(dst + kWBytes, &tm_x, kb * BK, m0, full0 + 8 * s);
        issued = kb + 1;
      }
      for (int kb = max(kb0, issued - C::kStages); kb < issued; ++kb) {  // own copies have landed
        const int i = kb - kb0;
        mbar_wait(full0 + 8 * (i % C::kStages), (i / C::kStages) & 1, status);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, s = i % C::kStages;
        if (!mbar_wait(full0 + 8 * s, (i / C::kStages) & 1, status)) {
          aborted = 1;
          break;
        }
        tc_fence_after();
        const uint32_t src = sb + s * C::kStageBytes;
        const uint64_t da = smem_desc(src), db = smem_desc(src + kWBytes);
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk)  // +32 bytes along K inside the swizzle atom
          umma_i8(tmem, da + (uint64_t)(2 * kk), db + (uint64_t)(2 * kk), idesc_i8(BMW, BN),
                  (i > 0 || kk > 0) ? 1u : 0u);
        umma_commit(empty0 + 8 * s);
      }
      umma_commit(accum);
    }
  } else {
    // under the loads
    for (int c = threadIdx.x - 64; c < BN; c += 32 * C::kEpiWarps)
      sx[c] = m0 + c < M ? __ldg(e.scale + m0 + c) : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = n_first + j * n_step;
      ws[j] = n < N ? __ldg(e.weight_scale + n) : 0.f;
      bias[j] = e.bias && n < N ? ep_f(static_cast<const T*>(e.bias)[n]) : 0.f;
    }
  }
  __syncwarp();
  // every warp waits for the accumulator: after it no MMA reads the stages
  const bool done = mbar_wait(accum, 0, status);
  if (!done) aborted = 1;
  tc_fence_after();
  __syncthreads();
  const bool ok = !aborted;

  // The sums, over the (now idle) stages, token by token: sums[slot][weight row].  Token c of the
  // tile is finished by CTA c % splits of the cluster; the sums are laid out by receiver, slot
  // (c % splits) * run + c / splits, so that each receiver's part is one run.  (Short loops on
  // purpose: every launch runs this code once, and straight-line code for 32 columns spent 3 us, a
  // K-split one 9, waiting for instructions.)
  const int run = BN >> log_splits;
  if (epi) {
    const uint32_t acc = tmem + ((uint32_t)(32 * q) << 16);
    const uint32_t at = sb + (uint32_t)(32 * q + lane) * 4;
    const int c_first = ((warp - 2) >> 2) * C::kCols;
#pragma unroll 1
    for (int c0 = c_first; c0 < c_first + C::kCols && c0 < cols; c0 += 16) {
      uint32_t v[16];
      tmem_ld16(acc + (uint32_t)c0, v);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int c = c0 + j;
        st_shared(at + ((c & (splits - 1)) * run + (c >> log_splits)) * kColBytes, v[j]);
      }
    }
    if (splits > 1) fence_proxy_async_smem();  // before the copies that read them
    asm volatile("bar.sync 1, %0;" ::"r"(32 * C::kEpiWarps) : "memory");
  }
  if (splits > 1) {
    cluster_wait();               // the other CTAs' barriers are there
    // each receiver's run (this CTA's own too) in one bulk copy, counted on the receiver's barrier
    if (epi && et < splits && ok && share(et) > 0)
      bulk_send(map_rank(sb + C::kOffPart + rank * run * kColBytes, et), sb + et * run * kColBytes,
                share(et) * kColBytes, map_rank(parts, et));
  }
  // (A CTA whose own sums are not there waits for the others' all the same, as long as a wait lasts:
  // they may be on their way, and must not find its shared memory, or their senders', gone.)
  if (epi && share(rank) > 0 && (splits == 1 || mbar_wait(parts, 0, status)) && ok) {
    const uint32_t got = sb + (splits > 1 ? C::kOffPart : 0);
    const T* res = static_cast<const T*>(e.residual);
    T* out = static_cast<T*>(e.out);
    // (a token's residuals are loaded while the one before it is finished)
    auto at = [&](int t) { return (int64_t)(m0 + (t << log_splits) + rank) * N + n_first; };
    if constexpr (WIDE) {
      constexpr int kTokens = 2 * C::kEpiWarps;
      const bool mine = n_first < N;
      int t = et >> 4;
      Eight<T> r = {}, next = {};
      if (RES && mine && t < share(rank)) next.load(res + at(t));
#pragma unroll 1
      for (; t < share(rank); t += kTokens) {
        r = next;
        if (RES && mine && t + kTokens < share(rank)) next.load(res + at(t + kTokens));
        const uint32_t from = got + t * kColBytes + 32 * (et & 15);
        int sum[8];
        ld_shared8(from, sum);
#pragma unroll 1
        for (int k = 1; k < splits; ++k) {
          int part[8];
          ld_shared8(from + k * run * kColBytes, part);
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] += part[j];
        }
        if (mine)
          store8<T>(sum, sx[(t << log_splits) + rank], ws, bias, RES, r, out + at(t));
      }
    } else {
      int t = warp - 2;
      float r[4], next[4] = {};
      auto load = [&](int t) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n_first + 32 * j < N) next[j] = ep_f(res[at(t) + 32 * j]);
      };
      if (RES && t < share(rank)) load(t);
#pragma unroll 1
      for (; t < share(rank); t += C::kEpiWarps) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = next[j];
        if (RES && t + C::kEpiWarps < share(rank)) load(t + C::kEpiWarps);
        int sum[4] = {};
#pragma unroll 1
        for (int k = 0; k < splits; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sum[j] += ld_shared(got + (k * run + t) * kColBytes + (lane + 32 * j) * 4);
        const TokenScale s(sx[(t << log_splits) + rank]);
        T* o = out + at(t);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n_first + 32 * j < N)
            o[32 * j] = ep_t<T>(s.apply(sum[j], ws[j], bias[j]) + r[j]);
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_arrive();   // what was sent to this CTA is here
    cluster_wait();     // what this CTA sent has left its shared memory
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------
// pair kernel
// ---------------------------------------------------------------------------------------------

constexpr int kPairRows = 256;                  // weight rows of a tile, 128 of each CTA
constexpr int kPairTokens = 256;                // tokens of a tile: each CTA loads half
constexpr int kPairStageBytes = kWBytes + kPairTokens / 2 * BK;
constexpr int kPairStages = 6;
constexpr int kPairEpiWarps = 8;                // four for each half of the columns
constexpr int kPairOffOut = kPairStages * kPairStageBytes;       // 16 tokens x 32 sums of a warp
constexpr int kPairOffBars = kPairOffOut + kPairEpiWarps * 16 * 32 * 4;
// full[], empty[], acc_full[2], acc_empty[2]
constexpr int kPairOffTmem = kPairOffBars + (2 * kPairStages + 4) * 8;
constexpr int kPairSmem = kPairOffTmem + 8 + 1024;
constexpr int kPairThreads = 32 * (2 + kPairEpiWarps);
constexpr uint32_t kPairTmemCols = 2 * kPairTokens;              // two accumulators
constexpr int kPairGroup = 8;                   // weight tiles that run side by side
static_assert(kPairSmem <= 227 * 1024, "shared memory budget");
// A CTA whose TMEM allocation waits must not wait for a cluster that waits in turn for this one's.
// This kernel takes all columns, but its shared memory leaves an SM no room for a CTA of another
// cluster kernel that allocates any; the CTAs of the split kernel that fit on an SM leave each other
// their columns.
static_assert(kPairSmem + SplitCfg<16>::kSmem > 228 * 1024 &&
              kPairSmem + SplitCfg<32>::kSmem > 228 * 1024 &&
              kPairSmem + SplitCfg<64>::kSmem > 228 * 1024 &&
              kPairSmem + SplitCfg<128>::kSmem > 228 * 1024, "no pair CTA beside a split CTA");
static_assert(2 * (SplitCfg<64>::kTmemCols + SplitCfg<128>::kTmemCols) <= 512, "TMEM columns");

// Plain load into this CTA's shared memory whose bytes complete on a barrier of the pair's leader.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                                 uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(leader_bar)
      : "memory");
}

__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive on the barrier at this offset in both CTAs once the MMAs issued so far have completed.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}

// The tiles of a call: a grid of n_tiles x m_tiles, and how its last wave is cut.
struct PairGrid {
  int n_tiles, m_tiles;
  int full;       // tiles that are taken whole, whole waves of them
  int cut;        // each tile after them is taken as 1 << cut strips of 256 >> cut tokens
  int items;      // tiles and strips
};

struct PairItem {
  int n0, m0, width;   // first weight row, first token, tokens
};

// Item t.  Tiles come in groups of kPairGroup weight tiles, tokens in the middle, so that the tiles in
// flight form a near-square block whose operands L2 holds.
__device__ __forceinline__ PairItem pair_item(int t, const PairGrid& g) {
  int strip = 0, width = kPairTokens;
  if (t >= g.full) {
    const int u = t - g.full;
    strip = u & ((1 << g.cut) - 1);
    t = g.full + (u >> g.cut);
    width = kPairTokens >> g.cut;
  }
  const int per = kPairGroup * g.m_tiles;
  const int group = t / per, r = t - group * per;
  const int side = min(kPairGroup, g.n_tiles - group * kPairGroup);
  const int tm = r / side, tn = group * kPairGroup + r - tm * side;
  return {tn * kPairRows, tm * kPairTokens + strip * width, width};
}

template <typename T, bool WIDE, bool RES>
__global__ void __launch_bounds__(kPairThreads, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap tm_strip, const Epilogue e, int M, int N,
                     int nkb, const PairGrid g, unsigned int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  __shared__ int aborted;
  const uint32_t sb = smem_addr(smem);
  const uint32_t full0 = sb + kPairOffBars;             // leader's: both CTAs' bytes have landed
  const uint32_t empty0 = full0 + 8 * kPairStages;      // each CTA's: the stage's MMAs are done
  const uint32_t afull0 = empty0 + 8 * kPairStages;     // each CTA's: an accumulator is complete
  const uint32_t aempty0 = afull0 + 16;                 // leader's: both CTAs have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kPairOffTmem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    aborted = 0;
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(afull0 + 8 * b, 1);
      mbar_init(aempty0 + 8 * b, 2 * kPairEpiWarps);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(tmem_slot)),
                 "r"(kPairTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
    prefetch_tensormap(&tm_strip);
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();  // the peer's barriers are initialised too
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch();

  if (warp == 0) {
    if (lane == 0) {
      // both CTAs load their own halves; the bytes of both are counted on the leader's barrier,
      // which the leader arms.  (The peer may load first: the phase cannot complete before the
      // leader's arrival, and neither starts a stage before the commit of the MMAs that read it.)
      int i = 0;
      bool ok = true;
      for (int t = first; t < g.items && ok; t += stride) {
        const PairItem it = pair_item(t, g);
        if (it.m0 >= M) continue;   // a strip past the last token (in every role)
        const int n0 = it.n0 + rank * 128, m0 = it.m0 + rank * (it.width / 2);
        const CUtensorMap* mx = t < g.full ? &tm_x : &tm_strip;
        const uint32_t bytes = 2 * kWBytes + it.width * BK;   // of both CTAs
        for (int kb = 0; kb < nkb; ++kb, ++i) {
          const int s = i % kPairStages;
          if (!mbar_wait(empty0 + 8 * s, ((i / kPairStages) & 1) ^ 1, status)) {
            aborted = 1;
            ok = false;
            break;
          }
          const uint32_t bar = map_rank(full0 + 8 * s, 0);
          const uint32_t dst = sb + s * kPairStageBytes;
          if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, bytes);
          tma_load_2d_pair(dst, &tm_w, kb * BK, n0, bar);
          tma_load_2d_pair(dst + kWBytes, mx, kb * BK, m0, bar);
        }
      }
      if (!ok) {
        // the stages in flight land within microseconds; leave them time before the CTA goes
        const unsigned long long t0 = globaltimer();
        while (globaltimer() - t0 < 2000000ull) __nanosleep(1000);
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      int i = 0, j = 0;
      bool ok = true;
      for (int t = first; t < g.items && ok; t += stride) {
        const PairItem it = pair_item(t, g);
        if (it.m0 >= M) continue;
        const uint32_t idesc = idesc_i8(kPairRows, it.width);
        const int b = j & 1;
        if (!mbar_wait(aempty0 + 8 * b, ((j >> 1) & 1) ^ 1, status)) {
          aborted = 1;
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < nkb; ++kb, ++i) {
          const int s = i % kPairStages;
          if (!mbar_wait(full0 + 8 * s, (i / kPairStages) & 1, status)) {
            aborted = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t src = sb + s * kPairStageBytes;
          const uint64_t da = smem_desc(src), db = smem_desc(src + kWBytes);
#pragma unroll
          for (int kk = 0; kk < BK / 32; ++kk)
            umma_i8_pair(tmem + b * kPairTokens, da + (uint64_t)(2 * kk), db + (uint64_t)(2 * kk),
                         idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          umma_commit_pair(empty0 + 8 * s);
        }
        umma_commit_pair(afull0 + 8 * b);
        ++j;
      }
    }
  } else {
    // epilogue: warp w reads TMEM lanes 32 (w % 4) .. +31; the two warps of a quarter take half of
    // the columns each.  Sixteen tokens at a time pass through the warp's own shared memory, so that
    // a thread holds eight adjacent outputs of a token.
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t leader_empty = map_rank(aempty0, 0);
    const uint32_t mine = sb + kPairOffOut + (warp - 2) * (16 * 32 * 4);
    const T* res = static_cast<const T*>(e.residual);
    T* out = static_cast<T*>(e.out);
    int j = 0;
    for (int t = first; t < g.items; t += stride) {
      const PairItem it = pair_item(t, g);
      if (it.m0 >= M) continue;
      const int b = j & 1;
      // wide: eight adjacent outputs of two of sixteen tokens; else one output of all of them
      const int n_warp = it.n0 + rank * 128 + 32 * q, m0 = it.m0;
      const int n_first = n_warp + (WIDE ? 8 * (lane & 3) : lane);
      float ws[8], bias[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int n = n_first + i;
        ws[i] = n < N ? __ldg(e.weight_scale + n) : 0.f;
        bias[i] = e.bias && n < N ? ep_f(static_cast<const T*>(e.bias)[n]) : 0.f;
      }
      if (!mbar_wait(afull0 + 8 * b, (j >> 1) & 1, status)) {
        aborted = 1;
        break;
      }
      tc_fence_after();
#pragma unroll 1
      for (int c0 = half * (it.width / 2); c0 < (half + 1) * (it.width / 2) && m0 + c0 < M; c0 += 16) {
        const int m = m0 + c0 + (lane & 15);
        const float sx = m < M ? __ldg(e.scale + m) : 0.f;
        uint32_t v[16];
        tmem_ld16(tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(b * kPairTokens + c0), v);
#pragma unroll
        for (int i = 0; i < 16; ++i) st_shared(mine + (i * 32 + lane) * 4, v[i]);
        __syncwarp();
        if constexpr (WIDE) {
          Eight<T> r[2] = {};
          const int a0 = lane >> 2;   // this thread's tokens of the sixteen: a0 and a0 + 8
          const int64_t at = (int64_t)(m0 + c0 + a0) * N + n_first;
          const bool in[2] = {n_first < N && m0 + c0 + a0 < M, n_first < N && m0 + c0 + a0 + 8 < M};
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (RES && in[i]) r[i].load(res + at + (int64_t)(8 * i) * N);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            int sum[8];
            ld_shared8(mine + ((a0 + 8 * i) * 32 + 8 * (lane & 3)) * 4, sum);
            const float s = __shfl_sync(0xffffffffu, sx, a0 + 8 * i);
            if (in[i])
              store8<T>(sum, s, ws, bias, RES, r[i], out + at + (int64_t)(8 * i) * N);
          }
        } else {
#pragma unroll 1
          for (int a0 = 0; a0 < 16; a0 += 8) {
            const int64_t at = (int64_t)(m0 + c0 + a0) * N + n_first;
            float r[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              r[i] = RES && n_first < N && m0 + c0 + a0 + i < M ? ep_f(res[at + (int64_t)i * N])
                                                                : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const TokenScale s(__shfl_sync(0xffffffffu, sx, a0 + i));
              const int sum = ld_shared(mine + ((a0 + i) * 32 + lane) * 4);
              if (n_first < N && m0 + c0 + a0 + i < M)
                out[at + (int64_t)i * N] = ep_t<T>(s.apply(sum, ws[0], bias[0]) + r[i]);
            }
          }
        }
        __syncwarp();   // read before the next tokens' sums are written
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(leader_empty + 8 * b);
      ++j;
    }
  }
  __syncwarp();
  // both CTAs are past their last use of either's shared memory and TMEM
  tc_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kPairTmemCols)
                 : "memory");
  }
  __syncthreads();
  cluster_arrive();
  cluster_wait();
}

// ---- host --------------------------------------------------------------------------------------

struct Problem {
  const int8_t* codes;
  const int8_t* weight;
  int64_t M, K, N;
  Epilogue e;
  unsigned int* status;
  cudaStream_t stream;
};

int set_smem(const void* kern, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && ((done.load() >> dev) & 1)) return RW4_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return fail(RW4_ECUDA, "int8_linear: cannot set the kernel's shared memory size");
  if (dev < 64) done.fetch_or(1ull << dev);
  return RW4_OK;
}

int weight_map(const Problem& p, CUtensorMap* w) {
  return make_tensor_map_2d(w, p.weight, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.N, p.K, p.K, BMW, BK,
                            CU_TENSOR_MAP_SWIZZLE_128B);
}

int token_map(const Problem& p, int box_tokens, CUtensorMap* x) {
  return make_tensor_map_2d(x, p.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.M, p.K, p.K, box_tokens,
                            BK, CU_TENSOR_MAP_SWIZZLE_128B);
}

int launch(const void* kern, int grid, int threads, int smem, int cluster, cudaStream_t stream,
           void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t err = cudaLaunchKernelExC(&cfg, kern, args);
  if (err != cudaSuccess) return cuda_status(err, "rw4 int8_linear launch");
  return launch_status("rw4 int8_linear launch");
}

template <int BN, typename T, bool WIDE, bool RES>
int launch_split(const Problem& p) {
  using C = SplitCfg<BN>;
  const void* kern = reinterpret_cast<const void*>(int8_split_kernel<BN, T, WIDE, RES>);
  static std::atomic<uint64_t> done{0};
  int st = set_smem(kern, C::kSmem, done);
  CUtensorMap w, x;
  if (st == RW4_OK) st = weight_map(p, &w);
  if (st == RW4_OK) st = token_map(p, BN, &x);
  if (st != RW4_OK) return st;
  int M = (int)p.M, N = (int)p.N, nkb = (int)((p.K + BK - 1) / BK);
  int m_tiles = (M + BN - 1) / BN;
  const int64_t tiles = (int64_t)m_tiles * ((N + BMW - 1) / BMW);
  // K is split until every SM has a CTA (four stages' worth of K left to each), and once more where
  // two fit on an SM and that leaves eight: 1 x 4096 x 4096 5.9 us at 128 CTAs (8 stages each), 6.6
  // at 256 (4 each); 64 x 14336 x 4096 16.6 at 128 (28 each), 15.5 at 256 (14 each).  More CTAs than
  // fit at once always lost (256 x 4096 x 6144: 96 CTAs 13.1 us, 192 in two waves 22.6).
  int log_splits = 0;
  auto may = [&](int64_t ctas, int stages) {
    return log_splits < 3 && (tiles << (log_splits + 1)) <= ctas &&
           (nkb >> (log_splits + 1)) >= stages;
  };
  while (may(sm_count(), 4)) ++log_splits;
  if (may((int64_t)sm_count() * C::kCtasPerSm, 8)) ++log_splits;
  Epilogue e = p.e;
  unsigned int* status = p.status;
  void* args[] = {&w, &x, &e, &M, &N, &nkb, &m_tiles, &log_splits, &status};
  return launch(kern, (int)(tiles << log_splits), C::kThreads, C::kSmem, 1 << log_splits, p.stream,
                args);
}

template <typename T, bool WIDE, bool RES>
int launch_pair(const Problem& p) {
  const void* kern = reinterpret_cast<const void*>(int8_pair_kernel<T, WIDE, RES>);
  static std::atomic<uint64_t> done{0};
  int st = set_smem(kern, kPairSmem, done);
  int M = (int)p.M, N = (int)p.N, nkb = (int)((p.K + BK - 1) / BK);
  PairGrid g;
  g.n_tiles = (N + kPairRows - 1) / kPairRows;
  g.m_tiles = (M + kPairTokens - 1) / kPairTokens;
  // The tiles that do not fill a last wave are cut into strips of 128 or 64 tokens, as long as those
  // fit in it (1500 x 4096 x 4096, 96 tiles for 74 pairs: 27.3 us whole, 25.2 cut; 700 x 8192 x 8192,
  // 96 tiles: 45.4 and 43.2; narrower strips only wait for their operands).
  const int tiles = g.n_tiles * g.m_tiles, pairs = sm_count() / 2, rest = tiles % pairs;
  g.full = tiles - rest;
  for (g.cut = 0; rest && g.cut < 2 && (rest << (g.cut + 1)) <= pairs;) ++g.cut;
  g.items = g.full + (rest << g.cut);
  CUtensorMap w, x, strip;
  if (st == RW4_OK) st = weight_map(p, &w);
  if (st == RW4_OK) st = token_map(p, kPairTokens / 2, &x);
  if (st == RW4_OK && g.cut) st = token_map(p, (kPairTokens >> g.cut) / 2, &strip);
  if (!g.cut) strip = x;
  if (st != RW4_OK) return st;
  Epilogue e = p.e;
  unsigned int* status = p.status;
  void* args[] = {&w, &x, &strip, &e, &M, &N, &nkb, &g, &status};
  return launch(kern, 2 * (g.items < pairs ? g.items : pairs), kPairThreads, kPairSmem, 2, p.stream,
                args);
}

// Which tiles (times of 148 SMs, in us):
//   up to 64 tokens   one tile of 16, 32 or 64 tokens, the narrowest that holds them
//   beyond            tiles of 128 tokens where one wave of CTAs takes them (384 x 4096 x 6144, 144
//                     tiles: 13.4 against 17.0 for pairs), of 64 where even that leaves most SMs idle
//                     (128 x 2048 x 2048, 16 tiles of 128: 6.1 against 7.6), else CTA pairs
//                     (512 x 4096 x 6144, 192 tiles: 17.3 against 24.2 in two waves)
template <typename T, bool WIDE, bool RES>
int run_tiles(const Problem& p, int32_t path) {
  const int64_t rows = (p.N + BMW - 1) / BMW, tiles128 = rows * ((p.M + 127) / 128);
  if (path == 2 || (path == 0 && p.M > 64 && tiles128 > sm_count()))
    return launch_pair<T, WIDE, RES>(p);
  if (p.M <= 16) return launch_split<16, T, WIDE, RES>(p);
  if (p.M <= 32) return launch_split<32, T, WIDE, RES>(p);
  if (p.M <= 64 || tiles128 <= 32) return launch_split<64, T, WIDE, RES>(p);
  return launch_split<128, T, WIDE, RES>(p);
}

// (the epilogue's forms are compiled apart: code that a launch does not run still cost a one-token
// call half a microsecond of instruction fetches)
template <typename T>
int run(const Problem& p, int32_t path) {
  const bool wide = wide_rows(p.e, p.N), res = p.e.residual != nullptr;
  if (wide)
    return res ? run_tiles<T, true, true>(p, path) : run_tiles<T, true, false>(p, path);
  return res ? run_tiles<T, false, true>(p, path) : run_tiles<T, false, false>(p, path);
}

}  // namespace

extern "C" int rw4_int8_linear(const int8_t* codes, const float* scale, int64_t M, int64_t K,
                               const int8_t* weight, const float* weight_scale, int64_t N,
                               const void* bias, const void* residual, void* out,
                               int32_t out_dtype, int32_t path, void* stream) {
  using namespace rw4;
  if (M < 0 || N < 0 || M > (1ll << 30) || N > (1ll << 30))
    return fail(RW4_EINVAL, "int8_linear: M=%lld N=%lld", (long long)M, (long long)N);
  if (K < 16 || K % 16 || K > kMaxK)
    return fail(RW4_EINVAL, "int8_linear: K=%lld (a multiple of 16 from 16 to %lld)", (long long)K,
                (long long)kMaxK);
  if (out_dtype != RW4_F32 && out_dtype != RW4_BF16 && out_dtype != RW4_F16)
    return fail(RW4_EINVAL, "int8_linear: out_dtype %d (0 f32, 1 bf16, 2 f16)", out_dtype);
  if (path < 0 || path > 2) return fail(RW4_EINVAL, "int8_linear: path %d (0, 1 or 2)", path);
  // tiles are counted in 32 bits: 128 weight rows x 16 tokens at the smallest, times 8 splits
  if (((M + 15) / 16) * ((N + 127) / 128) > (1ll << 27))
    return fail(RW4_EINVAL, "int8_linear: M=%lld x N=%lld is too large for one call", (long long)M,
                (long long)N);
  if (M == 0 || N == 0) return RW4_OK;
  if (!codes || !scale || !weight || !weight_scale || !out)
    return fail(RW4_EINVAL, "int8_linear: null pointer");
  if (!aligned(codes, 16) || !aligned(weight, 16))
    return fail(RW4_EINVAL, "int8_linear: codes and weight must be 16-byte aligned");
  const int es = out_dtype == RW4_F32 ? 4 : 2;
  if (!aligned(scale, 4) || !aligned(weight_scale, 4) || !aligned(out, es) || !aligned(bias, es) ||
      !aligned(residual, es))
    return fail(RW4_EINVAL, "int8_linear: a pointer is not aligned to its type");
  auto out_meets = [&](const void* p, int64_t bytes) { return meets(out, M * N * es, p, bytes); };
  if (out_meets(codes, M * K) || out_meets(weight, N * K) || out_meets(scale, 4 * M) ||
      out_meets(weight_scale, 4 * N) || out_meets(bias, N * es) ||
      (residual != out && out_meets(residual, M * N * es)))
    return fail(RW4_EINVAL, "int8_linear: out overlaps an input without being residual itself");
  Problem p;
  p.codes = codes;
  p.weight = weight;
  p.M = M;
  p.K = K;
  p.N = N;
  p.e = {scale, weight_scale, bias, residual, out};
  p.status = device_status_ptr();
  if (!p.status) return fail(RW4_ECUDA, "int8_linear: device status word unavailable");
  p.stream = as_stream(stream);
  if (out_dtype == RW4_F32) return run<float>(p, path);
  if (out_dtype == RW4_F16) return run<__half>(p, path);
  return run<__nv_bfloat16>(p, path);
}
