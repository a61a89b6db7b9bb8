// Self-attention on the 5th-generation tensor cores, forward and backward, for bf16 and fp16.
//
//   valid(i, j) = i < len, j < len and, if causal, j <= i        len: the sequence's length in a padded batch
//   S = scale Q K^T,  L_i = log sum_j exp S_ij,  P = exp(S - L) where valid and 0 elsewhere,  O = P V
//   dV = P^T dO,  dP = dO V^T,  D_i = dO_i . O_i,  dS = P (dP - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// Where rows have few keys, roundings to 16 bits show that average out elsewhere (and in a causal batch such rows make up most
// of dK).  So for rows of up to 128 keys, those of the first tile of queries if the batch is causal or the sequence ends there, the
// forward pass also leaves what the rounding of O dropped, in 8 bits, for D, which is a difference's other half.  And where no
// sequence has more than 128 positions, dS enters its products as a sum of two 16-bit values.  In the 2-norm, bf16, causal: 48 positions,
// dQ and dK off by 1.75e-3, of which the rounding of the result is 1.66e-3, instead of 2.6e-3; 8192 positions, dK 2.4e-3 instead of 2.5e-3.
//
// Nothing of size s x s reaches memory: the forward pass keeps a running maximum and sum per row and leaves L, the backward
// pass computes P again from S and L.  Exponentials are taken to base 2 (scale and log2 e in one factor), L is kept in
// units of log2.  Rows that the mask leaves empty (i >= len) get O = 0, L = +inf, and gradients of 0.
//
// All products run as tcgen05.mma on tiles of 128 rows with fp32 accumulators in TMEM.  A tile of probabilities goes back to
// TMEM in 16 bits and is the A operand of the next product from there; tiles of Q, K, V and dO come by TMA in the
// 128-byte-swizzled layout, which serves as a K-major operand (contraction over d) and as an MN-major one (contraction over
// tokens) alike.  Head sizes up to 128 run on tiles of 64 or 128 columns; TMA fills what lies beyond d with zeros.
//
// The last tile of a sequence may hold positions beyond its length.  Whatever stands there must not count, and 0 * NaN
// is NaN, so rows of a streamed tile that lie beyond the length are cleared in shared memory before they are contracted over.
//
// Every mbarrier wait is bounded; on a timeout the kernel sets an error word, frees its TMEM and returns.
//
// The reference contains no attention; this serves the BERT-shaped encoder.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "kernels/common.cuh"
#include "kernels/tcgen05.cuh"
#include "kernels/tips_kernels.h"

namespace tipsk {
namespace {

constexpr int kTile        = 128;  // rows of a tile of queries or keys
constexpr int kBoxBytes    = kTile * 128;  // 128 rows of 64 16-bit values
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFwdPoly = 8;  // forward, one pair of exponentials in so many by a polynomial (one in 4: 57 us where 8 takes 54, none: 56)
// fp16 has few exponents: forward, probabilities are held times 2^7 (so up to 2^15, see the lag of the maximum), which keeps those
// of the many small ones of a long row that 2^-25 of the largest would have lost.
constexpr float kHalfShift = 7.f;

__device__ int32_t g_attn_error;  // one per device

struct Strides {
  int64_t b, s, h;  // elements
};

__host__ __device__ __forceinline__ int TilesOf(int n, int tile) { return n / tile + (n % tile != 0); }

struct AttnParams {
  const void* lengths;  // [b] int32 or int64, or null
  int len64;
  int b, s, sp;         // sp: s rounded up to whole tiles, the row pitch of lse and delta
  int h, hk, d;
  int causal;
  float scale, c;       // c = scale * log2(e)
  float low;            // stands for the maximum of a row whose scores are -inf so far: low * c is finite
  float* lse;           // [b, h, sp]
  float* delta;         // [2][b, h, sp], and for fp16 [2][b, hk]
  uint8_t* rest;        // [b, min(s, 128), h, d]: what rounding dropped of O, times RestScale, as e5m2; null: not kept
  void *o, *dq, *dk, *dv;
  const void *dout, *v;
  Strides so, sdo, sdq, sdk, sdv, sv;
};

struct AttnMaps {
  CUtensorMap q, k, v, dout;
  CUtensorMap out, dq, dk, dv;  // written: boxes of 128 positions
};

// A value that all lanes of a warp hold, as the compiler can tell: what is computed from it stays in uniform registers, from
// which tcgen05.mma takes its operands, and branches on it do not diverge.
__device__ __forceinline__ uint32_t Uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

// Whether the rows of the first tile of a sequence of `len` positions have few keys.
__device__ __forceinline__ bool FewKeys(const AttnParams& p, int len) { return p.causal || len <= kTile; }
__device__ __forceinline__ int64_t RestAt(const AttnParams& p, int b, int row, int h) {
  return ((static_cast<int64_t>(b) * min(p.s, kTile) + row) * p.h + h) * p.d;
}
__device__ __forceinline__ int SeqLen(const AttnParams& p, int b) {
  if (p.lengths == nullptr) return p.s;
  const int64_t n = p.len64 ? static_cast<const int64_t*>(p.lengths)[b] : static_cast<const int32_t*>(p.lengths)[b];
  return static_cast<int>(n < 0 ? 0 : n > p.s ? p.s : n);
}

// Barriers and tiles by their shared-memory addresses: a base and constants, where pointers would take two registers each.
__device__ __forceinline__ void BarInit(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void BarExpect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void BarArrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void BarCommit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool BarTry(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity & 1)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ uint64_t NowNs() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Bounded waits of a whole warp, whose lanes get one answer: false on a timeout.  A poll that fails takes issue slots from
// the warps that compute, so the loop is short, and a warp that need not react at once (kIdle) sleeps between polls.
template <bool kIdle>
__device__ __forceinline__ bool BarWait(uint32_t bar, uint32_t parity) {
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (__all_sync(0xffffffffu, BarTry(bar, parity))) return true;
    if (kIdle) __nanosleep(100);
    if ((i & 1023) == 0) {
      const uint64_t now = NowNs();
      if (t0 == 0) t0 = now;
      else if (__any_sync(0xffffffffu, now - t0 > kWaitBudgetNs)) return false;
    }
  }
}
// Of one thread, which need not react at once.
__device__ __forceinline__ bool BarWaitOne(uint32_t bar, uint32_t parity) {
  uint64_t t0 = 0;
  for (uint32_t i = 1; !BarTry(bar, parity); ++i) {
    __nanosleep(40);
    if ((i & 1023) == 0) {
      const uint64_t now = NowNs();
      if (t0 == 0) t0 = now;
      else if (now - t0 > kWaitBudgetNs) return false;
    }
  }
  return true;
}

// 64 columns x 128 rows of one head: x along d, then position, head, batch.
__device__ __forceinline__ void TmaLoadHead(uint32_t dst, const CUtensorMap* map, int x, int s, int h, int b, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(s), "r"(h), "r"(b), "r"(bar)
      : "memory");
}
// kRows positions of a head by boxes of kBox rows; a box of 64 columns with all its rows follows the other.
template <int HD, int kRows, int kBox>
__device__ __forceinline__ void TmaLoadTile(uint32_t dst, const CUtensorMap* map, int s, int h, int b, uint32_t bar) {
#pragma unroll
  for (int x = 0; x < HD / 64; ++x)
#pragma unroll
    for (int r = 0; r < kRows; r += kBox) TmaLoadHead(dst + (x * kRows + r) * 128, map, x * 64, s + r, h, b, bar);
}
// `bytes` (a multiple of 16) from 16-byte-aligned global memory.
__device__ __forceinline__ void BulkLoad(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// D += A B with A (128 x 16) in TMEM: lane = row, two 16-bit values per column.
__device__ __forceinline__ void UmmaTmemA(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void TmemLoad16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void TmemStore16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void TmemStoreWait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <bool kBf16>
__device__ __forceinline__ uint32_t Pack2(float lo, float hi) {
  uint32_t r;
  if (kBf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    r = *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    r = *reinterpret_cast<const uint32_t*>(&v);
  }
  return r;
}
template <bool kBf16>
__device__ __forceinline__ float2 Unpack2(uint32_t r) {
  if (kBf16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r));
  return __half22float2(*reinterpret_cast<const __half2*>(&r));
}

// Instruction descriptor of a 128 x n product with fp32 accumulators; b_mn: B is MN-major.
template <bool kBf16>
__device__ __forceinline__ uint32_t InstrDesc(int n, bool b_mn) {
  return (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kTile >> 4) << 24);
}

// [128 x d] x [kN x d]^T: both operands K-major in shared memory, boxes of 64 columns.
template <bool kBf16, int kD, int kN>
__device__ __forceinline__ void IssueScores(uint32_t tmem_d, uint32_t a_addr, uint32_t b_addr, int ksteps) {
  const uint64_t a = SmemDescSw128(a_addr), b = SmemDescSw128(b_addr);
  const uint32_t idesc = InstrDesc<kBf16>(kN, false);
#pragma unroll
  for (int k = 0; k < kD / 16; ++k) {
    if (k < ksteps) UmmaBf16(tmem_d, a + (k >> 2) * (kBoxBytes >> 4) + (k & 3) * 2, b + (k >> 2) * (kN * 128 >> 4) + (k & 3) * 2, idesc, k > 0);
  }
}
// [128 x kK] (16-bit, TMEM) x [kK x n]: B MN-major in shared memory.  The columns of A lie in runs of kRun, two per TMEM
// column, kRun columns apart (each where the fp32 values that it was made of had been).
template <bool kBf16, int kK, int kRun>
__device__ __forceinline__ void IssueFromTmem(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_addr, int n, bool accum) {
  const uint64_t b     = SmemDescMnSw128(b_addr, kK * 128);
  const uint32_t idesc = InstrDesc<kBf16>(n, true);
#pragma unroll
  for (int k = 0; k < kK / 16; ++k)
    UmmaTmemA(tmem_d, tmem_a + k * 16 / kRun * kRun + k * 16 % kRun / 2, b + 128 * k, idesc, accum || k > 0);
}

// Clears rows [first, kRows) of `boxes` boxes of kRows rows (a whole warp; the swizzle stays within a row's 128 bytes) and
// orders the writes before the MMAs that follow.
template <int kRows>
__device__ __forceinline__ void ClearRows(uint32_t tile, int boxes, int first) {
  const int lane = threadIdx.x & 31;
  for (int x = 0; x < boxes; ++x)
    for (int i = first * 8 + lane; i < kRows * 8; i += 32)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + (x * kRows * 8 + i) * 16), "r"(0) : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

template <bool kBf16, int kCols>
__device__ __forceinline__ void StoreCols(uint16_t* row, int col0, int d, const uint32_t (&acc)[kCols], float factor) {
#pragma unroll
  for (int g = 0; g < kCols / 8; ++g) {
    if (col0 + g * 8 >= d) break;  // d is a multiple of 8
    uint4 v;
    v.x = Pack2<kBf16>(__uint_as_float(acc[g * 8 + 0]) * factor, __uint_as_float(acc[g * 8 + 1]) * factor);
    v.y = Pack2<kBf16>(__uint_as_float(acc[g * 8 + 2]) * factor, __uint_as_float(acc[g * 8 + 3]) * factor);
    v.z = Pack2<kBf16>(__uint_as_float(acc[g * 8 + 4]) * factor, __uint_as_float(acc[g * 8 + 5]) * factor);
    v.w = Pack2<kBf16>(__uint_as_float(acc[g * 8 + 6]) * factor, __uint_as_float(acc[g * 8 + 7]) * factor);
    *reinterpret_cast<uint4*>(row + col0 + g * 8) = v;
  }
}
// What the rounding of O to 16 bits drops is at most 2^-9 |O| (bf16) or 2^-12 |O|; e5m2 has 3 bits of it between 2^-14 and 2^15.
template <bool kBf16>
__device__ __forceinline__ constexpr float RestScale() { return kBf16 ? 256.f : 2048.f; }
template <bool kBf16, int kCols>
__device__ __forceinline__ void StoreRest(uint8_t* row, int col0, int d, const uint32_t (&acc)[kCols], float factor) {
#pragma unroll
  for (int g = 0; g < kCols / 8; ++g) {
    if (col0 + g * 8 >= d) break;
    uint32_t r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = __uint_as_float(acc[g * 8 + 2 * k]) * factor, b = __uint_as_float(acc[g * 8 + 2 * k + 1]) * factor;
      const float2 kept = Unpack2<kBf16>(Pack2<kBf16>(a, b));
      uint16_t pair;
      asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(pair) : "f"((b - kept.y) * RestScale<kBf16>()), "f"((a - kept.x) * RestScale<kBf16>()));
      r[k] = pair;
    }
    *reinterpret_cast<uint2*>(row + col0 + g * 8) = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
  }
}
__device__ __forceinline__ float2 UnpackE5m2(uint32_t pair) {
  uint32_t h;
  asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(pair)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// The same of a row into a staged tile, whose boxes of 64 columns and 128 rows have the swizzled layout that a TMA store reads;
// rows that are not live are zero.
template <bool kBf16, int kCols>
__device__ __forceinline__ void StageCols(uint32_t tile, int r, int col0, const uint32_t (&acc)[kCols], float factor, bool live) {
#pragma unroll
  for (int g = 0; g < kCols / 8; ++g) {
    uint32_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = live ? Pack2<kBf16>(__uint_as_float(acc[g * 8 + 2 * k]) * factor, __uint_as_float(acc[g * 8 + 2 * k + 1]) * factor) : 0u;
    const int c = col0 + g * 8;
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tile + (c >> 6) * kBoxBytes + r * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4)),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                 : "memory");
  }
}
// A staged tile into memory, by one thread: what lies beyond the tensor's positions and columns is not written.
template <int HD>
__device__ __forceinline__ void TmaStoreTile(uint32_t tile, const CUtensorMap* map, int s, int h, int b) {
#pragma unroll
  for (int x = 0; x < HD / 64; ++x)
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x * 64), "r"(s), "r"(h), "r"(b), "r"(tile + x * kBoxBytes)
                 : "memory");
}
// Until this thread's stores have read their tiles.
__device__ __forceinline__ void StoresRead() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
// Rows [first, last) of one head to zero, by a warp, neighbouring lanes within a row.
__device__ __forceinline__ void StoreZeroRows(void* tensor, const Strides& st, int b, int h, int first, int last, int d) {
  uint16_t* base = static_cast<uint16_t*>(tensor) + b * st.b + h * st.h;
  const int vecs = d >> 3;
  int row = first, c = threadIdx.x & 31;
  while (c >= vecs) {
    c -= vecs;
    ++row;
  }
  while (row < last) {
    *reinterpret_cast<uint4*>(base + row * st.s + c * 8) = make_uint4(0, 0, 0, 0);
    c += 32;
    while (c >= vecs) {
      c -= vecs;
      ++row;
    }
  }
}

__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Maximum that hands on a NaN of either operand.
__device__ __forceinline__ float MaxNan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 Add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float MaxNan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^x on the FMA pipe, for a share of the exponentials: ex2.approx runs at 16 per SM and clock, and a tile has 16384.
// x = n + f with n = rint(x) (by adding 1.5 * 2^23, whose last bits then hold n), |f| <= 0.5; 2^f by the polynomial of degree 4
// with the least relative error on that interval (2.6e-6, by the Remez exchange); times 2^n, made of n's bits.  Below -127
// the result is 0 (2^-127 has a zero exponent field), a NaN stays one.  One value at a time: constants are immediate
// operands then, where a pair would need them in registers.
__device__ __forceinline__ float Exp2Poly(float x) {
  x = MaxNan(x, -127.f);
  const float t = x + 12582912.f;
  const float f = x - (t - 12582912.f);
  float q = fmaf(f, 0.009570102207362652f, 0.05591785907745361f);
  q = fmaf(q, f, 0.240247443318367f);
  q = fmaf(q, f, 0.6931217908859253f);
  q = fmaf(q, f, 0.9999992847442627f);
  return q * __int_as_float((__float_as_int(t) << 23) + 0x3f800000);
}
// Pair k of a run: one in kEvery by the polynomial.
template <int kEvery>
__device__ __forceinline__ F2 Exp2Mixed(F2 x, int k) {
  if (k % kEvery != kEvery - 1) return Exp2Fast(x);
  const float2 v = SplitF2(x);
  return MakeF2(Exp2Poly(v.x), Exp2Poly(v.y));
}
__device__ __forceinline__ F2 Pair(uint32_t a, uint32_t b) { return MakeF2(__uint_as_float(a), __uint_as_float(b)); }
template <bool kBf16>
__device__ __forceinline__ uint32_t Pack2(F2 a) {
  const float2 x = SplitF2(a);
  return Pack2<kBf16>(x.x, x.y);
}

// What rounding to `kept` dropped of a pair, in 16 bits.
template <bool kBf16>
__device__ __forceinline__ uint32_t PackRest(F2 a, uint32_t kept) {
  const float2 x = SplitF2(a), y = Unpack2<kBf16>(kept);
  return Pack2<kBf16>(x.x - y.x, x.y - y.y);
}

__device__ __forceinline__ float LoadShared(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}
// Four neighbouring values, 16-byte aligned, as two pairs.
__device__ __forceinline__ void LoadPairs(uint32_t at, F2& a, F2& b) {
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(a.v), "=l"(b.v) : "r"(at) : "memory");
}

// ---------------------------------------------------------------- blocks that take one piece of work after another
// The grid has a block per piece of work, but a block that is done takes the place of one that has not started yet (cluster
// launch control): its barriers, its TMEM and its pipelines stay up, loads and scores of the next piece run under the
// last stores of this one, and pieces of different length still spread evenly.  The thread that issues TMA loads asks for the
// next piece while it works on the present one, works out what the piece consists of, and leaves that in one of two slots
// in shared memory for the other warps, which run through the same pieces.
struct Pieces {
  uint32_t at;  // two slots of eight words, an answer of 16 bytes, barriers: slots written [2], slots read [2], answer
  static constexpr int kBytes = 64 + 16 + 48;
  __device__ __forceinline__ uint32_t Slot(uint32_t turn) const { return at + (turn & 1) * 32; }
  __device__ __forceinline__ uint32_t Answer() const { return at + 64; }
  __device__ __forceinline__ uint32_t Full(uint32_t turn) const { return at + 80 + (turn & 1) * 8; }
  __device__ __forceinline__ uint32_t Empty(uint32_t turn) const { return at + 96 + (turn & 1) * 8; }
  __device__ __forceinline__ uint32_t Answered() const { return at + 112; }
  __device__ __forceinline__ void Init(int followers) const {  // warps that follow
    for (int i = 0; i < 2; ++i) {
      BarInit(Full(i), 1);
      BarInit(Empty(i), followers);
    }
    BarInit(Answered(), 1);
  }
  // By the thread that leads: `describe` turns a block index into eight words, the last not negative, and `load` starts the loads of
  // a piece; both come from the piece's type.  False on a timeout.
  template <typename Describe, typename Load>
  __device__ __forceinline__ bool Lead(Describe&& describe, Load&& load) const {
    int index = blockIdx.x;
    for (uint32_t turn = 0;; ++turn) {
      int w[8];
      if (index >= 0) describe(index, w);
      else w[7] = -1;
      if (!BarWaitOne(Empty(turn), (turn >> 1) ^ 1)) return false;
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(Slot(turn)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(Slot(turn) + 16), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
      BarArrive(Full(turn));
      if (index < 0) return true;
      BarExpect(Answered(), 16);
      asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(Answer()),
                   "r"(Answered())
                   : "memory");
      bool ok = load(w);
      ok      = BarWaitOne(Answered(), turn) && ok;
      uint32_t got, x;
      asm volatile(
          "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
          "ld.shared.b128 r, [%2];\n\t"
          "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t"
          "mov.u32 %1, 0;\n\t"
          "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
          : "=r"(got), "=r"(x)
          : "r"(Answer())
          : "memory");
      if (!ok) return false;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next answer is written to the same place
      index = got ? static_cast<int>(x) : -1;
    }
  }
  // By every other warp, from turn 0 on: the piece's words, the same in all lanes; false when there are no more.
  template <bool kIdle>
  __device__ __forceinline__ bool Take(uint32_t turn, int (&w)[8]) const {
    if (!BarWait<kIdle>(Full(turn), turn >> 1)) {
      if ((threadIdx.x & 31) == 0) atomicExch(&g_attn_error, 8);
      return false;
    }
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(Slot(turn)) : "memory");
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "r"(Slot(turn) + 16)
                 : "memory");
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = Uniform(w[k]);
    if ((threadIdx.x & 31) == 0) BarArrive(Empty(turn));
    return w[7] >= 0;
  }
};

// A wait that remembers a failure, for warps that go on to the next piece; reports it once under `code`.
template <bool kIdle>
struct WaiterOf {
  int code;
  bool ok = true;
  __device__ __forceinline__ explicit WaiterOf(int c) : code(c) {}
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) {
    if (ok && !BarWait<kIdle>(bar, parity)) {
      if ((threadIdx.x & 31) == 0) atomicExch(&g_attn_error, code);
      ok = false;
    }
    TcFenceAfter();
    return ok;
  }
};
using Waiter     = WaiterOf<false>;
using IdleWaiter = WaiterOf<true>;

__device__ __forceinline__ void AllocTmem(uint32_t slot, uint32_t columns) {  // by one warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t AlignedSmem(const uint8_t* raw) { return (SmemAddr(raw) + 1023) & ~1023u; }

// ---------------------------------------------------------------- forward
// A piece of work is 256 queries of one head as two tiles, past which the keys and values stream in units.  A thread has a row of a
// tile, so maximum and sum need no exchange; a tile's probabilities take the place of its scores, and the next scores follow the
// product with V, so that one barrier tells that both are done.  While one tile waits for its products, others compute:
// with 64 output columns, units of 64 keys leave TMEM for two blocks per SM, four tiles that run apart from each other
// (32 x 512, 16 heads of 64: 53 us; one block with units of 128, next scores beside the probabilities, and a row shared
// by two threads: 61).  With 128 one block fills TMEM, units have 128 keys, and one warp issues the products of both tiles, which
// makes them take turns (8192, 16 heads of 128 that share 4, causal: 225 us = 1220 TFLOP/s; with a warp for each tile 248; in a long loop
// of forward and backward passes, at the 1665 MHz that the power limit leaves, 268).
// Bound, within a long piece of 64 columns, by the unit for exponentials, which is busy four fifths of the time, and by issue slots
// beside it; at 512 positions also by the start and the end of a piece.  With 128 columns by the way from a tile's scores through its
// probabilities and products to its next scores (3300 clocks, of which the tensor cores work 2050 for both tiles).
template <int HD>
struct FwdCfg {
  static constexpr int kTileBytes = (HD / 64) * kBoxBytes;
  static constexpr int kUnit      = HD == 64 ? 64 : 128;
  static constexpr int kUnitBytes = kUnit * HD * 2;
  static constexpr int kBlocks    = HD == 64 ? 2 : 1;  // per SM
  static constexpr int kStages    = 4;  // units of K and V in turn
  static constexpr int kQBufs     = HD == 64 ? 2 : 1;  // queries of this piece of work and the next
  // outputs leave by TMA through the place of their queries, where the next piece has another
  static constexpr bool kStaged   = kQBufs == 2;
  static constexpr int kSoftWarps = 8;                 // four for each tile
  static constexpr int kTmaWarp   = kSoftWarps, kMmaWarp = kSoftWarps + 1;
  static constexpr int kThreads   = (kSoftWarps + 2) * 32;
  static constexpr int kColumns   = 2 * (kUnit + HD);  // of TMEM: scores and output of either tile
  // shared memory: queries [kQBufs][2], the ring, barriers
  static constexpr int kRing      = 2 * kQBufs * kTileBytes;
  static constexpr int kNext      = kRing + kStages * kUnitBytes;
  static constexpr int kFull      = kNext + Pieces::kBytes;
  static constexpr int kEmpty     = kFull + 8 * kStages;
  static constexpr int kQFull     = kEmpty + 8 * kStages;
  static constexpr int kQEmpty    = kQFull + 8 * kQBufs;
  static constexpr int kSFull     = kQEmpty + 8 * kQBufs;  // [2] scores of a tile are in TMEM, and the products before are done
  static constexpr int kPFull     = kSFull + 16;           // [2] the probabilities are in TMEM
  static constexpr int kOFull     = kPFull + 16;           // [2] a piece's output is complete
  static constexpr int kOStaged   = kOFull + 16;           // [2] it is in shared memory
  static constexpr int kTmemSlot  = kOStaged + 16;
  static constexpr int kSmemBytes = kTmemSlot + 16 + 1024;
};

struct FwdPiece {
  int b, h, q0, len, count0, count1, total;
  bool ragged;  // the last unit of V has rows to clear
  __device__ __forceinline__ explicit FwdPiece(const int (&w)[8])
      : b(w[0]), h(w[1]), q0(w[2]), len(w[3]), count0(w[4]), count1(w[5]), total(w[6]), ragged(w[7] != 0) {}
  template <int kUnit>
  __device__ __forceinline__ static void Describe(const AttnParams& p, int index, int (&w)[8]) {
    // causal: the tiles with the most keys first; otherwise neighbours share a head's keys
    const int blocks_q = TilesOf(p.s, 2 * kTile), heads = p.b * p.h;
    const int qb = p.causal ? blocks_q - 1 - index / heads : index % blocks_q;
    const int bh = p.causal ? index % heads : index / blocks_q;
    const int b = bh / p.h, q0 = qb * 2 * kTile, len = SeqLen(p, b), units = TilesOf(len, kUnit);
    // units of keys of either query tile
    const int count0 = q0 >= len ? 0 : p.causal ? min(units, (q0 + kTile) / kUnit) : units;
    const int count1 = q0 + kTile >= len ? 0 : p.causal ? min(units, (q0 + 2 * kTile) / kUnit) : units;
    const int total = max(count0, count1);
    w[0] = b;
    w[1] = bh % p.h;
    w[2] = q0;
    w[3] = len;
    w[4] = count0;
    w[5] = count1;
    w[6] = total;
    w[7] = total > 0 && total == units && len < p.s && len % kUnit != 0;
  }
};

template <int HD, bool kBf16>
__global__ void __launch_bounds__(FwdCfg<HD>::kThreads, FwdCfg<HD>::kBlocks)
AttnFwdKernel(const __grid_constant__ AttnMaps maps, const __grid_constant__ AttnParams p) {
  using Cfg = FwdCfg<HD>;
  constexpr int S = Cfg::kStages, QB = Cfg::kQBufs, kUnit = Cfg::kUnit;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = AlignedSmem(smem_raw);
  const Pieces pieces{base + Cfg::kNext};
  auto full = [&](uint32_t k) { return base + Cfg::kFull + k % S * 8; };
  auto empty = [&](uint32_t k) { return base + Cfg::kEmpty + k % S * 8; };
  auto q_full = [&](uint32_t n) { return base + Cfg::kQFull + n % QB * 8; };
  auto q_empty = [&](uint32_t n) { return base + Cfg::kQEmpty + n % QB * 8; };
  auto q_tile = [&](uint32_t n, int i) { return base + (n % QB * 2 + i) * Cfg::kTileBytes; };
  auto unit = [&](uint32_t k) { return base + Cfg::kRing + k % S * Cfg::kUnitBytes; };

  const int warp = Uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    pieces.Init(Cfg::kSoftWarps + 1);
    for (int i = 0; i < S; ++i) {
      BarInit(full(i), 1);
      BarInit(empty(i), 1);
    }
    for (int i = 0; i < QB; ++i) {
      BarInit(q_full(i), 1);
      BarInit(q_empty(i), Cfg::kStaged ? 2 : 1);  // the products are done with the queries, and what took their place is stored
    }
    for (int i = 0; i < 2; ++i) {
      BarInit(base + Cfg::kSFull + i * 8, 1);
      BarInit(base + Cfg::kPFull + i * 8, Cfg::kSoftWarps / 2);
      BarInit(base + Cfg::kOFull + i * 8, 1);
      BarInit(base + Cfg::kOStaged + i * 8, Cfg::kSoftWarps / 2);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == Cfg::kMmaWarp) AllocTmem(base + Cfg::kTmemSlot, Cfg::kColumns);
  TcFenceBefore();
  __syncthreads();
  TcFenceAfter();
  const uint32_t tmem = Uniform(__float_as_uint(LoadShared(base + Cfg::kTmemSlot)));
  const uint32_t t_s = tmem, t_o = tmem + 2 * kUnit;  // scores of either tile, in their place the probabilities; either output

  int words[8] = {};
  if (warp == Cfg::kTmaWarp) {
    if (ElectOne()) {
      uint32_t e = 0, n = 0;  // units of K and V, and pieces with any, so far
      const bool ok = pieces.Lead([&](int index, int (&v)[8]) { FwdPiece::Describe<kUnit>(p, index, v); }, [&](const int (&v)[8]) {
        const FwdPiece w(v);
        if (w.total == 0) return true;
        if (!BarWaitOne(q_empty(n), (n / QB) ^ 1)) return false;
        BarExpect(q_full(n), 2 * Cfg::kTileBytes);
        TmaLoadTile<HD, kTile, kTile>(q_tile(n, 0), &maps.q, w.q0, w.h, w.b, q_full(n));
        TmaLoadTile<HD, kTile, kTile>(q_tile(n, 1), &maps.q, w.q0 + kTile, w.h, w.b, q_full(n));
        ++n;
        const int hk = w.h / (p.h / p.hk);
        for (int k = 0; k < 2 * w.total; ++k, ++e) {
          if (!BarWaitOne(empty(e), (e / S) ^ 1)) return false;
          BarExpect(full(e), Cfg::kUnitBytes);
          TmaLoadTile<HD, kUnit, kUnit>(unit(e), k & 1 ? &maps.v : &maps.k, (k >> 1) * kUnit, hk, w.b, full(e));
        }
        return true;
      });
      if (!ok) atomicExch(&g_attn_error, 1);
    }
  } else if (warp == Cfg::kMmaWarp) {
    const int ksteps = (p.d + 15) >> 4, n_out = ksteps * 16;
    uint32_t e = 0, n = 0, done[2] = {0, 0}, staged[2] = {0, 0};  // done, staged: units and pieces of a tile so far
    Waiter wait(3);
    auto s_full = [&](int i) { return base + Cfg::kSFull + i * 8; };
    // The output of an earlier piece is stored when this piece's first scores are on their way.
    FwdPiece owed(words);
    owed.total = 0;
    auto settle = [&] {
      if (!Cfg::kStaged || owed.total == 0) return;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if ((i ? owed.count1 : owed.count0) == 0) continue;
        if (!wait(base + Cfg::kOStaged + i * 8, staged[i]++)) return;
        if (ElectOne()) TmaStoreTile<HD>(q_tile(n - 1, i), &maps.out, owed.q0 + i * kTile, owed.h, owed.b);
      }
      if (ElectOne()) {
        StoresRead();
        BarArrive(q_empty(n - 1));
      }
      __syncwarp();
      owed.total = 0;
    };
    for (uint32_t turn = 0; pieces.Take<false>(turn, words); ++turn) {
      const FwdPiece w(words);
      if (w.total == 0 || !wait.ok) continue;
      const int count[2] = {w.count0, w.count1};
      auto scores = [&](int i, int j) {  // tile i, unit j
        IssueScores<kBf16, HD, kUnit>(t_s + i * kUnit, q_tile(n, i), unit(e + 2 * j), ksteps);
        BarCommit(s_full(i));
      };
      auto entry = [&](uint32_t k) { return wait(full(k), k / S); };
      if (wait(q_full(n), n / QB) && entry(e) && ElectOne()) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (count[i] > 0) scores(i, 0);
        BarCommit(empty(e));
        if (w.total == 1) BarCommit(q_empty(n));
      }
      __syncwarp();
      settle();
      for (int j = 0; j < w.total && wait.ok; ++j) {
        const uint32_t ev = e + 2 * j + 1;
        if (!entry(ev)) break;
        if (w.ragged && j + 1 == w.total) ClearRows<kUnit>(unit(ev), HD / 64, w.len % kUnit);
        if (j + 1 < w.total && !entry(ev + 1)) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (j >= count[i] || !wait(base + Cfg::kPFull + i * 8, done[i]++)) continue;
          if (ElectOne()) {
            IssueFromTmem<kBf16, kUnit, kUnit>(t_o + i * HD, t_s + i * kUnit, unit(ev), n_out, j > 0);
            if (j + 1 < count[i]) scores(i, j + 1);  // products complete in the order of their issue
            else BarCommit(base + Cfg::kOFull + i * 8);
          }
          __syncwarp();
        }
        if (!wait.ok) break;
        if (ElectOne()) {
          BarCommit(empty(ev));
          if (j + 1 < w.total) BarCommit(empty(ev + 1));
          if (j + 2 == w.total) BarCommit(q_empty(n));
        }
        __syncwarp();
      }
      e += 2 * w.total;
      ++n;
      owed = w;
    }
    if (wait.ok) settle();
    if (Cfg::kStaged && ElectOne()) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else {
    const int i = warp / 4, quarter = warp & 3;  // query tile, TMEM lanes that this warp may access
    const int r = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t ts = t_s + lanes + i * kUnit, to = t_o + lanes + i * HD;
    const F2 c2 = Both(p.c);
    const uint32_t s_full = base + Cfg::kSFull + i * 8, p_full = base + Cfg::kPFull + i * 8;
    uint32_t done = 0, pieces_done = 0, outputs = 0;
    Waiter wait(4);
    for (uint32_t turn = 0; pieces.Take<false>(turn, words); ++turn) {
      const FwdPiece w(words);
      const int row = w.q0 + i * kTile + r, count = i ? w.count1 : w.count0;
      float m = 0.f, l = 0.f;  // row maximum (of the raw scores) that the exponents refer to, and the sum
      for (int j = 0; j < count; ++j, ++done) {
        wait(s_full, done);  // on a failure the values are void: they are neither handed on nor stored
        uint32_t s[kUnit / 32][32];
#pragma unroll
        for (int g = 0; g < kUnit / 32; ++g) TmemLoad32Async(ts + g * 32, s[g]);
#pragma unroll
        for (int g = 0; g < kUnit / 32; ++g) TmemLoadWait(s[g]);
        const int kv0 = j * kUnit;
        if (kv0 + kUnit > w.len || (p.causal && kv0 + kUnit - 1 > w.q0 + i * kTile)) {
          const int limit = (p.causal ? min(w.len, row + 1) : w.len) - kv0;
#pragma unroll
          for (int k = 0; k < kUnit; ++k)
            if (k >= limit) s[k >> 5][k & 31] = 0xff800000u;  // -inf
        }
        float part[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          constexpr int kRun = kUnit / 4;
          auto at = [&](int k) { return __uint_as_float(s[(u * kRun + k) >> 5][(u * kRun + k) & 31]); };
          part[u] = MaxNan(at(0), at(1));
#pragma unroll
          for (int k = 2; k < kRun; k += 2) part[u] = MaxNan(part[u], at(k), at(k + 1));
        }
        float top = MaxNan(MaxNan(part[0], part[1], part[2]), part[3]);
        // a row whose scores are -inf so far: any finite reference below the scores to come; and inf - inf: the row is NaN, as by the
        // formula
        if (top == -INFINITY) top = p.low;
        else if (top == INFINITY) top = __uint_as_float(0x7fc00000u);
        // The exponents' reference may lag behind the maximum by up to 2^8: probabilities of up to 256 lose nothing in 16 bits,
        // and the output in TMEM is rescaled a few times per row instead of with every new maximum.
        if (j == 0) {
          m = top;
        } else if (__any_sync(0xffffffffu, !((top - m) * p.c <= 8.f))) {
          const float up = MaxNan(top, m);
          const float f  = Exp2((m - up) * p.c);
          m = up;
          l *= f;
#pragma unroll 1
          for (int g = 0; g < HD / 16; ++g) {  // the products before these scores are done
            uint32_t o[16];
            TmemLoad16(to + g * 16, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            TmemStore16(to + g * 16, o);
          }
        }
        const F2 nm = Both(fmaf(-m, p.c, kBf16 ? 0.f : kHalfShift));
        F2 sum[2];
#pragma unroll
        for (int g = 0; g < kUnit / 32; ++g) {
          uint32_t v[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const F2 x = Exp2Mixed<kFwdPoly>(Fma2(Pair(s[g][2 * k], s[g][2 * k + 1]), c2, nm), k);
            sum[k & 1] = g == 0 && k < 2 ? x : Add2(sum[k & 1], x);
            v[k] = Pack2<kBf16>(x);
          }
          TmemStore16(ts + g * 16, v);
        }
        const float2 both = SplitF2(Add2(sum[0], sum[1]));
        l += both.x + both.y;
        TmemStoreWait();
        TcFenceBefore();
        __syncwarp();
        if (lane == 0 && wait.ok) BarArrive(p_full);
      }
      const bool live = row < w.len;
      uint16_t* dst = static_cast<uint16_t*>(p.o) + w.b * p.so.b + row * p.so.s + w.h * p.so.h;
      if (count > 0) {
        wait(base + Cfg::kOFull + i * 8, outputs++);
        const float inv = 1.f / l;
        const bool rest = p.rest && w.q0 + i * kTile == 0 && FewKeys(p, w.len);
#pragma unroll
        for (int g = 0; g < HD / 32; ++g) {
          uint32_t o[32];
          TmemLoad32(to + g * 32, o);
          if (Cfg::kStaged) StageCols<kBf16, 32>(q_tile(pieces_done, i), r, g * 32, o, inv, live);
          else if (live && wait.ok) StoreCols<kBf16, 32>(dst, g * 32, p.d, o, inv);
          if (rest && live && wait.ok) StoreRest<kBf16, 32>(p.rest + RestAt(p, w.b, row, w.h), g * 32, p.d, o, inv);
        }
        TcFenceBefore();
        if (Cfg::kStaged) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && wait.ok) BarArrive(base + Cfg::kOStaged + i * 8);
        }
      }
      pieces_done += w.total > 0;
      if (!Cfg::kStaged || count == 0) {  // rows beyond the sequence
        const int first = w.q0 + i * kTile + quarter * 32;
        StoreZeroRows(p.o, p.so, w.b, w.h, max(first, w.len), min(first + 32, p.s), p.d);
      }
      if (row < p.sp && wait.ok)
        p.lse[(static_cast<int64_t>(w.b) * p.h + w.h) * p.sp + row] = live ? fmaf(m, p.c, log2f(l) - (kBf16 ? 0.f : kHalfShift)) : INFINITY;
    }
  }
  TcFenceBefore();
  __syncthreads();
  if (warp == Cfg::kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(static_cast<uint32_t>(Cfg::kColumns)) : "memory");
}

// ---------------------------------------------------------------- backward
// fp16 has few exponents: gradients are scaled by whole powers of two on their way through it.  P, at most 1, is held times 2^10,
// so that the probabilities of long sequences stay clear of its smallest numbers; dS times 2^k, with k from the largest |dO| of the
// heads that share a key and value head and the largest |V|: |dS| <= 2 d max|dO| max|V|, and 2^k times that is below 2^15.
constexpr int kHalfP = 10;
__device__ __forceinline__ float TwoTo(int k) { return __int_as_float((k + 127) << 23); }

// D_i = dO_i . O_i, with what rounding dropped of O, eight lanes per row.  A block takes 32 positions of eight heads: it reads runs of heads, which are neighbours
// in a contiguous tensor, and writes runs of positions.  Writes [2][b, h, sp]: -L and -D, the addends as the main kernel uses them.
// For fp16 further blocks read V, and the largest magnitudes go to [2][b, hk] behind that, cleared before.
// Bound by HBM: 32 x 512, 16 heads of 64, 67 MB read in 20 us from a cold L2 (3.4 TB/s; 10 us at HBM's rate, which so short a
// launch does not reach), 13 us behind the forward pass.
template <bool kBf16>
__global__ void __launch_bounds__(256) AttnDeltaKernel(const __grid_constant__ AttnParams p) {
  __shared__ float sums[8][33];
  const int b = blockIdx.z, len = SeqLen(p, b), runs = TilesOf(p.h, 8);
  const int64_t plane = static_cast<int64_t>(p.b) * p.h * p.sp;
  const int h = (threadIdx.x >> 3) & 7, part = threadIdx.x & 7;
  const bool values = !kBf16 && static_cast<int>(blockIdx.y) >= runs;
  const int h0 = (blockIdx.y - (values ? runs : 0)) * 8, heads = values ? p.hk : p.h;
  const uint16_t* out  = static_cast<const uint16_t*>(p.o) + b * p.so.b + (h0 + h) * p.so.h + part * 8;
  const uint16_t* grad = values ? static_cast<const uint16_t*>(p.v) + b * p.sv.b + (h0 + h) * p.sv.h + part * 8
                                : static_cast<const uint16_t*>(p.dout) + b * p.sdo.b + (h0 + h) * p.sdo.h + part * 8;
  const int64_t step = values ? p.sv.s : p.sdo.s;
  uint32_t largest = 0;  // of the magnitudes that this thread has read, as fp32 bits
  for (int i0 = blockIdx.x * 32; i0 < p.sp; i0 += gridDim.x * 32) {
#pragma unroll 4
    for (int t = 0; t < 8; ++t) {
      const int j = t * 4 + (threadIdx.x >> 6), i = i0 + j;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (i < len && h0 + h < heads && part * 8 + k * 64 < p.d) {
          const uint4 y = *reinterpret_cast<const uint4*>(grad + i * step + k * 64);
          uint4 x = make_uint4(0, 0, 0, 0);
          uint2 z = make_uint2(0, 0);
          if (!values) {
            x = *reinterpret_cast<const uint4*>(out + i * p.so.s + k * 64);
            if (p.rest && i < kTile && FewKeys(p, len)) z = *reinterpret_cast<const uint2*>(p.rest + RestAt(p, b, i, h0 + h) + part * 8 + k * 64);
          }
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[4] = {z.x, z.x >> 16, z.y, z.y >> 16};
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float2 a = Unpack2<kBf16>(xs[v]), c = Unpack2<kBf16>(ys[v]), e = UnpackE5m2(zs[v]);
            sum = fmaf(fmaf(e.x, 1 / RestScale<kBf16>(), a.x), c.x, fmaf(fmaf(e.y, 1 / RestScale<kBf16>(), a.y), c.y, sum));
            if (!kBf16) largest = max(largest, max(__float_as_uint(c.x) & 0x7fffffffu, __float_as_uint(c.y) & 0x7fffffffu));
          }
        }
#pragma unroll
      for (int k = 4; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
      if (part == 0) sums[h][j] = sum;
    }
    __syncthreads();
    const int hw = threadIdx.x >> 5, j = threadIdx.x & 31;
    if (!values && h0 + hw < p.h) {  // i0 + j < sp, a multiple of 32
      const int64_t at = (static_cast<int64_t>(b) * p.h + h0 + hw) * p.sp + i0 + j;
      p.delta[at]         = (kBf16 ? 0.f : kHalfP) - p.lse[at];
      p.delta[plane + at] = -sums[hw][j];
    }
    __syncthreads();
  }
  if (!kBf16) {
#pragma unroll
    for (int k = 4; k > 0; k >>= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, k));
    if (part == 0 && h0 + h < heads && largest)  // a maximum does not depend on the order
      atomicMax(reinterpret_cast<uint32_t*>(p.delta + 2 * plane) + (values ? p.b * p.hk : 0) + b * p.hk +
                    (values ? h0 + h : (h0 + h) / (p.h / p.hk)),
                largest);
  }
}

// The k of a key and value head's dS.
__device__ __forceinline__ int GradExponent(const AttnParams& p, int b, int hk) {
  const float* most = p.delta + 2 * static_cast<int64_t>(p.b) * p.h * p.sp + b * p.hk + hk;
  const uint32_t bits = __float_as_uint(2.f * p.d * most[0] * most[p.b * p.hk]);
  if (bits == 0 || bits >= 0x7f800000u) return 0;  // no gradient, or one that is not finite anyway
  const int k = 14 - (static_cast<int>(bits >> 23) - 127);
  return k < -100 ? -100 : k > 100 ? 100 : k;
}

// A piece of work is one tile of 128 keys (kKeys) or queries (!kKeys), which stays; the tiles of the other side (units) stream
// past it:
//             stays (X1, X2)   streams (Y1, Y2)   S = X1 Y1^T, dP = X2 Y2^T       accumulated
//   kKeys     K, V             Q, dO              rows are keys: P^T and dS^T     dV += P^T dO,  dK += dS^T Q
//   !kKeys    Q, dO            K, V               rows are queries                dQ += dS K
// Both passes compute S and dP, seven products instead of five, and in exchange every sum has one owner: no atomics, no
// fp32 copy of dQ in memory, and results that do not depend on the order of the blocks.
// A unit of 64 positions goes through S, P, dP, dS in turn, and every step hands over between the tensor cores and eight softmax
// warps, each of which has 32 rows x 32 columns.  While one unit waits for the tensor cores, another computes:
// with 64 accumulator columns that of the other block on the SM; with 128, where one block fills TMEM, that of a second set of
// warps with its own S and dP.  There two warps issue the products (a wait costs such a warp as much time as an MMA or two, so each
// gets half of them; one for all: 8192, 16 heads that share 4, causal, 1143 us where two take 810), and one clears rows beyond a
// sequence's length; two blocks have no registers for more warps, so the one that issues clears as well.
// D included: 32 x 512, 16 heads of 64: 182 us = 473 TFLOP/s counting five products, with lengths spread over 1..512: 114; 4 x 2048: 269 us =
// 640; 8192 positions, 16 heads of 128 that share 4, causal: 810 us = 847 (906 at 1665 MHz, see above).  (One block per SM with units of 128
// for 64 columns, and the next scores beside them: 183, 126 and 264.)  Bound by the way from one unit to the next: S, exponentials, dP, dS and the
// products' latencies follow one another, with the tensor cores busy a third to a half of the time, the exponentials' unit half.
template <int HD>
struct BwdCfg {
  static constexpr int kTileBytes  = (HD / 64) * kBoxBytes;    // what stays: X1 or X2
  static constexpr int kBlocks     = HD == 64 ? 2 : 1;         // per SM
  static constexpr int kSets       = HD == 64 ? 1 : 2;
  static constexpr int kSetWarps   = 8;
  static constexpr int kSoftWarps  = kSets * kSetWarps;
  static constexpr int kMmaWarps   = HD == 64 ? 1 : 2;
  static constexpr int kTmaWarp    = kSoftWarps, kMmaWarp = kSoftWarps + 1;
  static constexpr bool kClears    = kMmaWarps == 2;            // a warp of its own clears rows beyond a sequence's length
  static constexpr int kClearWarp  = kClears ? kMmaWarp + 2 : -1;
  static constexpr int kThreads    = (kSoftWarps + 1 + kMmaWarps + kClears) * 32;
  static constexpr int kColumns    = kSets * 128 + 2 * HD;     // of TMEM
  static constexpr int kUnit       = 64;                       // positions of a streamed unit
  static constexpr int kUnitBytes  = kUnit * HD * 2;
  static constexpr int kStageBytes = 2 * kUnitBytes;           // Y1, Y2
  static constexpr int kStages     = 4;
  static constexpr int kRowBytes   = 2 * kUnit * 4;            // -L and -D of a unit of queries
  // shared memory: X1, X2, the ring [kStages][Y1, Y2], [kStages][-L, -D], barriers
  static constexpr int kRing       = 2 * kTileBytes;
  static constexpr int kRows       = kRing + kStages * kStageBytes;
  static constexpr int kXRows      = kRows + kStages * kRowBytes;  // -L and -D of the tile of queries that stays
  static constexpr int kNext       = kXRows + 2 * kTile * 4;
  static constexpr int kFull       = kNext + Pieces::kBytes;
  static constexpr int kEmpty      = kFull + 8 * kStages;
  static constexpr int kRaw        = kEmpty + 8 * kStages;       // a unit has arrived and has rows to clear before it counts as full
  static constexpr int kXFull      = kRaw + 8 * kStages;
  static constexpr int kXEmpty     = kXFull + 8;
  static constexpr int kSFull      = kXEmpty + 8;                // [sets] S of a unit is in TMEM
  static constexpr int kSDone      = kSFull + 8 * kSets;         // [sets] keys: P has taken its place, queries: S has been read
  static constexpr int kDpFull     = kSDone + 8 * kSets;         // [sets] dP is in TMEM
  static constexpr int kDsFull     = kDpFull + 8 * kSets;        // [sets] dS has taken its place
  static constexpr int kTurn       = kDsFull + 8 * kSets;        // [sets] a unit's exponentials are done
  static constexpr int kAccFull    = kTurn + 8 * kSets;          // a piece's sums are complete
  static constexpr int kAccFree    = kAccFull + 8;               // all softmax warps have read them, and staged them for the store
  static constexpr int kTmemSlot   = kAccFree + 8;
  static constexpr int kSmemBytes  = kTmemSlot + 16 + 1024;
};

struct BwdWords {  // what stands in a slot
  int b, head, x0, len, first, per, total;
  bool ragged, keys;  // a head's last unit has rows to clear; keys stay
  int exponent;       // of the factor of dS, for fp16
  __device__ __forceinline__ explicit BwdWords(const int (&w)[8])
      : b(w[0]), head(w[1]), x0(w[2]), len(w[3]), first(w[4]), per(w[5]), total(w[6]), ragged(w[7] & 1), keys(w[7] & 2),
        exponent((w[7] >> 8) - 128) {}
  // First the pieces of the keys, whose tiles stream past every query head of their group; causal: the tiles with the longest
  // streams first; otherwise neighbours share a head.
  template <int kUnit, bool kBf16>
  __device__ __forceinline__ static void Describe(const AttnParams& p, int index, int (&w)[8]) {
    const int tiles = p.sp / kTile, group = p.h / p.hk, key_pieces = tiles * p.b * p.hk;
    const bool keys = index < key_pieces;
    if (!keys) index -= key_pieces;
    const int kh = keys ? p.hk : p.h, heads = p.b * kh;
    const int tile = !p.causal ? index % tiles : keys ? index / heads : tiles - 1 - index / heads;
    const int bh = p.causal ? index % heads : index / tiles, b = bh / kh, x0 = tile * kTile;
    const int len = SeqLen(p, b), units = TilesOf(len, kUnit);
    // streamed units: [first, last) of the one head, or of each head of the group
    const int first = keys && p.causal ? x0 / kUnit : 0;
    const int last  = !keys && p.causal ? min(units, (x0 + kTile) / kUnit) : units;
    const int total = x0 >= len ? 0 : (last - first) * (keys ? group : 1);
    w[0] = b;
    w[1] = bh % kh;
    w[2] = x0;
    w[3] = len;
    w[4] = first;
    w[5] = last - first;
    w[6] = total;
    w[7] = (total > 0 && last == units && len < p.s && len % kUnit != 0 ? 1 : 0) | (keys ? 2 : 0);
    if (!kBf16) w[7] |= (GradExponent(p, b, keys ? w[1] : w[1] / group) + 128) << 8;
  }
};
template <bool kKeys>
struct BwdPiece : BwdWords {
  using BwdWords::BwdWords;
};

template <int HD>
struct BwdSmem {
  using C = BwdCfg<HD>;
  uint32_t base, tmem;
  __device__ __forceinline__ uint32_t X() const { return base; }
  __device__ __forceinline__ uint32_t Y(uint32_t u) const { return base + C::kRing + u % C::kStages * C::kStageBytes; }
  __device__ __forceinline__ uint32_t Rows(uint32_t u) const { return base + C::kRows + u % C::kStages * C::kRowBytes; }
  __device__ __forceinline__ uint32_t XRows() const { return base + C::kXRows; }
  __device__ __forceinline__ uint32_t Full(uint32_t u) const { return base + C::kFull + u % C::kStages * 8; }
  __device__ __forceinline__ uint32_t Empty(uint32_t u) const { return base + C::kEmpty + u % C::kStages * 8; }
  __device__ __forceinline__ uint32_t Raw(uint32_t u) const { return base + C::kRaw + u % C::kStages * 8; }
  __device__ __forceinline__ uint32_t XFull() const { return base + C::kXFull; }
  __device__ __forceinline__ uint32_t XEmpty() const { return base + C::kXEmpty; }
  __device__ __forceinline__ uint32_t SFull(uint32_t u) const { return base + C::kSFull + u % C::kSets * 8; }
  __device__ __forceinline__ uint32_t SDone(uint32_t u) const { return base + C::kSDone + u % C::kSets * 8; }
  __device__ __forceinline__ uint32_t DpFull(uint32_t u) const { return base + C::kDpFull + u % C::kSets * 8; }
  __device__ __forceinline__ uint32_t DsFull(uint32_t u) const { return base + C::kDsFull + u % C::kSets * 8; }
  __device__ __forceinline__ uint32_t Turn(uint32_t u) const { return base + C::kTurn + u % C::kSets * 8; }
  // columns: S and dP of either set, then the accumulators
  __device__ __forceinline__ uint32_t S(uint32_t u) const { return tmem + u % C::kSets * 128; }
  __device__ __forceinline__ uint32_t Dp(uint32_t u) const { return S(u) + 64; }
  __device__ __forceinline__ uint32_t Acc(int i) const { return tmem + C::kSets * 128 + i * HD; }
};

// What each kind of warp does for one piece.  u0: units so far, n: pieces with any so far.
template <int HD, bool kKeys>
__device__ __forceinline__ bool BwdLoad(const AttnMaps& maps, const AttnParams& p, const BwdSmem<HD>& m, const BwdPiece<kKeys>& w,
                                        uint32_t u0, uint32_t n) {  // one thread
  using Cfg = BwdCfg<HD>;
  constexpr int ST = Cfg::kStages, kUnit = Cfg::kUnit;
  if (!BarWaitOne(m.XEmpty(), n ^ 1)) return false;
  BarExpect(m.XFull(), 2 * Cfg::kTileBytes + (kKeys ? 0 : 2 * kTile * 4));
  TmaLoadTile<HD, kTile, kUnit>(m.X(), kKeys ? &maps.k : &maps.q, w.x0, w.head, w.b, m.XFull());
  TmaLoadTile<HD, kTile, kUnit>(m.X() + Cfg::kTileBytes, kKeys ? &maps.v : &maps.dout, w.x0, w.head, w.b, m.XFull());
  const int64_t plane = static_cast<int64_t>(p.b) * p.h * p.sp;  // of -L, -D
  if (!kKeys) {
    const float* src = p.delta + (static_cast<int64_t>(w.b) * p.h + w.head) * p.sp + w.x0;
    BulkLoad(m.XRows(), src, kTile * 4, m.XFull());
    BulkLoad(m.XRows() + kTile * 4, src + plane, kTile * 4, m.XFull());
  }
  const int group = p.h / p.hk;
  int at = 0, yh = kKeys ? w.head * group : w.head / group;  // unit within a head
  for (int k = 0; k < w.total; ++k) {
    const uint32_t u = u0 + k;
    if (!BarWaitOne(m.Empty(u), (u / ST) ^ 1)) return false;
    const int y0 = (w.first + at) * kUnit;
    const uint32_t bar = Cfg::kClears && w.ragged && at == w.per - 1 ? m.Raw(u) : m.Full(u);
    BarExpect(bar, Cfg::kStageBytes + (kKeys ? Cfg::kRowBytes : 0));
    TmaLoadTile<HD, kUnit, kUnit>(m.Y(u), kKeys ? &maps.q : &maps.k, y0, yh, w.b, bar);
    TmaLoadTile<HD, kUnit, kUnit>(m.Y(u) + Cfg::kUnitBytes, kKeys ? &maps.dout : &maps.v, y0, yh, w.b, bar);
    if (kKeys) {
      const float* src = p.delta + (static_cast<int64_t>(w.b) * p.h + yh) * p.sp + y0;
      BulkLoad(m.Rows(u), src, kUnit * 4, bar);
      BulkLoad(m.Rows(u) + kUnit * 4, src + plane, kUnit * 4, bar);
    }
    if (++at == w.per) {
      at = 0;
      ++yh;
    }
  }
  return true;
}

// uses: bit st is the parity of the next use of raw[st].
template <int HD, bool kKeys>
__device__ __forceinline__ void BwdClear(const BwdSmem<HD>& m, const BwdPiece<kKeys>& w, uint32_t u0, uint32_t& uses, IdleWaiter& wait) {
  for (int k = w.per - 1; w.ragged && k < w.total; k += w.per) {
    const uint32_t st = (u0 + k) % BwdCfg<HD>::kStages;
    if (!wait(m.Raw(st), uses >> st)) break;
    uses ^= 1u << st;
    ClearRows<BwdCfg<HD>::kUnit>(m.Y(st), 2 * (HD / 64), w.len % BwdCfg<HD>::kUnit);
    if ((threadIdx.x & 31) == 0) BarArrive(m.Full(st));
  }
}

// Stores of a piece whose sums are, or will be, staged in the place of its X.
struct Owed {
  int b = -1, head, x0;
  bool keys;
  uint32_t n;
};
template <int HD>
__device__ __forceinline__ void BwdSettle(const AttnMaps& maps, const BwdSmem<HD>& m, Owed& o, Waiter& wait) {
  using Cfg = BwdCfg<HD>;
  if (o.b < 0 || !wait(m.base + Cfg::kAccFree, o.n)) return;
  if (ElectOne()) {
    TmaStoreTile<HD>(m.X(), o.keys ? &maps.dk : &maps.dq, o.x0, o.head, o.b);
    if (o.keys) TmaStoreTile<HD>(m.X() + Cfg::kTileBytes, &maps.dv, o.x0, o.head, o.b);
    StoresRead();
    BarArrive(m.XEmpty());
  }
  __syncwarp();
  o.b = -1;
}

// Which: 0 issues S and P^T dO, 1 issues dP and dS^T Q or dS K, 2 issues all.
template <bool kBf16, bool kFine, int kWhich, int HD, bool kKeys>
__device__ __forceinline__ void BwdMma(const AttnMaps& maps, const AttnParams& p, const BwdSmem<HD>& m, const BwdPiece<kKeys>& w,
                                       uint32_t u0, uint32_t n, Owed& owed, Waiter& wait) {
  using Cfg = BwdCfg<HD>;
  constexpr int ST = Cfg::kStages, NS = Cfg::kSets, kUnit = Cfg::kUnit;
  const int ksteps = (p.d + 15) >> 4, n_out = ksteps * 16;
  const uint32_t x1 = m.X(), x2 = x1 + Cfg::kTileBytes;
  u0 = Uniform(u0);
  n  = Uniform(n);
  const uint32_t end = u0 + w.total;
  int at = 0;  // the next unit's place within its head
  auto arrived = [&](uint32_t u) {
    if (!wait(m.Full(u), u / ST)) return false;
    if (!Cfg::kClears && ++at == w.per) {
      at = 0;
      if (w.ragged) ClearRows<kUnit>(m.Y(u), 2 * (HD / 64), w.len % kUnit);
    }
    return true;
  };
  auto scores = [&](uint32_t u) {
    IssueScores<kBf16, HD, kUnit>(m.S(u), x1, m.Y(u), ksteps);
    BarCommit(m.SFull(u));
    if (kWhich == 0 && u + 1 == end) BarCommit(m.XEmpty());
  };
  auto grads = [&](uint32_t u) {
    IssueScores<kBf16, HD, kUnit>(m.Dp(u), x2, m.Y(u) + Cfg::kUnitBytes, ksteps);
    BarCommit(m.DpFull(u));
    if (u + 1 == end) BarCommit(m.XEmpty());
  };
  if (kWhich != 1) BwdSettle(maps, m, owed, wait);  // this piece's X comes to the same place
  wait(m.XFull(), n);
  for (uint32_t u = u0; u < min(u0 + NS, end) && arrived(u); ++u)
    if (ElectOne()) {
      if (kWhich != 1) scores(u);
      if (kWhich != 0) grads(u);
    }
  if (kWhich != 1) owed = Owed{w.b, w.head, w.x0, kKeys, n};
  for (uint32_t u = u0; u < end && wait.ok; ++u) {
    const uint32_t next = u + NS;
    if (next < end && !arrived(next)) break;
    if (kWhich != 1) {
      if (!wait(m.SDone(u), u / NS)) break;
      if (ElectOne()) {
        if (kKeys) IssueFromTmem<kBf16, kUnit, 32>(m.Acc(1), m.S(u), m.Y(u) + Cfg::kUnitBytes, n_out, u > u0);
        if (kWhich == 0) BarCommit(m.Empty(u));
        if (next < end) scores(next);  // in the place of P, which the product before it reads
      }
    }
    if (kWhich != 0) {
      if (!wait(m.DsFull(u), u / NS)) break;
      if (kWhich == 1 && u == u0 && n > 0 && !wait(m.base + Cfg::kAccFree, n - 1)) break;
      if (ElectOne()) {
        IssueFromTmem<kBf16, kUnit, 32>(m.Acc(0), m.Dp(u), m.Y(u), n_out, u > u0);
        if (kFine) IssueFromTmem<kBf16, kUnit, 32>(m.Acc(0), m.Dp(u) + 16, m.Y(u), n_out, true);
        BarCommit(m.Empty(u));
        if (next < end) grads(next);
      }
    }
  }
  if (wait.ok && ElectOne()) BarCommit(m.base + Cfg::kAccFull);
}

template <bool kBf16, bool kFine, int HD, bool kKeys>
__device__ __forceinline__ void BwdSoftmax(const AttnParams& p, const BwdSmem<HD>& m, const BwdPiece<kKeys>& w, uint32_t u0, uint32_t n,
                                           Waiter& wait) {
  using Cfg = BwdCfg<HD>;
  constexpr int ST = Cfg::kStages, NS = Cfg::kSets, kUnit = Cfg::kUnit;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3;      // TMEM lanes
  const int set = warp / Cfg::kSetWarps;
  const int col = warp / 4 % 2 * 32;  // first column of this warp in a unit
  const int row = w.x0 + quarter * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
  F2 row_l{}, row_d{};  // -L, -D
  if (w.total > 0) {
    if (!kKeys) {
      wait(m.XFull(), n);
      row_l = Both(LoadShared(m.XRows() + (quarter * 32 + lane) * 4));
      row_d = Both(LoadShared(m.XRows() + (kTile + quarter * 32 + lane) * 4));
    }
  }
  const F2 c2 = Both(p.c), grad2 = Both(kBf16 ? 1.f : TwoTo(w.exponent - kHalfP));
  int at = NS == 1 ? 0 : static_cast<int>((set ^ u0) & 1);  // unit within a head
  for (uint32_t u = u0 + at; u < u0 + w.total; u += NS, at += NS) {
    if (at >= w.per) at %= w.per;  // the group's next head
    const int y0 = (w.first + at) * kUnit;
    if (!wait(m.SFull(u), u / NS)) break;
    uint32_t s[32];
    TmemLoad32Async(m.S(u) + lanes + col, s);
    const bool here = !kKeys || wait(m.Full(u), u / ST);  // -L and -D
    TmemLoadWait(s);
    if (!here) break;
    if (!kKeys) {
      TcFenceBefore();
      __syncwarp();
      if (lane == 0) BarArrive(m.SDone(u));
    }
    // the sets take turns at the exponentials: side by side they would share the unit for them, wait for the tensor cores at
    // the same time, and stay in step
    if (NS > 1 && u > 0 && !wait(m.Turn(u - 1), (u - 1) / NS)) break;
    const uint32_t ls = m.Rows(u) + col * 4;
    F2 pr[16];
#pragma unroll
    for (int k = 0; k < 16; k += 2) {
      F2 l0 = row_l, l1 = row_l;
      if (kKeys) {
        LoadPairs(ls + 8 * k, l0, l1);
      }
      pr[k]     = Exp2Fast(Fma2(Pair(s[2 * k], s[2 * k + 1]), c2, l0));
      pr[k + 1] = Exp2Fast(Fma2(Pair(s[2 * k + 2], s[2 * k + 3]), c2, l1));
    }
    if (NS > 1) {
      __syncwarp();
      if (lane == 0) BarArrive(m.Turn(u));
    }
    if (kKeys ? p.causal && y0 < w.x0 + kTile : y0 + kUnit > w.len || (p.causal && y0 + kUnit > w.x0)) {
      // rows are keys: they count for the queries from their own position on; rows are queries: keys up to a limit
      const int from  = kKeys ? row - y0 - col : 0;
      const int limit = kKeys ? 32 : (p.causal ? min(w.len, row + 1) : w.len) - y0 - col;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float2 x = SplitF2(pr[k]);
        pr[k] = MakeF2(2 * k >= from && 2 * k < limit ? x.x : 0.f, 2 * k + 1 >= from && 2 * k + 1 < limit ? x.y : 0.f);
      }
    }
    if (kKeys) {
      uint32_t v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = Pack2<kBf16>(pr[k]);
      TmemStore16(m.S(u) + lanes + col, v);
      TmemStoreWait();
      TcFenceBefore();
      __syncwarp();
      if (lane == 0) BarArrive(m.SDone(u));
    }
    if (!wait(m.DpFull(u), u / NS)) break;
    TmemLoad32(m.Dp(u) + lanes + col, s);
    uint32_t v[16], low[16];
#pragma unroll
    for (int k = 0; k < 16; k += 2) {
      F2 d0 = row_d, d1 = row_d;
      if (kKeys) {
        LoadPairs(ls + kUnit * 4 + 8 * k, d0, d1);
      }
      F2 g0 = Mul2(pr[k], Add2(Pair(s[2 * k], s[2 * k + 1]), d0)), g1 = Mul2(pr[k + 1], Add2(Pair(s[2 * k + 2], s[2 * k + 3]), d1));
      if (!kBf16) {
        g0 = Mul2(g0, grad2);
        g1 = Mul2(g1, grad2);
      }
      v[k]     = Pack2<kBf16>(g0);
      v[k + 1] = Pack2<kBf16>(g1);
      if (kFine) {
        low[k]     = PackRest<kBf16>(g0, v[k]);
        low[k + 1] = PackRest<kBf16>(g1, v[k + 1]);
      }
    }
    TmemStore16(m.Dp(u) + lanes + col, v);
    if (kFine) TmemStore16(m.Dp(u) + lanes + col + 16, low);
    TmemStoreWait();
    TcFenceBefore();
    __syncwarp();
    if (lane == 0) BarArrive(m.DsFull(u));
  }
  if (w.total > 0) wait(m.base + Cfg::kAccFull, n);
  if (!wait.ok) return;
  const bool live = row < w.len;
  constexpr int kCols = 32;  // of the accumulators, for every warp
  const int c0 = warp / 4 * kCols, r = quarter * 32 + lane;
  if (w.total > 0) {  // dK (dQ) into the place of X1, dV of X2
#pragma unroll
    for (int out = 0; out < (kKeys ? 2 : 1); ++out) {
      uint32_t o[kCols];
      TmemLoad32(m.Acc(out) + lanes + c0, o);
      StageCols<kBf16, kCols>(m.X() + out * Cfg::kTileBytes, r, c0, o,
                              out ? (kBf16 ? 1.f : TwoTo(-kHalfP)) : kBf16 ? p.scale : p.scale * TwoTo(-w.exponent), live);
    }
    TcFenceBefore();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) BarArrive(m.base + Cfg::kAccFree);
  } else {
    const int first = w.x0 + warp * (kTile / Cfg::kSoftWarps);
#pragma unroll
    for (int out = 0; out < (kKeys ? 2 : 1); ++out)
      StoreZeroRows(out ? p.dv : kKeys ? p.dk : p.dq, out ? p.sdv : kKeys ? p.sdk : p.sdq, w.b, w.head, first,
                    min(first + kTile / Cfg::kSoftWarps, p.s), p.d);
  }
}

// Both passes in one launch, so that neither leaves a tail of idle SMs.  kFine: dS as a sum of two values (a branch in the loop
// instead costs long sequences 4 %).
template <int HD, bool kBf16, bool kFine>
__global__ void __launch_bounds__(BwdCfg<HD>::kThreads, BwdCfg<HD>::kBlocks)
AttnBwdKernel(const __grid_constant__ AttnMaps maps, const __grid_constant__ AttnParams p) {
  using Cfg = BwdCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  BwdSmem<HD> m{AlignedSmem(smem_raw), 0};
  const Pieces pieces{m.base + Cfg::kNext};
  const int warp = Uniform(threadIdx.x >> 5);
  if (threadIdx.x == 0) {
    pieces.Init(Cfg::kThreads / 32 - 1);
    for (int i = 0; i < Cfg::kStages; ++i) {
      BarInit(m.Full(i), 1);
      BarInit(m.Empty(i), Cfg::kMmaWarps);
      BarInit(m.Raw(i), 1);
    }
    BarInit(m.XFull(), 1);
    BarInit(m.XEmpty(), Cfg::kMmaWarps + 1);  // the products are done with it, and the sums that took its place are stored
    for (int i = 0; i < Cfg::kSets; ++i) {
      BarInit(m.SFull(i), 1);
      BarInit(m.SDone(i), Cfg::kSetWarps);
      BarInit(m.DpFull(i), 1);
      BarInit(m.DsFull(i), Cfg::kSetWarps);
      BarInit(m.Turn(i), Cfg::kSetWarps);
    }
    BarInit(m.base + Cfg::kAccFull, Cfg::kMmaWarps);
    BarInit(m.base + Cfg::kAccFree, Cfg::kSoftWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == Cfg::kMmaWarp) AllocTmem(m.base + Cfg::kTmemSlot, Cfg::kColumns);
  TcFenceBefore();
  __syncthreads();
  TcFenceAfter();
  m.tmem = Uniform(__float_as_uint(LoadShared(m.base + Cfg::kTmemSlot)));

  uint32_t u0 = 0, n = 0;  // units, and pieces with any, so far
  // what a warp does for a piece
  auto each = [&](const int (&v)[8], auto&& step) {
    const BwdWords w(v);
    bool ok = true;
    if (w.keys) ok = step(BwdPiece<true>(v));
    else ok = step(BwdPiece<false>(v));
    u0 += w.total;
    n += w.total > 0;
    return ok;
  };
  auto follow = [&](auto idle, auto&& step) {
    int v[8];
    for (uint32_t turn = 0; pieces.Take<decltype(idle)::value>(turn, v); ++turn) each(v, step);
  };
  if (warp == Cfg::kTmaWarp) {
    if (ElectOne()) {
      const bool ok = pieces.Lead([&](int index, int (&v)[8]) { BwdWords::Describe<Cfg::kUnit, kBf16>(p, index, v); }, [&](const int (&v)[8]) {
        return each(v, [&](const auto& w) { return w.total == 0 || BwdLoad(maps, p, m, w, u0, n); });
      });
      if (!ok) atomicExch(&g_attn_error, 5);
    }
  } else if (warp == Cfg::kClearWarp) {
    uint32_t uses = 0;
    IdleWaiter wait(6);
    follow(std::true_type{}, [&](const auto& w) {
      BwdClear(m, w, u0, uses, wait);
      return true;
    });
  } else if (warp == Cfg::kMmaWarp) {
    constexpr int kWhich = Cfg::kMmaWarps == 1 ? 2 : 0;
    Waiter wait(6);
    Owed owed;
    follow(std::false_type{}, [&](const auto& w) {
      if (w.total > 0 && wait.ok) BwdMma<kBf16, kFine, kWhich>(maps, p, m, w, u0, n, owed, wait);
      return true;
    });
    if (wait.ok) BwdSettle(maps, m, owed, wait);
    if (ElectOne()) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else if (Cfg::kMmaWarps == 2 && warp == Cfg::kMmaWarp + 1) {
    Waiter wait(6);
    Owed none;
    follow(std::false_type{}, [&](const auto& w) {
      if (w.total > 0 && wait.ok) BwdMma<kBf16, kFine, 1>(maps, p, m, w, u0, n, none, wait);
      return true;
    });
  } else {
    Waiter wait(7);
    follow(std::false_type{}, [&](const auto& w) {
      BwdSoftmax<kBf16, kFine>(p, m, w, u0, n, wait);
      return true;
    });
  }
  TcFenceBefore();
  __syncthreads();
  if (warp == Cfg::kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(m.tmem), "r"(static_cast<uint32_t>(Cfg::kColumns)) : "memory");
}

// ---------------------------------------------------------------- host side

// One head-split tensor [b, s, heads, d] with any strides that are multiples of 16 bytes; boxes of 64 columns x
// box_rows positions.
int HeadMap(CUtensorMap* out, const void* base, int dtype, int b, int s, int heads, int d, const Strides& st, int box_rows) {
  EncodeFn enc = GetEncodeFn();
  if (!enc) return SetError(-7, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[4]    = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(s), static_cast<cuuint64_t>(heads),
                           static_cast<cuuint64_t>(b)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(st.s) * 2, static_cast<cuuint64_t>(st.h) * 2,
                           static_cast<cuuint64_t>(st.b) * 2};
  cuuint32_t box[4]     = {64, static_cast<cuuint32_t>(box_rows), 1, 1};
  cuuint32_t estr[4]    = {1, 1, 1, 1};
  CUresult r = enc(out, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                   const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return SetError(-7, "attention: cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return 0;
}

bool Aligned(const void* base, const Strides& st) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && st.b % 8 == 0 && st.s % 8 == 0 && st.h % 8 == 0;
}
// What a tensor map can express on top: every stride a positive number of bytes below 2^40.
bool Mappable(const Strides& st) {
  for (int64_t v : {st.b, st.s, st.h})
    if (v <= 0 || v >= (int64_t{1} << 39)) return false;
  return true;
}

// Raises a kernel's limit of dynamic shared memory once per device.
template <typename Kernel>
int AllowSmem(Kernel* kernel, int bytes, std::atomic<uint64_t>* done) {
  int dev = 0;
  TIPSK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
  if (bit && (done->load(std::memory_order_acquire) & bit)) return 0;
  TIPSK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done->fetch_or(bit, std::memory_order_release);
  return 0;
}

int CheckSizes(int b, int s, int h, int hk, int d, int dtype, float scale) {
  TIPSK_REQUIRE(dtype == kBF16 || dtype == kF16, "attention: bf16 or fp16");
  TIPSK_REQUIRE(b > 0 && s > 0 && h > 0 && hk > 0 && h % hk == 0, "attention: empty shape, or heads that kv_heads does not divide");
  TIPSK_REQUIRE(d > 0 && d <= 128 && d % 8 == 0, "attention: the head size must be a multiple of 8 up to 128");
  TIPSK_REQUIRE(scale > 0.f && std::isfinite(scale * kLog2e), "attention: scale must be positive and finite");
  // a tile's stream past a group's heads has to end well within the kernels' bounded waits
  TIPSK_REQUIRE(b <= 65535 && h <= (1 << 17) && static_cast<int64_t>(s) * (h / hk) <= (1 << 25) &&
                    static_cast<int64_t>(b) * (h + hk) * TilesOf(s, kTile) < (int64_t{1} << 31),
                "attention: too many rows for one launch");
  return 0;
}

Strides Take(const int64_t* host, int i) { return Strides{host[3 * i], host[3 * i + 1], host[3 * i + 2]}; }

AttnParams MakeParams(const void* lengths, int len64, int b, int s, int h, int hk, int d, float scale, int causal) {
  AttnParams p{};
  p.lengths = lengths;
  p.len64   = len64;
  p.b = b; p.s = s; p.h = h; p.hk = hk; p.d = d;
  p.sp      = TilesOf(s, kTile) * kTile;
  p.causal  = causal ? 1 : 0;
  p.scale   = scale;
  p.c       = scale * kLog2e;
  p.low     = std::max(-1e30f, -1e37f / p.c);
  return p;
}

template <int HD, bool kBf16>
int LaunchFwd(const AttnMaps& maps, const AttnParams& p, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  int rc = AllowSmem(AttnFwdKernel<HD, kBf16>, FwdCfg<HD>::kSmemBytes, &done);
  if (rc) return rc;
  const int grid = TilesOf(p.s, 2 * kTile) * p.b * p.h;
  AttnFwdKernel<HD, kBf16><<<grid, FwdCfg<HD>::kThreads, FwdCfg<HD>::kSmemBytes, s>>>(maps, p);
  TIPSK_LAUNCH_CHECK();
  return 0;
}

template <int HD, bool kBf16, bool kFine>
int LaunchBwd(const AttnMaps& maps, const AttnParams& p, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  int rc = AllowSmem(AttnBwdKernel<HD, kBf16, kFine>, BwdCfg<HD>::kSmemBytes, &done);
  if (rc) return rc;
  int runs = TilesOf(p.h, 8);
  if (!kBf16) {
    runs += TilesOf(p.hk, 8);
    TIPSK_CUDA(cudaMemsetAsync(p.delta + 2 * static_cast<int64_t>(p.b) * p.h * p.sp, 0, static_cast<size_t>(2) * p.b * p.hk * 4, s));
  }
  AttnDeltaKernel<kBf16><<<dim3(std::min(p.sp / 32, 4096), runs, p.b), 256, 0, s>>>(p);
  TIPSK_LAUNCH_CHECK();
  const int grid = (p.sp / kTile) * p.b * (p.h + p.hk);
  AttnBwdKernel<HD, kBf16, kFine><<<grid, BwdCfg<HD>::kThreads, BwdCfg<HD>::kSmemBytes, s>>>(maps, p);
  TIPSK_LAUNCH_CHECK();
  return 0;
}
template <int HD, bool kBf16>
int LaunchBwd(const AttnMaps& maps, const AttnParams& p, cudaStream_t s) {
  return p.s <= kTile ? LaunchBwd<HD, kBf16, true>(maps, p, s) : LaunchBwd<HD, kBf16, false>(maps, p, s);
}

}  // namespace
}  // namespace tipsk

using namespace tipsk;

extern "C" {

/* O = softmax(scale Q K^T + mask) V and L [b, h, s rounded up to 128].  rest (optional): [b, min(s, 128), h, d]
 * bytes, what the rounding of O dropped in rows of few keys, for the backward pass to take.  host_strides: q, k, v, out. */
int tipsk_attention_fwd(const void* q, const void* k, const void* v, void* out, float* lse, void* rest, const void* lengths, int len64,
                        int b, int s, int h, int hk, int d, int dtype, const int64_t* host_strides, float scale, int causal,
                        void* stream) {
  int rc = CheckSizes(b, s, h, hk, d, dtype, scale);
  if (rc) return rc;
  const Strides sq = Take(host_strides, 0), sk = Take(host_strides, 1), sv = Take(host_strides, 2);
  AttnParams p = MakeParams(lengths, len64, b, s, h, hk, d, scale, causal);
  p.so  = Take(host_strides, 3);
  p.o    = out;
  p.lse  = lse;
  p.rest = static_cast<uint8_t*>(rest);
  TIPSK_REQUIRE(Aligned(q, sq) && Aligned(k, sk) && Aligned(v, sv) && Aligned(out, p.so),
                "attention: tensors must be 16-byte aligned with strides of whole 16 bytes");
  TIPSK_REQUIRE(reinterpret_cast<uintptr_t>(rest) % 8 == 0, "attention: rest must be 8-byte aligned");
  TIPSK_REQUIRE(Mappable(sq) && Mappable(sk) && Mappable(sv) && Mappable(p.so), "attention: strides must be positive");
  AttnMaps maps;
  if ((rc = HeadMap(&maps.q, q, dtype, b, s, h, d, sq, kTile))) return rc;
  const int unit = d <= 64 ? FwdCfg<64>::kUnit : FwdCfg<128>::kUnit;
  if ((rc = HeadMap(&maps.k, k, dtype, b, s, hk, d, sk, unit))) return rc;
  if ((rc = HeadMap(&maps.v, v, dtype, b, s, hk, d, sv, unit))) return rc;
  if ((rc = HeadMap(&maps.out, out, dtype, b, s, h, d, p.so, kTile))) return rc;
  maps.dout = maps.dq = maps.dk = maps.dv = maps.q;  // not used
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == kBF16) return d <= 64 ? LaunchFwd<64, true>(maps, p, st) : LaunchFwd<128, true>(maps, p, st);
  return d <= 64 ? LaunchFwd<64, false>(maps, p, st) : LaunchFwd<128, false>(maps, p, st);
}

/* Gradients from dO, the inputs, O, L and (optional) rest of the forward pass.  host_strides: q, k, v, out, dout, dq, dk, dv. */
int tipsk_attention_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse,
                        const void* rest, float* delta, void* dq, void* dk, void* dv, const void* lengths, int len64, int b, int s, int h,
                        int hk, int d, int dtype, const int64_t* host_strides, float scale, int causal, void* stream) {
  int rc = CheckSizes(b, s, h, hk, d, dtype, scale);
  if (rc) return rc;
  const Strides sq = Take(host_strides, 0), sk = Take(host_strides, 1), sv = Take(host_strides, 2);
  AttnParams p = MakeParams(lengths, len64, b, s, h, hk, d, scale, causal);
  p.so    = Take(host_strides, 3);
  p.sdo   = Take(host_strides, 4);
  p.sdq   = Take(host_strides, 5);
  p.sdk   = Take(host_strides, 6);
  p.sdv   = Take(host_strides, 7);
  p.o     = const_cast<void*>(out);
  p.dout  = dout;
  p.lse   = const_cast<float*>(lse);
  p.delta = delta;
  p.rest  = static_cast<uint8_t*>(const_cast<void*>(rest));
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.v  = v;
  p.sv = sv;
  TIPSK_REQUIRE(Aligned(q, sq) && Aligned(k, sk) && Aligned(v, sv) && Aligned(out, p.so) && Aligned(dout, p.sdo) &&
                    Aligned(dq, p.sdq) && Aligned(dk, p.sdk) && Aligned(dv, p.sdv),
                "attention: tensors must be 16-byte aligned with strides of whole 16 bytes");
  TIPSK_REQUIRE(reinterpret_cast<uintptr_t>(lse) % 16 == 0 && reinterpret_cast<uintptr_t>(delta) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(rest) % 8 == 0,
                "attention: lse and delta must be 16-byte aligned, rest 8-byte aligned");
  TIPSK_REQUIRE(Mappable(sq) && Mappable(sk) && Mappable(sv) && Mappable(p.sdo) && Mappable(p.sdq) && Mappable(p.sdk) &&
                    Mappable(p.sdv),
                "attention: strides must be positive");
  const int box = d <= 64 ? BwdCfg<64>::kUnit : BwdCfg<128>::kUnit;
  AttnMaps maps;
  if ((rc = HeadMap(&maps.q, q, dtype, b, s, h, d, sq, box))) return rc;
  if ((rc = HeadMap(&maps.k, k, dtype, b, s, hk, d, sk, box))) return rc;
  if ((rc = HeadMap(&maps.v, v, dtype, b, s, hk, d, sv, box))) return rc;
  if ((rc = HeadMap(&maps.dout, dout, dtype, b, s, h, d, p.sdo, box))) return rc;
  if ((rc = HeadMap(&maps.dq, dq, dtype, b, s, h, d, p.sdq, kTile))) return rc;
  if ((rc = HeadMap(&maps.dk, dk, dtype, b, s, hk, d, p.sdk, kTile))) return rc;
  if ((rc = HeadMap(&maps.dv, dv, dtype, b, s, hk, d, p.sdv, kTile))) return rc;
  maps.out = maps.q;  // not used
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == kBF16) return d <= 64 ? LaunchBwd<64, true>(maps, p, st) : LaunchBwd<128, true>(maps, p, st);
  return d <= 64 ? LaunchBwd<64, false>(maps, p, st) : LaunchBwd<128, false>(maps, p, st);
}

/* Reads and clears the attention error word of the current device (0: ok), once all that was launched on any of its streams is
 * done (a copy by itself waits for the streams that synchronise with the default one only, which PyTorch's do not). */
int tipsk_attention_status(void) {
  int32_t v = 0;
  const int32_t zero = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return -7;
  if (cudaMemcpyFromSymbol(&v, g_attn_error, sizeof(v)) != cudaSuccess) return -7;
  if (v && cudaMemcpyToSymbol(g_attn_error, &zero, sizeof(zero)) != cudaSuccess) return -7;
  return v;
}

}  // extern "C"
