// Activations kept for the backward pass in 8 bits (the form: pack8.cuh).  The GEMM writes it too, from its accumulators.
//
// The reference keeps no activations (it trains TensorFlow models); these serve the linear layers of the encoder.
#include "kernels/common.cuh"
#include "kernels/pack8.cuh"
#include "kernels/tips_kernels.h"

namespace tipsk {
namespace {

__device__ __forceinline__ float Dequantise(int q, float step) { return q == -128 ? __uint_as_float(0x7fc00000u) : q * step; }
// Four stored values.  Without a NaN among them: the byte, with its sign bit flipped, becomes the last bits of 2^23 + q + 128.
__device__ __forceinline__ void Dequantise4(uint32_t w, float step, float* x) {
  const uint32_t u = w ^ 0x80808080u;  // 0 where q is -128
  if (((u - 0x01010101u) & ~u & 0x80808080u) == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 + j)) - 8388736.f) * step;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = Dequantise(static_cast<int8_t>(w >> (8 * j)), step);
  }
}

// A block of 32 values per thread, so nothing is exchanged.  A block whose values are all finite, and not so large that the step is
// clamped, takes a short path of about four instructions a value.  Bound by HBM: 16384 x 4096 bf16, 203 MB in 33 us (6.2 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) Pack8Kernel(const T* __restrict__ x, int8_t* __restrict__ q, int8_t* __restrict__ e, int64_t n) {
  constexpr int N = 16 / sizeof(T);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t g = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; g * kBlock8 < n; g += stride) {
    const int64_t at = g * kBlock8;
    float v[kBlock8];
    const bool whole = at + kBlock8 <= n;
    if (whole) {
#pragma unroll
      for (int k = 0; k < kBlock8; k += N) {
        const Vec16<T> w = LoadVec(x + at + k);
#pragma unroll
        for (int j = 0; j < N; ++j) v[k + j] = ToFloat<T>(w.v[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kBlock8; ++j) v[j] = at + j < n ? ToFloat<T>(x[at + j]) : 0.f;
    }
    // as whole numbers, magnitudes compare like the values, and what is not finite is above all that is
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < kBlock8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
    const bool finite = amax < 0x7f800000u;
    if (!finite) {
      amax = 0;
#pragma unroll
      for (int j = 0; j < kBlock8; ++j) amax = max(amax, FiniteBits(v[j]));
    }
    const int ex    = StepExponent(amax);
    const float inv = PowerOfTwo(-ex);
    uint32_t w[kBlock8 / 4];
    if (finite && ex < 121) {
#pragma unroll
      for (int j = 0; j < kBlock8 / 4; ++j) w[j] = Quantise4(&v[4 * j], inv);
    } else {
#pragma unroll
      for (int j = 0; j < kBlock8 / 4; ++j)
        w[j] = Quantise(v[4 * j], inv) | Quantise(v[4 * j + 1], inv) << 8 | Quantise(v[4 * j + 2], inv) << 16 |
               Quantise(v[4 * j + 3], inv) << 24;
    }
    if (whole) {
      *reinterpret_cast<uint4*>(q + at)      = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(q + at + 16) = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
#pragma unroll
      for (int j = 0; j < kBlock8; ++j)
        if (at + j < n) q[at + j] = static_cast<int8_t>(w[j / 4] >> (8 * (j % 4)));
    }
    e[g] = static_cast<int8_t>(ex);
  }
}

// A stored value in fp16, at most `most` in magnitude (infinity: as it is).  What was fp16 may have been stored as 64 * 2^10, the first
// number beyond fp16's 65504, from which 65504 is no further off than half a step, like what it stands for.
__device__ __forceinline__ __half FromStored(float x, float most, __half) {
  return FromFloat<__half>(x > most ? most : x < -most ? -most : x);  // a NaN stays one
}
template <typename T>
__device__ __forceinline__ T FromStored(float x, float, T) {
  return FromFloat<T>(x);
}

// Eight values per thread and step, four steps in flight.  Bound by HBM: 16384 x 4096 into bf16, 203 MB in 33 us (6.2 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) Unpack8Kernel(const int8_t* __restrict__ q, const int8_t* __restrict__ e, T* __restrict__ y, int64_t n,
                                                     float most) {
  constexpr int N = 16 / sizeof(T), U = 4;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t g = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; g * 8 < n; g += U * stride) {
    uint2 w[U];
    int ex[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (g + u * stride) * 8;
      if (at < n) ex[u] = e[at / kBlock8];
      if (at + 8 <= n) w[u] = *reinterpret_cast<const uint2*>(q + at);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (g + u * stride) * 8;
      if (at + 8 <= n) {
        const float step = PowerOfTwo(ex[u]);
        float v[8];
        Dequantise4(w[u].x, step, v);
        Dequantise4(w[u].y, step, v + 4);
#pragma unroll
        for (int k = 0; k < 8; k += N) {
          Vec16<T> o;
#pragma unroll
          for (int j = 0; j < N; ++j) o.v[j] = FromStored(v[k + j], most, T{});
          StoreVec(y + at + k, o);
        }
      } else {
        for (int j = 0; at + j < n; ++j) y[at + j] = FromStored(Dequantise(q[at + j], PowerOfTwo(ex[u])), most, T{});
      }
    }
  }
}

// dz = dy gelu'(z) with z in 8 bits, and sums of dz per column, in fp32 before dz is rounded; without kGelu only the sums, of
// dy.  Block (32, 8): a thread takes a vector of columns (which lies within a block of the 8-bit form, because both start at
// multiples of 8 values), every block a share of the rows; the shares' sums go to partial [gridDim.y][cols] and are added in
// their order by ColumnSumKernel, so a result does not depend on the order of the blocks.
// With kTable a block first writes down the derivative for every stored value at the sixteen steps 2^-14 .. 2^1 (of values up to
// 0.008 .. 254), and looks it up: the derivative's two exponential-unit instructions and some thirty others per value kept
// the kernel at 76 us for 16384 x 4096 bf16 (335 MB), where HBM needs 51; with the table it takes 68.
// Other steps are computed as without a table.
constexpr int kGradTables = 16, kGradFirst = -14;
template <typename T, bool kGelu, bool kTable>
__global__ void __launch_bounds__(256, 4)
ActBwd8Kernel(const T* __restrict__ dy, const int8_t* __restrict__ q, const int8_t* __restrict__ e, T* __restrict__ dz,
              float* __restrict__ partial, int64_t rows, int cols) {
  constexpr int N = 8, U = sizeof(T) == 4 ? 1 : 2;  // rows in flight
  __shared__ float red[8][32][N + 1];
  __shared__ float table[kTable ? kGradTables * 256 : 1];
  if (kTable) {
    for (int i = threadIdx.y * 32 + threadIdx.x; i < kGradTables * 256; i += 256) {
      const float z = Dequantise(static_cast<int8_t>(i & 255), PowerOfTwo(kGradFirst + (i >> 8)));
      table[i] = SplitF2(GeluGrad2(MakeF2(z, z))).x;
    }
    __syncthreads();
  }
  const int vc = blockIdx.x * 32 + threadIdx.x;
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  if (vc < cols / N) {
    const int64_t step = static_cast<int64_t>(gridDim.y) * 8;
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * 8 + threadIdx.y; r < rows; r += U * step) {
      alignas(16) T g[U][N];
      uint2 w[U];
      int ex[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + u * step < rows) {
          const int64_t off = (r + u * step) * cols + static_cast<int64_t>(vc) * N;
#pragma unroll
          for (int k = 0; k < N; k += 16 / sizeof(T)) *reinterpret_cast<uint4*>(&g[u][k]) = *reinterpret_cast<const uint4*>(dy + off + k);
          if (kGelu) {
            w[u] = *reinterpret_cast<const uint2*>(q + off);
            ex[u] = e[off / kBlock8];
          }
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + u * step >= rows) continue;
        if (!kGelu) {
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += ToFloat<T>(g[u][k]);
          continue;
        }
        float slope[N];
        const int row = ex[u] - kGradFirst;
        if (kTable && static_cast<unsigned>(row) < kGradTables) {
          const float* t = table + row * 256;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            slope[k]     = t[(w[u].x >> (8 * k)) & 255];
            slope[k + 4] = t[(w[u].y >> (8 * k)) & 255];
          }
        } else {
          float z[N];
          Dequantise4(w[u].x, PowerOfTwo(ex[u]), z);
          Dequantise4(w[u].y, PowerOfTwo(ex[u]), z + 4);
#pragma unroll
          for (int k = 0; k < N; k += 2) {
            const float2 v = SplitF2(GeluGrad2(MakeF2(z[k], z[k + 1])));
            slope[k]     = v.x;
            slope[k + 1] = v.y;
          }
        }
        alignas(16) T o[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float v = ToFloat<T>(g[u][k]) * slope[k];
          acc[k] += v;
          o[k] = FromFloat<T>(v);
        }
        const int64_t off = (r + u * step) * cols + static_cast<int64_t>(vc) * N;
#pragma unroll
        for (int k = 0; k < N; k += 16 / sizeof(T)) *reinterpret_cast<uint4*>(dz + off + k) = *reinterpret_cast<uint4*>(&o[k]);
      }
    }
  }
  if (!partial) return;
#pragma unroll
  for (int k = 0; k < N; ++k) red[threadIdx.y][threadIdx.x][k] = acc[k];
  __syncthreads();
  const int t = threadIdx.y * 32 + threadIdx.x, c = blockIdx.x * 256 + t;
  if (c < cols) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += red[j][t / N][t % N];
    partial[static_cast<int64_t>(blockIdx.y) * cols + c] = s;
  }
}

// The shares' sums of 32 columns, in their order: 37 x 4096 floats in 4 us, little more than a launch takes.
template <typename T>
__global__ void __launch_bounds__(256) ColumnSumKernel(const float* __restrict__ partial, T* __restrict__ out, int parts, int cols) {
  const int c = blockIdx.x * 32 + threadIdx.x;
  __shared__ float red[8][33];
  float s = 0.f;
  if (c < cols)
    for (int p = threadIdx.y; p < parts; p += 8) s += partial[static_cast<int64_t>(p) * cols + c];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
#pragma unroll
    for (int j = 1; j < 8; ++j) s += red[j][threadIdx.x];
    out[c] = FromFloat<T>(s);
  }
}

int Blocks(int64_t threads, int per_sm) {
  const int64_t want = (threads + 255) / 256, most = static_cast<int64_t>(NumSMs()) * per_sm;
  return static_cast<int>(want < most ? want : most);
}
bool Aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace tipsk

using namespace tipsk;

extern "C" {

/* q[n], e[ceil(n / 32)] = the 8-bit form of x[n] (fp32, bf16 or fp16). */
int tipsk_pack8(const void* x, void* q, void* e, int64_t n, int dtype, void* stream) {
  TIPSK_REQUIRE(n > 0 && (dtype == kF32 || dtype == kBF16 || dtype == kF16), "pack8: fp32, bf16 or fp16 and at least one value");
  TIPSK_REQUIRE(Aligned16(x) && Aligned16(q), "pack8: the values must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = Blocks((n + 31) / 32, 8);
  int8_t *qq = static_cast<int8_t*>(q), *ee = static_cast<int8_t*>(e);
  if (dtype == kF32) Pack8Kernel<float><<<grid, 256, 0, s>>>(static_cast<const float*>(x), qq, ee, n);
  else if (dtype == kBF16) Pack8Kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(x), qq, ee, n);
  else Pack8Kernel<__half><<<grid, 256, 0, s>>>(static_cast<const __half*>(x), qq, ee, n);
  TIPSK_LAUNCH_CHECK();
  return 0;
}

/* y[n] = the values that q, e stand for; exact in fp32 and bf16, rounded to fp16 where that has fewer bits (below 2^-14).  Values
 * beyond fp16's range become infinite, or with `from_half`, which says that fp16 was packed, the nearest that it has. */
int tipsk_unpack8(const void* q, const void* e, void* y, int64_t n, int dtype, int from_half, void* stream) {
  TIPSK_REQUIRE(n > 0 && (dtype == kF32 || dtype == kBF16 || dtype == kF16), "unpack8: fp32, bf16 or fp16 and at least one value");
  TIPSK_REQUIRE(Aligned16(y) && Aligned16(q), "unpack8: the values must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = Blocks((n + 7) / 8, 8);
  const int8_t *qq = static_cast<const int8_t*>(q), *ee = static_cast<const int8_t*>(e);
  const float most = from_half ? 65504.f : INFINITY;
  if (dtype == kF32) Unpack8Kernel<float><<<grid, 256, 0, s>>>(qq, ee, static_cast<float*>(y), n, most);
  else if (dtype == kBF16) Unpack8Kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(qq, ee, static_cast<__nv_bfloat16*>(y), n, most);
  else Unpack8Kernel<__half><<<grid, 256, 0, s>>>(qq, ee, static_cast<__half*>(y), n, most);
  TIPSK_LAUNCH_CHECK();
  return 0;
}

/* Shares of the rows of tipsk_act_bwd8, for its workspace. */
int tipsk_act_bwd8_parts(int64_t rows, int cols) {
  const int64_t tiles = (cols + 255) / 256, fill = (static_cast<int64_t>(NumSMs()) * 4 + tiles - 1) / tiles;
  const int64_t most  = (rows + 7) / 8;
  return static_cast<int>(fill < most ? fill : most);
}

/* dz = dy * gelu'(z) for z [rows, cols] in 8 bits (q, e); without q, e and dz there is no activation.  dbias (optional with z,
 * of dtype bias_dtype) receives the column sums of dz, or of dy.  partial: fp32 workspace of tipsk_act_bwd8_parts * cols.
 * cols a multiple of 8. */
int tipsk_act_bwd8(const void* dy, const void* q, const void* e, void* dz, void* dbias, int bias_dtype, float* partial,
                   int64_t rows, int cols, int dtype, void* stream) {
  TIPSK_REQUIRE(rows > 0 && cols > 0 && cols % 8 == 0, "act_bwd8: the number of columns must be a multiple of 8");
  TIPSK_REQUIRE((dtype == kF32 || dtype == kBF16 || dtype == kF16) &&
                    (dbias == nullptr || bias_dtype == kF32 || bias_dtype == kBF16 || bias_dtype == kF16),
                "act_bwd8: fp32, bf16 or fp16");
  TIPSK_REQUIRE((q == nullptr) == (e == nullptr) && (q == nullptr) == (dz == nullptr), "act_bwd8: q, e and dz go together");
  TIPSK_REQUIRE(Aligned16(dy) && Aligned16(dz) && reinterpret_cast<uintptr_t>(q) % 8 == 0, "act_bwd8: alignment");
  TIPSK_REQUIRE(dbias == nullptr ? q != nullptr : partial != nullptr, "act_bwd8: nothing to do, or no workspace for the sums");
  cudaStream_t s  = static_cast<cudaStream_t>(stream);
  const int parts = tipsk_act_bwd8_parts(rows, cols);
  const dim3 grid((cols + 255) / 256, parts), block(32, 8);
  const int8_t *qq = static_cast<const int8_t*>(q), *ee = static_cast<const int8_t*>(e);
  float* part = dbias ? partial : nullptr;
  auto run = [&](auto t) {
    using T = decltype(t);
    // a table costs a thread 16 derivatives, which pays from about 64 values per thread on
    auto* kernel = !q ? ActBwd8Kernel<T, false, false>
                      : rows >= static_cast<int64_t>(parts) * 8 * 8 ? ActBwd8Kernel<T, true, true> : ActBwd8Kernel<T, true, false>;
    kernel<<<grid, block, 0, s>>>(static_cast<const T*>(dy), qq, ee, static_cast<T*>(dz), part, rows, cols);
  };
  if (dtype == kF32) run(float{});
  else if (dtype == kBF16) run(__nv_bfloat16{});
  else run(__half{});
  TIPSK_LAUNCH_CHECK();
  if (dbias) {
    auto sum = [&](auto t) {
      using T = decltype(t);
      ColumnSumKernel<T><<<(cols + 31) / 32, block, 0, s>>>(partial, static_cast<T*>(dbias), parts, cols);
    };
    if (bias_dtype == kF32) sum(float{});
    else if (bias_dtype == kBF16) sum(__nv_bfloat16{});
    else sum(__half{});
    TIPSK_LAUNCH_CHECK();
  }
  return 0;
}

}  // extern "C"
