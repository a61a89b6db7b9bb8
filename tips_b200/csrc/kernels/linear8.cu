// A linear layer that keeps its activations in 8 bits: its forward and its backward pass as one call each, on the kernels of
// gemm_tcgen05.cu and saved8.cu.  A small layer waits for the host, not for the GPU, and most of what the
// host does is done per call: 128 rows of 128 into 512, forward and backward, took 197 us with a call per kernel and takes 143.
// A large one is bound by its three products.  16384 rows of 1024 into 4096 with GELU, pass after pass: 476 us at the 1620 MHz that
// the power limit leaves; with events between the kernels 488: first product with GELU and the 8-bit form 155, dx 112, dw 112, GELU's
// derivative and the bias gradient 77, packing and unpacking x 17 + 15.  A few passes at 1965 MHz: 427, 133 + 96 + 96 + 73 + 16 + 15.
#include <algorithm>

#include "kernels/common.cuh"
#include "kernels/pack8.cuh"
#include "kernels/tips_kernels.h"

namespace tipsk {
namespace {

int64_t Round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t ExponentsAt(int64_t n) { return (n + 15) / 16 * 16; }  // in a buffer of n packed values

// Hands out 256-byte-aligned pieces of the workspace, or only counts them.
struct Workspace {
  char* at;
  int64_t used = 0;
  void* Take(int64_t bytes) {
    void* p = at ? at + used : nullptr;
    used += Round256(bytes);
    return p;
  }
};

int64_t PartialBytes(int m, int n, int k) {
  const int splits = tipsk_gemm_splits(m, n, k);
  return splits > 1 ? static_cast<int64_t>(splits) * m * n * 4 : 0;
}

struct Forward {
  void *pre, *partial;
  int64_t bytes;
  Forward(void* ws, int m, int n, int k, bool want_pre) {
    Workspace w{static_cast<char*>(ws)};
    pre     = want_pre && !tipsk_gemm_pre8_fits(m, n, k) ? w.Take(static_cast<int64_t>(m) * n * 2) : nullptr;
    partial = w.Take(PartialBytes(m, n, k));
    bytes   = w.used;
  }
};

struct Backward {
  void *dz, *sums, *x, *partial;
  int64_t bytes;
  Backward(void* ws, int m, int n, int k, bool gelu, bool want_dw, bool want_db) {
    Workspace w{static_cast<char*>(ws)};
    dz   = gelu ? w.Take(static_cast<int64_t>(m) * n * 2) : nullptr;
    sums = want_db ? w.Take(static_cast<int64_t>(tipsk_act_bwd8_parts(m, n)) * n * 4) : nullptr;
    x    = want_dw ? w.Take(static_cast<int64_t>(m) * k * 2) : nullptr;
    partial = w.Take(std::max(PartialBytes(m, k, n), want_dw ? PartialBytes(n, k, m) : 0));
    bytes   = w.used;
  }
};

}  // namespace
}  // namespace tipsk

using namespace tipsk;

extern "C" {

/* Bytes of workspace of the two calls below. */
int64_t tipsk_linear8_fwd_ws(int m, int n, int k, int want_pre) { return Forward(nullptr, m, n, k, want_pre != 0).bytes; }
int64_t tipsk_linear8_bwd_ws(int m, int n, int k, int gelu, int want_dw, int want_db) {
  return Backward(nullptr, m, n, k, gelu != 0, want_dw != 0, want_db != 0).bytes;
}

/* y[m,n] = act(x[m,k] w[n,k]^T + bias), bf16 (act 0 or 2: GELU).  x8 (optional): x in 8 bits; pre8 (optional): the value before the
 * activation in 8 bits, from its rounding to bf16; both are the values and, from the next multiple of 16 bytes on, the
 * exponents.  x is contiguous, w has rows of ldw elements. */
int tipsk_linear8_fwd(const void* x, const void* w, const void* bias, void* y, void* x8, void* pre8, void* ws, int m, int n, int k,
                      int ldw, int act, void* stream) {
  TIPSK_REQUIRE(m > 0 && n > 0 && k > 0 && n % 8 == 0 && k % 8 == 0 && ldw % 8 == 0 && (act == 0 || act == 2),
                "linear8: sizes must be multiples of 8, the activation none or GELU");
  TIPSK_REQUIRE(reinterpret_cast<uintptr_t>(y) % 16 == 0 && reinterpret_cast<uintptr_t>(ws) % 16 == 0, "linear8: alignment");
  const Forward f(ws, m, n, k, pre8 != nullptr);
  TIPSK_REQUIRE(f.bytes == 0 || ws != nullptr, "linear8: no workspace");
  const int64_t mn = static_cast<int64_t>(m) * n, mk = static_cast<int64_t>(m) * k;
  const int splits = tipsk_gemm_splits(m, n, k);
  int rc;
  if (pre8 && f.pre == nullptr) {
    rc = tipsk_gemm_bf16_pre8(x, w, y, bias, pre8, static_cast<char*>(pre8) + ExponentsAt(mn), m, n, k, k, ldw, act, stream);
  } else if (splits > 1) {
    rc = tipsk_gemm_bf16_split(0, x, w, y, bias, f.pre, static_cast<float*>(f.partial), splits, m, n, k, k, ldw, n, act, 0, stream);
  } else {
    rc = tipsk_gemm_bf16(x, w, y, bias, f.pre, m, n, k, k, ldw, n, act, stream);
  }
  if (rc == 0 && f.pre) rc = tipsk_pack8(f.pre, pre8, static_cast<char*>(pre8) + ExponentsAt(mn), mn, kBF16, stream);
  if (rc == 0 && x8) rc = tipsk_pack8(x, x8, static_cast<char*>(x8) + ExponentsAt(mk), mk, kBF16, stream);
  return rc;
}

/* The gradients: dz = dy gelu'(pre8), or dy without pre8; dx[m,k] = dz w, added to what dx holds with `accumulate`;
 * dw[n,k] = dz^T x8; db = column sums of dz, of dtype db_dtype.  dx, dw and db are optional.  n and k at least 64.
 * The weight gradient runs on the CTA-pair GEMM whatever its shape: the convolution's kernel, which spreads long sums over more
 * SMs, adds them in no fixed order. */
int tipsk_linear8_bwd(const void* dy, const void* w, const void* x8, const void* pre8, void* dx, void* dw, void* db, int db_dtype,
                      void* ws, int m, int n, int k, int ldw, int accumulate, void* stream) {
  TIPSK_REQUIRE(m > 0 && n >= 64 && k >= 64 && n % 8 == 0 && k % 8 == 0 && ldw % 8 == 0, "linear8: unsupported shape");
  TIPSK_REQUIRE(dw == nullptr || x8 != nullptr, "linear8: the weight gradient needs the stored input");
  TIPSK_REQUIRE(reinterpret_cast<uintptr_t>(dy) % 16 == 0 && reinterpret_cast<uintptr_t>(dx) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(dw) % 16 == 0 && reinterpret_cast<uintptr_t>(ws) % 16 == 0,
                "linear8: alignment");
  const Backward f(ws, m, n, k, pre8 != nullptr, dw != nullptr, db != nullptr);
  TIPSK_REQUIRE(f.bytes == 0 || ws != nullptr, "linear8: no workspace");
  float* partial  = static_cast<float*>(f.partial);
  const void* dz  = pre8 ? f.dz : dy;
  int rc = 0;
  if (pre8 || db)
    rc = tipsk_act_bwd8(dy, pre8, pre8 ? static_cast<const char*>(pre8) + ExponentsAt(static_cast<int64_t>(m) * n) : nullptr, f.dz, db,
                        db_dtype, static_cast<float*>(f.sums), m, n, kBF16, stream);
  if (rc == 0 && dx) {
    const int splits = tipsk_gemm_splits(m, k, n);
    rc = splits > 1 ? tipsk_gemm_bf16_split(1, dz, w, dx, nullptr, nullptr, partial, splits, m, k, n, n, ldw, k, 0, accumulate, stream)
                    : tipsk_gemm_bf16_nn(dz, w, dx, m, k, n, n, ldw, k, accumulate, stream);
  }
  if (rc == 0 && dw) {
    const int64_t mk = static_cast<int64_t>(m) * k;
    rc = tipsk_unpack8(x8, static_cast<const char*>(x8) + ExponentsAt(mk), f.x, mk, kBF16, 0, stream);
    const int splits = tipsk_gemm_splits(n, k, m);
    if (rc == 0) {
      rc = splits > 1 ? tipsk_gemm_bf16_split(2, dz, f.x, dw, nullptr, nullptr, partial, splits, n, k, m, n, k, k, 0, 0, stream)
                      : tipsk_gemm_bf16_tt(dz, f.x, dw, n, k, m, n, k, k, stream);
    }
  }
  return rc;
}

}  // extern "C"
