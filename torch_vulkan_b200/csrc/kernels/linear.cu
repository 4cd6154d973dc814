// tvb_linear and tvb_linear_backward: argument checks and the choice of kernels.
#include "../core/common.h"
#include "launch.h"
#include "linear.h"

namespace tvb {
namespace {

bool is_float(int dt) { return dt == TVB_F32 || dt == TVB_F16 || dt == TVB_BF16; }

int check_linear(const std::string& fn, int dtype, int activation, int64_t m, int64_t n, int64_t k) {
  TVB_REQUIRE(is_float(dtype), fn + ": float32, float16 or bfloat16 only");
  TVB_REQUIRE(activation >= TVB_ACT_NONE && activation <= TVB_ACT_SILU, fn + ": unknown activation");
  TVB_REQUIRE(m >= 0 && n >= 0 && k >= 0, fn + ": negative size");
  // (the last tile's far end must fit 32 bits too)
  constexpr int64_t kMost = (int64_t(1) << 31) - 1024;
  TVB_REQUIRE(m <= kMost && n <= kMost && k <= kMost, fn + ": a size beyond 2^31 - 1024");
  return 0;
}

// Bytes from the first element of a matrix to behind its last.
int64_t span(int64_t rows, int64_t cols, int64_t ld, int64_t es) { return rows == 0 || cols == 0 ? 0 : ((rows - 1) * ld + cols) * es; }

int64_t round8(int64_t n) { return (n + 7) & ~int64_t(7); }

// Whether TMA can read a 16-bit matrix where it is: it begins on 16 bytes, and so does every row.
bool readable(const void* p, int64_t rows, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (rows <= 1 || ld % 8 == 0); }

// Bytes of the copy that an unreadable 16-bit operand takes in the workspace, each begun on 256 bytes.
uint64_t copy_bytes(int dtype, const void* p, int64_t rows, int64_t cols, int64_t ld) {
  if (dtype == TVB_F32 || rows <= 0 || cols <= 0 || readable(p, rows, ld)) return 0;
  return (static_cast<uint64_t>(rows) * static_cast<uint64_t>(round8(cols)) * 2 + 255) & ~uint64_t(255);
}

// One operand where TMA can read it: in place, or to be copied to the workspace at *at (which moves on).
LinearCopy make_readable(int dtype, const void** p, int64_t rows, int64_t cols, int64_t* ld, uint8_t** at) {
  LinearCopy c{};
  c.dst_ld = 8;
  const uint64_t bytes = copy_bytes(dtype, *p, rows, cols, *ld);
  if (bytes != 0) {
    c = LinearCopy{*at, *p, round8(cols), *ld, rows, cols};
    *p = *at;
    *ld = round8(cols);
    *at += bytes;
  } else if (rows <= 1) {
    *ld = round8(cols);  // (one row: the distance to the next is never used, but has to be a legal one)
  }
  return c;
}

int run_product(int device, cudaStream_t stream, const LinearProduct& p) {
  if (p.dtype == TVB_F32) return linear_simt(device, stream, p);
  return linear_large(p) ? linear_pair(device, stream, &p, 1) : linear_split(device, stream, &p, 1);
}

// dz needs a matrix of its own: there is an activation to differentiate, or TMA cannot read dy.
uint64_t dz_bytes(int dtype, const void* dy, int64_t dy_sm, int activation, int want, int64_t m, int64_t n) {
  if (m <= 0 || n <= 0 || (want & (TVB_WANT_DX | TVB_WANT_DW)) == 0) return 0;
  if (activation == TVB_ACT_NONE && (dtype == TVB_F32 || readable(dy, m, dy_sm))) return 0;
  return (static_cast<uint64_t>(m) * static_cast<uint64_t>(round8(n)) * dtype_size(dtype) + 255) & ~uint64_t(255);
}

}  // namespace
}  // namespace tvb

using namespace tvb;

extern "C" uint64_t tvb_linear_workspace_bytes(int dtype, const void* x, int64_t x_sm, const void* w, int64_t w_sn, int64_t m, int64_t n,
                                               int64_t k) {
  return copy_bytes(dtype, x, m, k, x_sm) + copy_bytes(dtype, w, n, k, w_sn);
}

extern "C" int tvb_linear(int device, const void* x, int dtype, int64_t x_sm, const void* w, int64_t w_sn, const void* bias,
                          int activation, const void* residual, int64_t residual_sm, void* y, void* preact, int64_t m, int64_t n,
                          int64_t k, void* workspace, uint64_t workspace_bytes, void* caller_stream) {
  if (check_linear("tvb_linear", dtype, activation, m, n, k) != 0) return -1;
  TVB_REQUIRE((m <= 1 || x_sm >= k) && (n <= 1 || w_sn >= k), "tvb_linear: rows of x and w must be at least k apart");
  TVB_REQUIRE(residual == nullptr || m <= 1 || residual_sm >= n, "tvb_linear: rows of the residual must be at least n apart");
  if (m == 0 || n == 0) return 0;
  TVB_REQUIRE(y != nullptr && (k == 0 || (x != nullptr && w != nullptr)), "tvb_linear: NULL pointer");
  if (m <= 1) x_sm = k, residual_sm = n;
  if (n <= 1) w_sn = k;
  const int64_t es = dtype_size(dtype), y_bytes = m * n * es;
  const uint64_t need = tvb_linear_workspace_bytes(dtype, x, x_sm, w, w_sn, m, n, k);
  TVB_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0),
              "tvb_linear: the workspace is too small or not 256-byte aligned");
  const void* outs[3] = {y, preact, need != 0 ? workspace : nullptr};
  const int64_t out_bytes[3] = {y_bytes, y_bytes, static_cast<int64_t>(need)};
  for (int i = 0; i < 3; i++) {
    const bool in_place = i == 0 && residual == y && residual_sm == n;  // every element is read before it is written, by the same thread or the same warp
    TVB_REQUIRE(!overlap(outs[i], out_bytes[i], x, span(m, k, x_sm, es)) && !overlap(outs[i], out_bytes[i], w, span(n, k, w_sn, es)) &&
                    !overlap(outs[i], out_bytes[i], bias, n * es) &&
                    (in_place || !overlap(outs[i], out_bytes[i], residual, span(m, n, residual_sm, es))),
                "tvb_linear: an output or the workspace overlaps an operand (only y may be the residual itself)");
    for (int j = 0; j < i; j++) TVB_REQUIRE(!overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]), "tvb_linear: two outputs overlap");
  }
  cudaStream_t stream;
  if (enter_on(device, caller_stream, &stream) != 0) return -1;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  const LinearCopy cx = make_readable(dtype, &x, m, k, &x_sm, &at), cw = make_readable(dtype, &w, n, k, &w_sn, &at);
  if (linear_copy(device, stream, cx, cw) != 0) return -1;
  LinearProduct p{};
  p.p = w; p.p_si = w_sn; p.p_sr = 1;
  p.q = x; p.q_sj = x_sm; p.q_sr = 1;
  p.bias = bias; p.residual = residual; p.residual_ld = residual_sm;
  p.out = y; p.preact = preact;
  p.I = n; p.J = m; p.R = k;
  p.dtype = dtype; p.activation = activation;
  return run_product(device, stream, p);
}

extern "C" uint64_t tvb_linear_backward_workspace_bytes(int dtype, const void* dy, int64_t dy_sm, const void* x, int64_t x_sm, const void* w,
                                                        int64_t w_sn, int activation, int want, int64_t m, int64_t n, int64_t k) {
  return dz_bytes(dtype, dy, dy_sm, activation, want, m, n) + ((want & TVB_WANT_DW) != 0 ? copy_bytes(dtype, x, m, k, x_sm) : 0) +
         ((want & TVB_WANT_DX) != 0 ? copy_bytes(dtype, w, n, k, w_sn) : 0);
}

extern "C" int tvb_linear_backward(int device, const void* dy, int dtype, int64_t dy_sm, const void* preact, const void* x, int64_t x_sm,
                                   const void* w, int64_t w_sn, int activation, void* dx, void* dw, void* db, int64_t m, int64_t n,
                                   int64_t k, void* workspace, uint64_t workspace_bytes, void* caller_stream) {
  if (check_linear("tvb_linear_backward", dtype, activation, m, n, k) != 0) return -1;
  TVB_REQUIRE((m <= 1 || (x_sm >= k && dy_sm >= n)) && (n <= 1 || w_sn >= k),
              "tvb_linear_backward: rows of x and w must be at least k apart, those of dy at least n");
  TVB_REQUIRE(activation == TVB_ACT_NONE || m == 0 || n == 0 || preact != nullptr,
              "tvb_linear_backward: an activation's gradient needs the values before it");
  if (m <= 1) x_sm = k, dy_sm = n;
  if (n <= 1) w_sn = k;
  const bool want_dx = dx != nullptr && m > 0 && k > 0, want_dw = dw != nullptr && n > 0 && k > 0, want_db = db != nullptr && n > 0;
  if (!want_dx && !want_dw && !want_db) return 0;
  TVB_REQUIRE((m == 0 || n == 0 || dy != nullptr) && (!want_dw || m == 0 || x != nullptr) && (!want_dx || n == 0 || w != nullptr),
              "tvb_linear_backward: NULL pointer");
  const int64_t es = dtype_size(dtype);
  const int want = (want_dx ? TVB_WANT_DX : 0) | (want_dw ? TVB_WANT_DW : 0) | (want_db ? TVB_WANT_DB : 0);
  const uint64_t need = tvb_linear_backward_workspace_bytes(dtype, dy, dy_sm, x, x_sm, w, w_sn, activation, want, m, n, k);
  TVB_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0),
              "tvb_linear_backward: the workspace is too small or not 256-byte aligned");
  const void* outs[4] = {want_dx ? dx : nullptr, want_dw ? dw : nullptr, want_db ? db : nullptr, need != 0 ? workspace : nullptr};
  const int64_t out_bytes[4] = {m * k * es, n * k * es, n * es, static_cast<int64_t>(need)};
  for (int i = 0; i < 4; i++) {
    TVB_REQUIRE(!overlap(outs[i], out_bytes[i], dy, span(m, n, dy_sm, es)) && !overlap(outs[i], out_bytes[i], preact, m * n * es) &&
                    !overlap(outs[i], out_bytes[i], x, span(m, k, x_sm, es)) && !overlap(outs[i], out_bytes[i], w, span(n, k, w_sn, es)),
                "tvb_linear_backward: an output or the workspace overlaps an operand");
    for (int j = 0; j < i; j++)
      TVB_REQUIRE(!overlap(outs[i], out_bytes[i], outs[j], out_bytes[j]), "tvb_linear_backward: two outputs overlap");
  }
  cudaStream_t stream;
  if (enter_on(device, caller_stream, &stream) != 0) return -1;
  const void* dz = dy;
  int64_t dz_ld = m > 1 ? dy_sm : round8(n);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  const uint64_t own_dz = dz_bytes(dtype, dy, dy_sm, activation, want, m, n);
  if (own_dz != 0) {
    dz = at;
    dz_ld = round8(n);
    at += own_dz;
  }
  if (own_dz != 0 || want_db) {
    LinearDz d{};
    d.dy = dy; d.z = preact; d.dz = own_dz != 0 ? workspace : nullptr; d.db = want_db ? db : nullptr;
    d.dy_ld = dy_sm; d.dz_ld = dz_ld; d.m = m; d.n = n;
    d.dtype = dtype; d.activation = activation;
    if (linear_dz(device, stream, d) != 0) return -1;
  }
  LinearCopy cx{}, cw{};
  if (want_dw) cx = make_readable(dtype, &x, m, k, &x_sm, &at);
  if (want_dx) cw = make_readable(dtype, &w, n, k, &w_sn, &at);
  if (linear_copy(device, stream, cx, cw) != 0) return -1;
  LinearProduct p[2] = {};
  int count = 0;
  if (want_dx) {
    LinearProduct& d = p[count++];
    d.p = w; d.p_si = 1; d.p_sr = w_sn; d.p_mn = true;
    d.q = dz; d.q_sj = dz_ld; d.q_sr = 1;
    d.out = dx;
    d.I = k; d.J = m; d.R = n;
    d.dtype = dtype;
  }
  if (want_dw) {
    LinearProduct& d = p[count++];
    d.p = x; d.p_si = 1; d.p_sr = x_sm; d.p_mn = true;
    d.q = dz; d.q_sj = 1; d.q_sr = dz_ld; d.q_mn = true;
    d.out = dw;
    d.I = k; d.J = n; d.R = m;
    d.dtype = dtype;
  }
  if (count == 2 && dtype != TVB_F32) {  // in one launch, where the same kernel suits both
    const bool large0 = linear_large(p[0]), large1 = linear_large(p[1]);
    if (large0 && large1) return linear_pair(device, stream, p, 2);
    if (!large0 && !large1) return linear_split(device, stream, p, 2);
  }
  for (int i = 0; i < count; i++)
    if (run_product(device, stream, p[i]) != 0) return -1;
  return 0;
}
