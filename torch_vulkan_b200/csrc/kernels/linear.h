// The products behind tvb_linear and tvb_linear_backward, as one form:
//   out[j, i] = act(sum_r P(i, r) Q(j, r) + bias[i]) + residual[j, i]        i < I, j < J, r < R
// with P(i, r) at p[i * p_si + r * p_sr] and Q(j, r) at q[j * q_sj + r * q_sr], one of the two strides of each being 1 (p_mn, q_mn: which).
//   forward  y = act(x w^T + b) + res   P = w  (i: output feature, r: input feature)  Q = x   (j: row)
//   dx = dz w                           P = w^T (i: input feature, r: output feature) Q = dz  (j: row)
//   dw = dz^T x                         P = x^T (i: input feature, r: row)            Q = dz^T (j: output feature)
// `out` is row-major and contiguous in i whatever the operands' order.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace tvb {

struct LinearProduct {
  const void* p;
  const void* q;
  int64_t p_si, p_sr, q_sj, q_sr;
  bool p_mn, q_mn;       // the operand is contiguous in i / j (else in r)
  const void* bias;      // I values, or NULL
  const void* residual;  // [J, I], row stride residual_ld, or NULL
  void* out;             // [J, I] contiguous
  void* preact;          // [J, I] contiguous: the sums (with the bias) before the activation, or NULL
  int64_t residual_ld;
  int64_t I, J, R;
  int dtype;             // of every operand and output
  int activation;        // TvbActivation
};

int linear_simt(int device, cudaStream_t stream, const LinearProduct& p);  // float32
// float16 and bfloat16, on the tensor cores; every operand begins on 16 bytes and its rows are a multiple of 16 bytes apart.
// `count`: one product, or two that share nothing but their launch.
int linear_split(int device, cudaStream_t stream, const LinearProduct* p, int count);  // two: dx and dw, in this order
bool linear_large(const LinearProduct& p);  // whether linear_pair is the faster of the two
int linear_pair(int device, cudaStream_t stream, const LinearProduct* p, int count);  // R > 0

// Copies 16-bit [rows, cols] matrices to rows dst_ld (a multiple of 8) apart: one or two (rows == 0: none) in one launch.
struct LinearCopy {
  void* dst;
  const void* src;
  int64_t dst_ld, src_ld, rows, cols;
};
int linear_copy(int device, cudaStream_t stream, const LinearCopy& a, const LinearCopy& b);

// dz = dy * act'(z) (row stride dz_ld) and db = its sums over the rows; dz or db may be NULL. activation TVB_ACT_NONE: dz = dy.
struct LinearDz {
  const void* dy;
  const void* z;  // contiguous [m, n]; unused without an activation
  void* dz;
  void* db;
  int64_t dy_ld, dz_ld, m, n;
  int dtype, activation;
};
int linear_dz(int device, cudaStream_t stream, const LinearDz& p);

}  // namespace tvb
