// Declarations of the 8-bit layer operators: the product of 8-bit integers
// with scales (i8_plan.cpp, contract_i8*.hip) and the operators that round
// rows to 8 bits (quant_rows.hip).
#ifndef ETIR_I8_INTERNAL_H
#define ETIR_I8_INTERNAL_H

#include "etir_internal.h"

namespace etir {

// ---------------------------------------------------------------------------
// product of 8-bit integers
//   out[c,m,n] = last( sa[c,m] sb[c,n] sum_k A[c,m,k] B[c,n,k] + bias )
// m: the rows, n: the columns of the kernels; the output's unit-stride loop is
// a column loop where it is not a batch loop (A and B change places for that)
// ---------------------------------------------------------------------------
constexpr int kI8MaxLoops = 6;       // fused loops of one type

// The tensors of a product.  All offsets are elements; 8-bit elements are bytes.
enum I8Tensor : int32_t { I8_A = 0, I8_B = 1, I8_OUT = 2, I8_SA = 3, I8_SB = 4, I8_BIAS = 5, I8_TENSORS = 6 };

// The fused loops of one type, outermost first.
struct I8Loops {
  int32_t n = 0;
  int32_t size[kI8MaxLoops] = {};
  int64_t stride[kI8MaxLoops][I8_TENSORS] = {};
};

// Any loops: the general kernel decodes its indices.
struct I8GeneralArgs {
  int8_t const * a;
  int8_t const * b;
  float const  * sa;       // null: 1
  float const  * sb;       // null: 1
  float const  * bias;     // null: 0
  void         * out;
  I8Loops c, m, n, k;
  int64_t C, M, N, K;
  int32_t tiles_m, tiles_n;
  int32_t out_bf16;
  int32_t relu;
  int32_t bias_rows;       // the bias runs over rows (A and B have changed places)
};

enum class I8Kernel : int32_t {
  GENERAL = 0      // any strides, 64 x 64 tiles (contract_i8.hip)
};

struct I8Plan {
  I8Kernel kernel = I8Kernel::GENERAL;
  bool     swapped = false;            // A = right tensor, B = left tensor
  bool     has_sa = false, has_sb = false, has_bias = false;
  I8GeneralArgs args{};                // pointers set at execution
  int64_t  flops = 0;
  int64_t  bytes = 0;
  std::string desc;
};

int plan_i8( int64_t         num_loops,
             int32_t const * dim_types,
             int64_t const * sizes,
             int64_t const * strides_left,
             int64_t const * strides_right,
             int64_t const * strides_scale_left,
             int64_t const * strides_scale_right,
             int64_t const * strides_bias,
             int64_t const * strides_out,
             int32_t         dtype_out,
             int32_t         ktype_last_touch,
             I8Plan        & plan );
int launch_i8( I8Plan const & plan,
               void const   * left,
               void const   * right,
               void const   * scale_left,
               void const   * scale_right,
               void const   * bias,
               void         * out,
               hipStream_t    stream );

int launch_i8_general( I8GeneralArgs const & a, hipStream_t stream );

// ---------------------------------------------------------------------------
// rows rounded to 8-bit integers with one scale a row
// ---------------------------------------------------------------------------
struct QuantPlan {
  bool    norm = false;                // RMS norm (else: activation)
  int64_t rows = 0;
  int64_t cols = 0;
  int32_t dtype = ETIR_BF16;
  int32_t dtype_weight = ETIR_BF16;
  int32_t ktype = ETIR_KTYPE_UNDEFINED;
  float   eps = 0.0f;
  int64_t ld_in = 0, ld_second = 0, ld_total = 0, ld_q = 0, ld_values = 0;
  int64_t bytes = 0;                   // with every optional tensor
  std::string desc;
};
void describe_quant( QuantPlan & plan );

// One row: y = norm or activation of the inputs, q = rint( y * 127 / max|y| ).
struct QuantArgs {
  void const * in;
  void const * second;      // residual (norm) or gate (activation); null: none
  void const * weight;      // norm: null: 1
  void       * total;       // norm: in + residual; null: not wanted
  int8_t     * q;
  float      * scale;
  void       * values;      // q * scale; null: not wanted
  int64_t rows, cols;
  int64_t ld_in, ld_second, ld_total, ld_q, ld_values;
  float   eps;
  int32_t weight_f32;
  int32_t ktype;
};

int launch_quant( QuantPlan const & plan, QuantArgs const & a, hipStream_t stream );

}  // namespace etir

#endif
