// Element types and activations of the operators that round rows to 8 bits
// (quant_rows.hip, quant_f8.hip).
#ifndef ETIR_ROWS_H
#define ETIR_ROWS_H

#include "contract_kernel.h"

namespace etir {
namespace rows {

template< class T > __device__ inline float to_f32( T v );
template<> __device__ inline float to_f32< float >( float v ) { return v; }
template<> __device__ inline float to_f32< uint16_t >( uint16_t v ) { return kern::bf16_to_f32( v ); }
template< class T > __device__ inline T from_f32( float v );
template<> __device__ inline float from_f32< float >( float v ) { return v; }
template<> __device__ inline uint16_t from_f32< uint16_t >( float v ) { return kern::f32_to_bf16_rne( v ); }

__device__ inline float activate( float v, int32_t ktype ) {
  if( ktype == ETIR_KTYPE_RELU ) return v < 0.0f ? 0.0f : v;          // a NaN stays
  if( ktype == ETIR_KTYPE_SILU ) {
    // exp(-v) = 2^t (1 + r ln 2), t + r = -v log2(e), t rounded, r its rest:
    // with the hardware's exponential and reciprocal (1 ulp each) within 8
    // half ulps of v / (1 + exp(-v)), at a third of the instructions of the
    // library's, which bounded the kernel (gated, 8192 x 8192 bf16: 98 -> 86 us).
    // A quarter of 1 + exp(-v) is inverted, whose reciprocal stays above 2^-126 up
    // to the end of exp's range (the hardware's is 0 below): near there, v < -87.3,
    // the quotient has up to 2 bits less, and below -88.7 exp(-v) is infinite and
    // y is 0.  Both factors lie between 0 and 1, and the clamp is part of the
    // instruction in front of it (NaN becomes 0): beyond 2.3e38 t and r are
    // infinite, so 2^t = 0 meets 1 and the quotient is 1, 2^t infinite meets 0
    // and it is 0; infinities and NaN come back in the last product.
    float const l_t = -v * 0x1.715476p+0f;
    float const l_r = fmaf( -v, 0x1.4ae0cp-26f, fmaf( -v, 0x1.715476p+0f, -l_t ) );
    float const l_f = __builtin_amdgcn_fmed3f( fmaf( l_r, 0x1.62e43p-3f, 0.25f ), 0.0f, 1.0f );
    float const l_e = __builtin_amdgcn_exp2f( l_t ) * l_f;
    return v * __builtin_amdgcn_fmed3f( 0.25f * __builtin_amdgcn_rcpf( 0.25f + l_e ), 0.0f, 1.0f );
  }
  return v;
}

}  // namespace rows
}  // namespace etir

#endif
