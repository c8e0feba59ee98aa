// gfx950 rows rounded to 8-bit integers with one scale a row: RMS norm with the
// residual's addition, and activations.
//
//   norm: s = in + residual,  y = s * weight       activation: y = f(in) or f(gate) * in
//   a = max |y|,  q = rint( y * (127 / a) ),  scale = a / 127 (norm: times 1 / rms(s))
//
// The norm's factor 1 / rms is the same for a whole row, so it cancels out of
// y / a: q needs the row's maximum only, and no sum's order shows in it.  The
// mean square is summed in fp64 (squares of fp32 stay in range), which costs
// nothing beside the row's bytes.
//
// One workgroup takes a row; two passes over it, the first for the sum and the
// maximum, the second for the outputs.
#include "i8_internal.h"
#include "contract_kernel.h"
#include <algorithm>
#include <cmath>

namespace etir {
namespace {

template< class T > __device__ inline float to_f32( T v );
template<> __device__ inline float to_f32< float >( float v ) { return v; }
template<> __device__ inline float to_f32< uint16_t >( uint16_t v ) { return kern::bf16_to_f32( v ); }
template< class T > __device__ inline T from_f32( float v );
template<> __device__ inline float from_f32< float >( float v ) { return v; }
template<> __device__ inline uint16_t from_f32< uint16_t >( float v ) { return kern::f32_to_bf16_rne( v ); }

__device__ inline float activate( float v, int32_t ktype ) {
  if( ktype == ETIR_KTYPE_RELU ) return v < 0.0f ? 0.0f : v;          // a NaN stays
  if( ktype == ETIR_KTYPE_SILU ) return v / ( 1.0f + expf( -v ) );
  return v;
}

// How a row's 8-bit integers follow from its maximum.  bits: the largest |y| as
// an integer; of non-negative floats the integers have the same order, with
// infinity and then every NaN above all finite ones.
struct RowScale {
  float pre;      // power of two that brings the row into range, exact
  float inv;      // 127 / ( a * pre )
  float a;        // max |y|
  bool  finite;
  __device__ explicit RowScale( uint32_t bits ) {
    a = __uint_as_float( bits );
    finite = bits < 0x7f800000u;
    // 127 / a is beyond fp32 for a below 2^-121: such rows are multiplied by 2^64 first
    pre = a < 0x1p-100f ? 0x1p64f : 1.0f;
    inv = finite && bits != 0u ? 127.0f / ( a * pre ) : 0.0f;
  }
  __device__ float q( float y ) const { return finite ? rintf( ( y * pre ) * inv ) : 0.0f; }
};

template< class T, bool NORM >
__global__ __launch_bounds__( 256 )
void quant_rows_kernel( QuantArgs a ) {
  __shared__ double   l_sums[4];
  __shared__ uint32_t l_tops[4];
  int const l_t = threadIdx.x;
  for( int64_t l_row = blockIdx.x; l_row < a.rows; l_row += gridDim.x ) {
  T const * l_in = static_cast< T const * >( a.in ) + l_row * a.ld_in;
  T const * l_second = a.second ? static_cast< T const * >( a.second ) + l_row * a.ld_second : nullptr;

  // the row's element i before rounding (norm: s in *sum)
  auto value = [&]( int64_t i, float * sum ) -> float {
    float l_v = to_f32( l_in[i] );
    if constexpr( NORM ) {
      if( l_second ) l_v += to_f32( l_second[i] );
      *sum = l_v;
      if( a.weight ) {
        l_v *= a.weight_f32 ? static_cast< float const * >( a.weight )[i]
                            : kern::bf16_to_f32( static_cast< uint16_t const * >( a.weight )[i] );
      }
      return l_v;
    }
    else {
      return l_second ? activate( to_f32( l_second[i] ), a.ktype ) * l_v : activate( l_v, a.ktype );
    }
  };

  double l_sum = 0.0;
  uint32_t l_top = 0;
  for( int64_t l_i = l_t; l_i < a.cols; l_i += 256 ) {
    float l_s = 0.0f;
    float const l_y = value( l_i, &l_s );
    l_sum += double( l_s ) * double( l_s );
    l_top = max( l_top, __float_as_uint( l_y ) & 0x7fffffffu );
  }
  for( int l_d = 32; l_d > 0; l_d /= 2 ) {
    l_sum += __shfl_xor( l_sum, l_d );
    l_top = max( l_top, uint32_t( __shfl_xor( int( l_top ), l_d ) ) );
  }
  if( l_t % 64 == 0 ) {
    l_sums[l_t / 64] = l_sum;
    l_tops[l_t / 64] = l_top;
  }
  __syncthreads();
  l_sum = ( l_sums[0] + l_sums[1] ) + ( l_sums[2] + l_sums[3] );
  l_top = max( max( l_tops[0], l_tops[1] ), max( l_tops[2], l_tops[3] ) );

  RowScale const l_r( l_top );
  float l_scale = l_r.a / 127.0f;
  if constexpr( NORM ) {
    if( l_top != 0u ) l_scale = float( double( l_r.a ) / ( 127.0 * sqrt( l_sum / double( a.cols ) + double( a.eps ) ) ) );
  }
  if( !l_r.finite ) l_scale = __uint_as_float( 0x7fc00000u );
  if( l_t == 0 ) a.scale[l_row] = l_scale;

  // an element's inputs are read by the thread that writes its outputs, so
  // total may be in or residual itself
  for( int64_t l_i = l_t; l_i < a.cols; l_i += 256 ) {
    float l_s = 0.0f;
    float const l_q = l_r.q( value( l_i, &l_s ) );
    a.q[l_row * a.ld_q + l_i] = int8_t( int( l_q ) );
    if constexpr( NORM ) {
      if( a.total ) static_cast< T * >( a.total )[l_row * a.ld_total + l_i] = from_f32< T >( l_s );
    }
    if( a.values ) static_cast< T * >( a.values )[l_row * a.ld_values + l_i] = from_f32< T >( l_q * l_scale );
  }
  __syncthreads();
  }
}

}  // namespace

void describe_quant( QuantPlan & plan ) {
  int64_t const l_item = plan.dtype == ETIR_BF16 ? 2 : 4;
  plan.bytes = plan.rows * ( plan.cols * ( ( plan.norm ? 4 : 3 ) * l_item + 1 ) + 4 );
  if( plan.norm ) plan.bytes += plan.cols * ( plan.dtype_weight == ETIR_BF16 ? 2 : 4 );
  plan.desc = std::string( plan.norm ? "norm_quant" : "act_quant" ) + " rows=" + std::to_string( plan.rows )
            + " cols=" + std::to_string( plan.cols ) + ( plan.dtype == ETIR_BF16 ? " bf16" : " fp32" );
}

int launch_quant( QuantPlan const & plan, QuantArgs const & args, hipStream_t stream ) {
  if( plan.rows == 0 ) return ETIR_SUCCESS;
  QuantArgs a = args;
  if( a.scale == nullptr || ( plan.cols > 0 && ( a.in == nullptr || a.q == nullptr ) ) ) {
    return fail( ETIR_NO_DATA_PTR_PROVIDED, plan.norm ? "norm_quant: null tensor pointer" : "act_quant: null tensor pointer" );
  }
  a.rows = plan.rows;
  a.cols = plan.cols;
  a.ld_in = plan.ld_in;
  a.ld_second = plan.ld_second;
  a.ld_total = plan.ld_total;
  a.ld_q = plan.ld_q;
  a.ld_values = plan.ld_values;
  a.eps = plan.eps;
  a.weight_f32 = plan.dtype_weight == ETIR_FP32;
  a.ktype = plan.ktype;
  // a grid's threads are counted in 32 bits, so workgroups loop over rows
  dim3 const l_grid( static_cast< uint32_t >( std::min< int64_t >( plan.rows, 1 << 20 ) ) ), l_block( 256 );
  bool const l_bf16 = plan.dtype == ETIR_BF16;
  if( l_bf16 && plan.norm )  hipLaunchKernelGGL( ( quant_rows_kernel< uint16_t, true > ), l_grid, l_block, 0, stream, a );
  if( l_bf16 && !plan.norm ) hipLaunchKernelGGL( ( quant_rows_kernel< uint16_t, false > ), l_grid, l_block, 0, stream, a );
  if( !l_bf16 && plan.norm ) hipLaunchKernelGGL( ( quant_rows_kernel< float, true > ), l_grid, l_block, 0, stream, a );
  if( !l_bf16 && !plan.norm ) hipLaunchKernelGGL( ( quant_rows_kernel< float, false > ), l_grid, l_block, 0, stream, a );
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "quant_rows launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

}  // namespace etir
