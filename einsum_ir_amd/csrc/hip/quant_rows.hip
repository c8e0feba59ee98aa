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
// Bound by the row's bytes: every input is read once and kept in registers, as
// fp32, while the row's maximum (and mean square) is found; 16 bytes a lane and
// load, at any address.  A row longer than the registers hold is read twice.
#include "i8_internal.h"
#include "rows.h"
#include <algorithm>
#include <cmath>

namespace etir {
namespace {

using rows::to_f32;
using rows::from_f32;
using rows::activate;

// How a row's 8-bit integers follow from its maximum.  bits: the largest |y| as
// an integer; of non-negative floats the integers have the same order, with
// infinity and then every NaN above all finite ones.
// Adding 1.5 * 2^23 to a float of magnitude up to 127 rounds it to an integer
// (ties to even), which is then in the low bits.
constexpr float kMagic = 12582912.0f;
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
  // what y has to be made in rows that are not ordinary (uniform in a row)
  __device__ bool ordinary() const { return finite && pre == 1.0f; }
  __device__ float ready( float y ) const { return finite ? y * pre : 0.0f; }
  // rint( y * inv ) + kMagic of a ready y: the integer is the low byte
  __device__ float q( float y ) const {
#pragma clang fp contract( off )
    float const l_t = y * inv;
    return l_t + kMagic;
  }
};

// V elements of a row at any address: 16 bytes
template< class T > struct Vec;
template<> struct Vec< float > {
  static constexpr int V = 4;
  typedef float    t __attribute__( ( ext_vector_type( 4 ), aligned( 4 ) ) );
  typedef uint32_t q __attribute__( ( ext_vector_type( 1 ), aligned( 4 ) ) );
  __device__ static void unpack( t v, float * f ) {
#pragma unroll
    for( int l_i = 0; l_i < V; l_i++ ) f[l_i] = v[l_i];
  }
  __device__ static t pack( float const * f ) { return t{ f[0], f[1], f[2], f[3] }; }
};
template<> struct Vec< uint16_t > {
  static constexpr int V = 8;
  typedef uint32_t t __attribute__( ( ext_vector_type( 4 ), aligned( 2 ) ) );
  typedef uint32_t q __attribute__( ( ext_vector_type( 2 ), aligned( 4 ) ) );
  __device__ static void unpack( t v, float * f ) {
#pragma unroll
    for( int l_i = 0; l_i < V; l_i += 2 ) {
      f[l_i]     = __uint_as_float( v[l_i / 2] << 16 );
      f[l_i + 1] = __uint_as_float( v[l_i / 2] & 0xffff0000u );
    }
  }
  __device__ static t pack( float const * f ) {
    typedef __bf16 b2 __attribute__( ( ext_vector_type( 2 ) ) );
    t l_v;
#pragma unroll
    for( int l_i = 0; l_i < 4; l_i++ ) {
      l_v[l_i] = __builtin_bit_cast( uint32_t, b2{ static_cast< __bf16 >( f[2 * l_i] ), static_cast< __bf16 >( f[2 * l_i + 1] ) } );
    }
    return l_v;
  }
};

// A vector of a row of n elements: those of i .. i + V - 1 that the row has.
// It is read from `at`, where all V are inside the row (so that no lane waits
// for element-wise loads of its own); what does not belong to it counts as
// zeros and is not written.  n < V: read element by element, at = 0.
template< int V >
struct Place {
  int32_t i, at;
  __device__ Place( int32_t i_, int32_t n ) : i( i_ ), at( max( min( i_, n - V ), 0 ) ) {}
  __device__ bool whole( int32_t n ) const { return at == i && n >= V; }
  __device__ bool has( int e, int32_t n ) const { return at + e >= i && at + e < i + V && at + e < n; }
};

template< class T >
__device__ inline void load_v( T const * row, int32_t at, int32_t n, float * f ) {
  if( n >= Vec< T >::V ) {
    Vec< T >::unpack( *reinterpret_cast< typename Vec< T >::t const * >( row + at ), f );
    return;
  }
#pragma unroll
  for( int l_e = 0; l_e < Vec< T >::V; l_e++ ) f[l_e] = l_e < n ? to_f32( row[l_e] ) : 0.0f;
}

// Non-temporal: these rows are written whole and not read here again (norm of
// 16384 x 8192 bf16: 223 -> 215 us; with non-temporal loads 227, and 4072 x 2048
// 14.2 -> 19.2).
template< class T >
__device__ inline void store_v( T * row, Place< Vec< T >::V > p, int32_t n, float const * f ) {
  if( p.whole( n ) ) {
    __builtin_nontemporal_store( Vec< T >::pack( f ), reinterpret_cast< typename Vec< T >::t * >( row + p.at ) );
    return;
  }
#pragma unroll
  for( int l_e = 0; l_e < Vec< T >::V; l_e++ ) {
    if( p.has( l_e, n ) ) row[p.at + l_e] = from_f32< T >( f[l_e] );
  }
}

// Workgroups of a launch at most (a grid's threads are counted in 32 bits): they
// loop over rows.  A constant, since a kernel that reads its grid's size is
// given 256 bytes of further arguments, which cost 0.7 us of the host.
constexpr int64_t kMaxGroups = 1 << 20;

// THREADS threads a row; a workgroup takes 4 rows of a wave each, or one row.  CHUNKS > 0: the row fits
// CHUNKS vectors a thread; 0: it is read twice.
template< class T, bool NORM, int THREADS, int CHUNKS >
__global__ __launch_bounds__( THREADS == 64 ? 256 : THREADS )
void quant_rows_kernel( QuantArgs a ) {
  constexpr int V     = Vec< T >::V;
  constexpr int ROWS  = THREADS == 64 ? 4 : 1;               // rows a workgroup
  constexpr int WAVES = THREADS / 64;                        // waves a row
  constexpr int HELD  = CHUNKS > 0 ? CHUNKS : 1;
  __shared__ double   l_sums[WAVES];
  __shared__ uint32_t l_tops[WAVES];
  int const l_t = threadIdx.x % THREADS;
  int const l_sub = __builtin_amdgcn_readfirstlane( threadIdx.x / THREADS );
  int32_t const l_cols = a.cols;

  // rows of one workgroup's waves are apart only where a wave holds a whole
  // row, so every thread of a workgroup meets the same barriers
  for( int64_t l_row = int64_t( blockIdx.x ) * ROWS + l_sub; l_row < a.rows;
       l_row += kMaxGroups * ROWS ) {
    T const * l_in = static_cast< T const * >( a.in ) + l_row * a.ld_in;
    // Vectors start where those of q lie at multiples of 4 bytes: off them 16
    // bytes move at a third of the rate.  Where all rows are one after the
    // other that is a multiple of 4 elements in every tensor.
    int const l_shift = int( ( reinterpret_cast< uintptr_t >( a.q ) + l_row * a.ld_q ) & 3 );
    T const * l_second = a.second ? static_cast< T const * >( a.second ) + l_row * a.ld_second : nullptr;

    // V elements before rounding; norm: s in l_s
    auto value = [&]( Place< V > const & p, float * y, float * s ) {
      load_v( l_in, p.at, l_cols, y );
      float l_f[V];
      if constexpr( NORM ) {
        if( l_second ) {
          load_v( l_second, p.at, l_cols, l_f );
#pragma unroll
          for( int l_e = 0; l_e < V; l_e++ ) y[l_e] += l_f[l_e];
        }
#pragma unroll
        for( int l_e = 0; l_e < V; l_e++ ) s[l_e] = y[l_e];
        if( a.weight ) {
          if( ( a.mode != 0 ) != ( V == 4 ) ) {
            // the weight's type is not the row's
#pragma unroll
            for( int l_e = 0; l_e < V; l_e++ ) {
              int32_t const l_i = min( p.at + l_e, l_cols - 1 );
              l_f[l_e] = V == 8 ? static_cast< float const * >( a.weight )[l_i]
                                : to_f32( static_cast< uint16_t const * >( a.weight )[l_i] );
            }
          }
          else load_v( static_cast< T const * >( a.weight ), p.at, l_cols, l_f );
#pragma unroll
          for( int l_e = 0; l_e < V; l_e++ ) y[l_e] *= l_f[l_e];
        }
      }
      else if( l_second ) {
        load_v( l_second, p.at, l_cols, l_f );
#pragma unroll
        for( int l_e = 0; l_e < V; l_e++ ) y[l_e] *= activate( l_f[l_e], a.mode );
      }
      else {
#pragma unroll
        for( int l_e = 0; l_e < V; l_e++ ) y[l_e] = activate( y[l_e], a.mode );
      }
      if( !p.whole( l_cols ) ) {
#pragma unroll
        for( int l_e = 0; l_e < V; l_e++ ) {
          if( p.has( l_e, l_cols ) ) continue;
          y[l_e] = 0.0f;
          if constexpr( NORM ) s[l_e] = 0.0f;
        }
      }
    };

    float l_y[HELD][V];
    double l_sum = 0.0;
    uint32_t l_top = 0;
    auto first = [&]( int32_t i, float * y ) {
      float l_s[V];
      Place< V > const l_p( i, l_cols );
      value( l_p, y, l_s );
#pragma unroll
      for( int l_e = 0; l_e < V; l_e++ ) {
        if constexpr( NORM ) l_sum += double( l_s[l_e] ) * double( l_s[l_e] );
        l_top = max( l_top, __float_as_uint( y[l_e] ) & 0x7fffffffu );
      }
      // Total may be in or residual itself: an element is written by the thread
      // whose vector it belongs to, after it was read there for the last time;
      // a vector beside it that reads it too does not count it.
      if constexpr( NORM && CHUNKS > 0 ) {
        if( a.total ) store_v( static_cast< T * >( a.total ) + l_row * a.ld_total, l_p, l_cols, l_s );
      }
    };
    if constexpr( CHUNKS > 0 ) {
#pragma unroll
      for( int l_c = 0; l_c < CHUNKS; l_c++ ) {
        int32_t const l_i = ( l_c * THREADS + l_t ) * V - l_shift;
        if( l_i < l_cols ) first( l_i, l_y[l_c] );
      }
    }
    else {
      for( int32_t l_i = l_t * V - l_shift; l_i < l_cols; l_i += THREADS * V ) first( l_i, l_y[0] );
    }

#pragma unroll
    for( int l_d = 32; l_d > 0; l_d /= 2 ) {
      if constexpr( NORM ) l_sum += __shfl_xor( l_sum, l_d );
      l_top = max( l_top, uint32_t( __shfl_xor( int( l_top ), l_d ) ) );
    }
    if constexpr( WAVES > 1 ) {
      if( l_t % 64 == 0 ) {
        l_sums[l_t / 64] = l_sum;
        l_tops[l_t / 64] = l_top;
      }
      __syncthreads();
      l_sum = 0.0;
#pragma unroll
      for( int l_w = 0; l_w < WAVES; l_w++ ) {
        if constexpr( NORM ) l_sum += l_sums[l_w];
        l_top = max( l_top, l_tops[l_w] );
      }
    }

    RowScale const l_r( l_top );
    float l_scale = l_r.a / 127.0f;
    if constexpr( NORM ) {
      if( l_top != 0u ) l_scale = float( double( l_r.a ) / ( 127.0 * sqrt( l_sum / double( a.cols ) + double( a.eps ) ) ) );
    }
    if( !l_r.finite ) l_scale = __uint_as_float( 0x7fc00000u );
    if( l_t == 0 ) a.scale[l_row] = l_scale;

    if( !l_r.ordinary() ) {
#pragma unroll
      for( int l_c = 0; l_c < HELD; l_c++ ) {
#pragma unroll
        for( int l_e = 0; l_e < V; l_e++ ) l_y[l_c][l_e] = l_r.ready( l_y[l_c][l_e] );
      }
    }
    auto last = [&]( int32_t i, float const * y ) {
      Place< V > const l_p( i, l_cols );
      float l_q[V];
      uint32_t l_w[V / 4];
#pragma unroll
      for( int l_e = 0; l_e < V; l_e++ ) l_q[l_e] = l_r.q( y[l_e] );
#pragma unroll
      for( int l_e = 0; l_e < V; l_e += 4 ) {
        // low bytes of four floats
        uint32_t const l_lo = __builtin_amdgcn_perm( __float_as_uint( l_q[l_e + 1] ), __float_as_uint( l_q[l_e] ), 0x0c0c0400u );
        uint32_t const l_hi = __builtin_amdgcn_perm( __float_as_uint( l_q[l_e + 3] ), __float_as_uint( l_q[l_e + 2] ), 0x04000c0cu );
        l_w[l_e / 4] = l_lo | l_hi;
      }
      int8_t * l_to = a.q + l_row * a.ld_q + l_p.at;
      if( l_p.whole( l_cols ) ) {
        typename Vec< T >::q l_bits;
#pragma unroll
        for( int l_e = 0; l_e < V / 4; l_e++ ) l_bits[l_e] = l_w[l_e];
        *reinterpret_cast< typename Vec< T >::q * >( l_to ) = l_bits;
      }
      else {
#pragma unroll
        for( int l_e = 0; l_e < V; l_e++ ) if( l_p.has( l_e, l_cols ) ) l_to[l_e] = int8_t( l_w[l_e / 4] >> ( 8 * ( l_e % 4 ) ) );
      }
      if( a.values ) {
#pragma unroll
        for( int l_e = 0; l_e < V; l_e++ ) l_q[l_e] = ( l_q[l_e] - kMagic ) * l_scale;
        store_v( static_cast< T * >( a.values ) + l_row * a.ld_values, l_p, l_cols, l_q );
      }
    };
    if constexpr( CHUNKS > 0 ) {
#pragma unroll
      for( int l_c = 0; l_c < CHUNKS; l_c++ ) {
        int32_t const l_i = ( l_c * THREADS + l_t ) * V - l_shift;
        if( l_i < l_cols ) last( l_i, l_y[l_c] );
      }
    }
    else {
      for( int32_t l_i = l_t * V - l_shift; l_i < l_cols; l_i += THREADS * V ) {
        float l_s[V];
        Place< V > const l_p( l_i, l_cols );
        value( l_p, l_y[0], l_s );
        if( !l_r.ordinary() ) {
#pragma unroll
          for( int l_e = 0; l_e < V; l_e++ ) l_y[0][l_e] = l_r.ready( l_y[0][l_e] );
        }
        if constexpr( NORM ) {
          if( a.total ) store_v( static_cast< T * >( a.total ) + l_row * a.ld_total, l_p, l_cols, l_s );
        }
        last( l_i, l_y[0] );
      }
    }
    if constexpr( WAVES > 1 ) __syncthreads();
  }
}

template< class T, bool NORM, int THREADS, int CHUNKS >
void launch_shape( QuantArgs const & a, hipStream_t stream ) {
  constexpr int ROWS = THREADS == 64 ? 4 : 1;
  int64_t const l_grid = std::min( ( int64_t( a.rows ) + ROWS - 1 ) / ROWS, kMaxGroups );
  hipLaunchKernelGGL( ( quant_rows_kernel< T, NORM, THREADS, CHUNKS > ), dim3( uint32_t( l_grid ) ),
                      dim3( ROWS * THREADS ), 0, stream, a );
}

// Threads a row by its vectors of 16 bytes: a wave where one vector a lane
// holds the row (no exchange between waves), else few waves with two vectors a
// lane, which leaves most of a compute unit's registers to other rows: 4072
// rows of 256 vectors take 14.2 us so and 15.6 with one vector (a single row 4.1
// and 3.5); 300 of 88 take 5.8 with two vectors in a wave and 4.2 with one in two
// waves.
template< class T, bool NORM >
void launch_rows( QuantArgs const & a, hipStream_t stream ) {
  // a row of q that starts off a multiple of 4 bytes shifts its vectors
  bool const l_even = reinterpret_cast< uintptr_t >( a.q ) % 4 == 0 && ( a.ld_q % 4 == 0 || a.rows == 1 );
  int64_t const l_vecs = ( a.cols + ( l_even ? 0 : 3 ) + Vec< T >::V - 1 ) / Vec< T >::V;
  if( l_vecs <= 64 )        launch_shape< T, NORM, 64, 1 >( a, stream );
  else if( l_vecs <= 128 )  launch_shape< T, NORM, 128, 1 >( a, stream );
  else if( l_vecs <= 256 )  launch_shape< T, NORM, 128, 2 >( a, stream );
  else if( l_vecs <= 512 )  launch_shape< T, NORM, 256, 2 >( a, stream );
  else if( l_vecs <= 1024 ) launch_shape< T, NORM, 512, 2 >( a, stream );
  else if( l_vecs <= 1536 ) launch_shape< T, NORM, 768, 2 >( a, stream );
  else if( l_vecs <= 2048 ) launch_shape< T, NORM, 512, 4 >( a, stream );
  else {
    if constexpr( Vec< T >::V == 4 ) {
      if( l_vecs <= 4096 ) return launch_shape< T, NORM, 1024, 4 >( a, stream );
    }
    launch_shape< T, NORM, 1024, 0 >( a, stream );
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
  a.rows = int32_t( plan.rows );
  a.cols = int32_t( plan.cols );
  // rows of nothing: the scales are 0 (a vector in front of q's first dword would
  // take the weight of a column that is not there)
  if( a.cols == 0 ) a.weight = nullptr;
  a.ld_in = plan.ld_in;
  a.ld_second = plan.ld_second;
  a.ld_total = plan.ld_total;
  a.ld_q = plan.ld_q;
  a.ld_values = plan.ld_values;
  a.eps = plan.eps;
  a.mode = plan.norm ? int32_t( plan.dtype_weight == ETIR_FP32 ) : plan.ktype;
  if( plan.dtype == ETIR_BF16 ) plan.norm ? launch_rows< uint16_t, true >( a, stream ) : launch_rows< uint16_t, false >( a, stream );
  else                          plan.norm ? launch_rows< float, true >( a, stream ) : launch_rows< float, false >( a, stream );
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "quant_rows launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

}  // namespace etir
