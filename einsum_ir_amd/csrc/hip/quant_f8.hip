// gfx950 rounding to 8-bit floating point with one scale a block:
//
//   y = in or f(in) or f(gate) * in (fp32),  a = max |y| of a block
//   scale = 2^e, e the least integer >= -126 with a <= fmax 2^e,  q = rne( y / scale )
//
// fmax is 448 (e4m3) or 57344 (e5m2).  A power of two divides exactly, so q is
// y's own rounding to 3 (2) bits behind the point and no order of operations
// shows in it; against a / fmax it costs up to one of the 18 (32) binades below
// the block's maximum, and no precision above them.  A block of zeros has scale
// 1, one with an infinity or a NaN has q = 0 and a NaN for its scale.
//
// Bound by bytes: every input is read once and kept in registers while the
// block's maximum is found.  Blocks of a row (1 x 128): 16 lanes a block (fp32:
// 32), 16 bytes a lane and load, the maximum by exchanges between those lanes.
// Blocks of 128 rows: a workgroup takes 128 x 128 elements, 64 a thread.  8192 x
// 8192 gated bf16 in blocks of a row: 88 us, 5.3 TB/s; 4 x 2048 x 2048 fp32 in blocks
// of 128 x 128: 25 us, 6 TB/s with a part of the input in the cache.
#include "block_internal.h"
#include "rows.h"

namespace etir {
namespace {

typedef float f32x2 __attribute__( ( ext_vector_type( 2 ) ) );

struct QuantF8Args {
  void const * in;
  void const * gate;        // null: none
  void       * q;
  void       * scale;
  void       * values;      // q * scale; null: not wanted
  int64_t ld_in, ld_gate, ld_q, ld_values;
  int64_t rows;             // of one matrix (blocks of 128 rows), of all (blocks of a row)
  int32_t cols;
  int32_t ktype;
  int32_t e8m0;
};

// 16 bytes of a row at any address
template< class T > struct Vec;
template<> struct Vec< float > {
  static constexpr int V = 4;
  typedef float    t __attribute__( ( ext_vector_type( 4 ), aligned( 4 ) ) );
  typedef uint32_t q __attribute__( ( aligned( 1 ) ) );
  __device__ static void unpack( t v, float * f ) {
#pragma unroll
    for( int l_i = 0; l_i < V; l_i++ ) f[l_i] = v[l_i];
  }
  __device__ static t pack( float const * f ) { return t{ f[0], f[1], f[2], f[3] }; }
};
template<> struct Vec< uint16_t > {
  static constexpr int V = 8;
  typedef uint32_t t __attribute__( ( ext_vector_type( 4 ), aligned( 2 ) ) );
  typedef uint32_t q __attribute__( ( ext_vector_type( 2 ), aligned( 1 ) ) );
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

// n of V elements
template< class T >
__device__ inline void load_v( T const * p, int n, float * f ) {
  if( n >= Vec< T >::V ) {
    Vec< T >::unpack( *reinterpret_cast< typename Vec< T >::t const * >( p ), f );
    return;
  }
#pragma unroll
  for( int l_e = 0; l_e < Vec< T >::V; l_e++ ) f[l_e] = l_e < n ? rows::to_f32( p[l_e] ) : 0.0f;
}

// y of n elements at one place of in and gate
template< class T >
__device__ inline void values_v( QuantF8Args const & a, T const * in, T const * gate, int n, float * y ) {
  load_v( in, n, y );
  if( gate ) {
    float l_g[Vec< T >::V];
    load_v( gate, n, l_g );
#pragma unroll
    for( int l_e = 0; l_e < Vec< T >::V; l_e++ ) y[l_e] *= rows::activate( l_g[l_e], a.ktype );
  }
  else if( a.ktype != ETIR_KTYPE_UNDEFINED ) {
#pragma unroll
    for( int l_e = 0; l_e < Vec< T >::V; l_e++ ) y[l_e] = rows::activate( y[l_e], a.ktype );
  }
}

// |y| as an integer: of non-negative floats the integers have the same order,
// with infinity and then every NaN above all finite ones
__device__ inline uint32_t magnitude( float y ) { return __float_as_uint( y ) & 0x7fffffffu; }

// a block's scale from its largest magnitude
template< bool E5M2 >
struct BlockScale {
  uint32_t exponent;      // of the scale, biased by 127; 255: the block is not finite
  __device__ explicit BlockScale( uint32_t top ) {
    // fmax is 1.75 * 2^8 (2^15): the exponent of the least power of two times
    // 1.75 that is at least a
    constexpr int32_t TOP = E5M2 ? 15 : 8;
    exponent = top >= 0x7f800000u ? 255u
             : top == 0u ? 127u : uint32_t( max( int32_t( ( top + 0x1fffffu ) >> 23 ) - TOP, 1 ) );
  }
  __device__ bool finite() const { return exponent != 255u; }
  __device__ float scale() const { return finite() ? __uint_as_float( exponent << 23 ) : __uint_as_float( 0x7fc00000u ); }
  __device__ float inverse() const { return __uint_as_float( ( 254u - exponent ) << 23 ); }      // finite
  __device__ void store( void * at, int64_t i, int32_t e8m0 ) const {
    if( e8m0 ) static_cast< uint8_t * >( at )[i] = uint8_t( exponent );
    else       static_cast< float * >( at )[i] = scale();
  }
};

// four numbers to 8 bits, and back
template< bool E5M2 >
__device__ inline uint32_t round4( float const * y ) {
  int l_w = 0;
  if constexpr( E5M2 ) {
    l_w = __builtin_amdgcn_cvt_pk_bf8_f32( y[0], y[1], l_w, false );
    l_w = __builtin_amdgcn_cvt_pk_bf8_f32( y[2], y[3], l_w, true );
  }
  else {
    l_w = __builtin_amdgcn_cvt_pk_fp8_f32( y[0], y[1], l_w, false );
    l_w = __builtin_amdgcn_cvt_pk_fp8_f32( y[2], y[3], l_w, true );
  }
  return uint32_t( l_w );
}
template< bool E5M2 >
__device__ inline void widen4( uint32_t w, float * y ) {
  f32x2 l_lo, l_hi;
  if constexpr( E5M2 ) {
    l_lo = __builtin_amdgcn_cvt_pk_f32_bf8( int( w ), false );
    l_hi = __builtin_amdgcn_cvt_pk_f32_bf8( int( w ), true );
  }
  else {
    l_lo = __builtin_amdgcn_cvt_pk_f32_fp8( int( w ), false );
    l_hi = __builtin_amdgcn_cvt_pk_f32_fp8( int( w ), true );
  }
  y[0] = l_lo[0];
  y[1] = l_lo[1];
  y[2] = l_hi[0];
  y[3] = l_hi[1];
}

// Rounds n of V numbers and stores them; what is not finite becomes 0, the
// block's scale says so.  Outputs are written whole and not read here again.
template< class T, bool E5M2 >
__device__ inline void finish_v( float const * y, int n, float const * scale, float const * inverse, bool const * finite,
                                 uint8_t * q, T * values ) {
  constexpr int V = Vec< T >::V;
  float l_y[V];
#pragma unroll
  for( int l_e = 0; l_e < V; l_e++ ) l_y[l_e] = finite[l_e] ? y[l_e] * inverse[l_e] : 0.0f;
  uint32_t l_w[V / 4];
#pragma unroll
  for( int l_i = 0; l_i < V / 4; l_i++ ) l_w[l_i] = round4< E5M2 >( l_y + 4 * l_i );
  if( n >= V ) {
    typename Vec< T >::q l_q;
    if constexpr( V == 4 ) l_q = l_w[0];
    else {
      l_q[0] = l_w[0];
      l_q[1] = l_w[1];
    }
    *reinterpret_cast< typename Vec< T >::q * >( q ) = l_q;
  }
  else {
#pragma unroll
    for( int l_e = 0; l_e < V; l_e++ ) if( l_e < n ) q[l_e] = uint8_t( l_w[l_e / 4] >> ( 8 * ( l_e % 4 ) ) );
  }
  if( values ) {
    float l_v[V];
#pragma unroll
    for( int l_i = 0; l_i < V / 4; l_i++ ) widen4< E5M2 >( l_w[l_i], l_v + 4 * l_i );
#pragma unroll
    for( int l_e = 0; l_e < V; l_e++ ) l_v[l_e] *= scale[l_e];
    if( n >= V ) __builtin_nontemporal_store( Vec< T >::pack( l_v ), reinterpret_cast< typename Vec< T >::t * >( values ) );
    else {
#pragma unroll
      for( int l_e = 0; l_e < V; l_e++ ) if( l_e < n ) values[l_e] = rows::from_f32< T >( l_v[l_e] );
    }
  }
}

constexpr int kThreads = 256;

// Blocks of a row.  PASSES blocks for each group of lanes, all loaded before the
// first is rounded.
template< class T, bool E5M2, int PASSES >
__global__ __launch_bounds__( kThreads )
void quant_f8_rows_kernel( QuantF8Args a ) {
  constexpr int V = Vec< T >::V, LANES = kScaleBlock / V;       // lanes a block
  constexpr int EACH = kThreads / LANES;                        // blocks a pass
  int32_t const l_blocks = ( a.cols + kScaleBlock - 1 ) / kScaleBlock;
  uint64_t const l_first = uint64_t( blockIdx.x ) * ( EACH * PASSES );
  uint64_t const l_row0 = l_first / uint32_t( l_blocks );
  uint32_t const l_at = uint32_t( l_first % uint32_t( l_blocks ) ) + threadIdx.x / LANES;
  int const l_lane = threadIdx.x % LANES;

  float l_y[PASSES][V];
  int64_t l_row[PASSES];
  int32_t l_col[PASSES];
  int l_n[PASSES];
#pragma unroll
  for( int l_p = 0; l_p < PASSES; l_p++ ) {
    uint32_t const l_i = l_at + l_p * EACH;
    l_row[l_p] = int64_t( l_row0 + l_i / uint32_t( l_blocks ) );
    l_col[l_p] = int32_t( l_i % uint32_t( l_blocks ) ) * kScaleBlock + l_lane * V;
    l_n[l_p] = l_row[l_p] < a.rows ? a.cols - l_col[l_p] : 0;
    if( l_n[l_p] > 0 ) {
      values_v< T >( a, static_cast< T const * >( a.in ) + l_row[l_p] * a.ld_in + l_col[l_p],
                     a.gate ? static_cast< T const * >( a.gate ) + l_row[l_p] * a.ld_gate + l_col[l_p] : nullptr, l_n[l_p], l_y[l_p] );
    }
    else {
#pragma unroll
      for( int l_e = 0; l_e < V; l_e++ ) l_y[l_p][l_e] = 0.0f;
    }
  }
#pragma unroll
  for( int l_p = 0; l_p < PASSES; l_p++ ) {
    uint32_t l_top = 0;
#pragma unroll
    for( int l_e = 0; l_e < V; l_e++ ) l_top = max( l_top, magnitude( l_y[l_p][l_e] ) );
#pragma unroll
    for( int l_d = LANES / 2; l_d > 0; l_d /= 2 ) l_top = max( l_top, uint32_t( __shfl_xor( int( l_top ), l_d ) ) );
    if( l_n[l_p] <= 0 ) continue;
    BlockScale< E5M2 > const l_s( l_top );
    float l_scale[V], l_inverse[V];
    bool l_finite[V];
#pragma unroll
    for( int l_e = 0; l_e < V; l_e++ ) {
      l_scale[l_e] = l_s.scale();
      l_inverse[l_e] = l_s.inverse();
      l_finite[l_e] = l_s.finite();
    }
    finish_v< T, E5M2 >( l_y[l_p], l_n[l_p], l_scale, l_inverse, l_finite,
                         static_cast< uint8_t * >( a.q ) + l_row[l_p] * a.ld_q + l_col[l_p],
                         a.values ? static_cast< T * >( a.values ) + l_row[l_p] * a.ld_values + l_col[l_p] : nullptr );
    if( l_lane == 0 ) l_s.store( a.scale, l_row[l_p] * l_blocks + l_col[l_p] / kScaleBlock, a.e8m0 );
  }
}

// Blocks of 128 rows, and of 128 columns (SQUARE) or one.
template< class T, bool E5M2, bool SQUARE >
__global__ __launch_bounds__( kThreads )
void quant_f8_tile_kernel( QuantF8Args a ) {
  constexpr int V = Vec< T >::V, LANES = kScaleBlock / V;
  constexpr int ROWS = kThreads / LANES, PASSES = kScaleBlock / ROWS;
  __shared__ uint32_t l_tops[kThreads / 64][SQUARE ? 1 : kScaleBlock];
  int32_t const l_tiles_n = ( a.cols + kScaleBlock - 1 ) / kScaleBlock;
  int64_t const l_tiles_m = ( a.rows + kScaleBlock - 1 ) / kScaleBlock;
  int32_t const l_tile_n = int32_t( blockIdx.x % uint32_t( l_tiles_n ) );
  int64_t const l_bm = blockIdx.x / uint32_t( l_tiles_n );      // tile row, counted through the matrices
  int64_t const l_b = l_bm / l_tiles_m, l_m0 = l_bm % l_tiles_m * kScaleBlock;
  int const l_row = threadIdx.x / LANES;
  int32_t const l_c = threadIdx.x % LANES * V, l_col = l_tile_n * kScaleBlock + l_c;
  int const l_n = a.cols - l_col;
  int64_t const l_first = l_b * a.rows + l_m0 + l_row;          // row of the first pass, through the matrices

  float l_y[PASSES][V];
  uint32_t l_top[V];
#pragma unroll
  for( int l_e = 0; l_e < V; l_e++ ) l_top[l_e] = 0;
#pragma unroll
  for( int l_p = 0; l_p < PASSES; l_p++ ) {
    int64_t const l_r = l_first + l_p * ROWS;
    if( l_n > 0 && l_m0 + l_row + l_p * ROWS < a.rows ) {
      values_v< T >( a, static_cast< T const * >( a.in ) + l_r * a.ld_in + l_col,
                     a.gate ? static_cast< T const * >( a.gate ) + l_r * a.ld_gate + l_col : nullptr, l_n, l_y[l_p] );
    }
    else {
#pragma unroll
      for( int l_e = 0; l_e < V; l_e++ ) l_y[l_p][l_e] = 0.0f;
    }
  }
#pragma unroll
  for( int l_p = 0; l_p < PASSES; l_p++ ) {
#pragma unroll
    for( int l_e = 0; l_e < V; l_e++ ) l_top[l_e] = max( l_top[l_e], magnitude( l_y[l_p][l_e] ) );
  }
  // over the lanes of the same columns, or all
#pragma unroll
  for( int l_e = 0; l_e < V; l_e++ ) {
    if( SQUARE && l_e > 0 ) continue;
    if constexpr( SQUARE ) {
#pragma unroll
      for( int l_i = 1; l_i < V; l_i++ ) l_top[0] = max( l_top[0], l_top[l_i] );
    }
#pragma unroll
    for( int l_d = 32; l_d >= ( SQUARE ? 1 : LANES ); l_d /= 2 ) l_top[l_e] = max( l_top[l_e], uint32_t( __shfl_xor( int( l_top[l_e] ), l_d ) ) );
  }
  int const l_lane = threadIdx.x % 64, l_wave = threadIdx.x / 64;
  if constexpr( SQUARE ) {
    if( l_lane == 0 ) l_tops[l_wave][0] = l_top[0];
  }
  else if( l_lane < LANES ) {
#pragma unroll
    for( int l_e = 0; l_e < V; l_e++ ) l_tops[l_wave][l_c + l_e] = l_top[l_e];
  }
  __syncthreads();
  float l_scale[V], l_inverse[V];
  bool l_finite[V];
#pragma unroll
  for( int l_e = 0; l_e < V; l_e++ ) {
    uint32_t l_max = 0;
#pragma unroll
    for( int l_w = 0; l_w < kThreads / 64; l_w++ ) l_max = max( l_max, l_tops[l_w][SQUARE ? 0 : l_c + l_e] );
    BlockScale< E5M2 > const l_s( l_max );
    l_scale[l_e] = l_s.scale();
    l_inverse[l_e] = l_s.inverse();
    l_finite[l_e] = l_s.finite();
    if constexpr( SQUARE ) {
      if( threadIdx.x == 0 && l_e == 0 ) l_s.store( a.scale, l_bm * l_tiles_n + l_tile_n, a.e8m0 );
    }
    else {
      if( l_row == 0 && l_e < l_n ) l_s.store( a.scale, l_bm * a.cols + l_col + l_e, a.e8m0 );
    }
  }
  if( l_n <= 0 ) return;
#pragma unroll
  for( int l_p = 0; l_p < PASSES; l_p++ ) {
    int64_t const l_r = l_first + l_p * ROWS;
    if( l_m0 + l_row + l_p * ROWS >= a.rows ) break;
    finish_v< T, E5M2 >( l_y[l_p], l_n, l_scale, l_inverse, l_finite, static_cast< uint8_t * >( a.q ) + l_r * a.ld_q + l_col,
                         a.values ? static_cast< T * >( a.values ) + l_r * a.ld_values + l_col : nullptr );
  }
}

template< class T, bool E5M2 >
int launch_type( QuantF8Plan const & plan, QuantF8Args const & a, hipStream_t stream ) {
  int64_t const l_blocks_n = ( plan.cols + kScaleBlock - 1 ) / kScaleBlock;
  if( plan.block_rows == 1 ) {
    constexpr int PASSES = 4, EACH = kThreads / ( kScaleBlock / Vec< T >::V ) * PASSES;
    int64_t const l_grid = ( a.rows * l_blocks_n + EACH - 1 ) / EACH;
    hipLaunchKernelGGL( ( quant_f8_rows_kernel< T, E5M2, PASSES > ), dim3( uint32_t( l_grid ) ), dim3( kThreads ), 0, stream, a );
  }
  else {
    int64_t const l_grid = plan.batch * ( ( a.rows + kScaleBlock - 1 ) / kScaleBlock ) * l_blocks_n;
    if( plan.block_cols == 1 ) hipLaunchKernelGGL( ( quant_f8_tile_kernel< T, E5M2, false > ), dim3( uint32_t( l_grid ) ), dim3( kThreads ), 0, stream, a );
    else                       hipLaunchKernelGGL( ( quant_f8_tile_kernel< T, E5M2, true > ), dim3( uint32_t( l_grid ) ), dim3( kThreads ), 0, stream, a );
  }
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "quant_f8 launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

}  // namespace

int launch_quant_f8( QuantF8Plan const & plan, void const * in, void const * gate, void * q, void * scale, void * values,
                     hipStream_t stream ) {
  if( plan.batch == 0 || plan.rows == 0 || plan.cols == 0 ) return ETIR_SUCCESS;
  if( in == nullptr || q == nullptr || scale == nullptr ) return fail( ETIR_NO_DATA_PTR_PROVIDED, "quant_f8: null tensor pointer" );
  QuantF8Args a{};
  a.in = in;
  a.gate = gate;
  a.q = q;
  a.scale = scale;
  a.values = values;
  a.ld_in = plan.ld_in;
  a.ld_gate = plan.ld_gate;
  a.ld_q = plan.ld_q;
  a.ld_values = plan.ld_values;
  a.rows = plan.block_rows == 1 ? plan.batch * plan.rows : plan.rows;
  a.cols = int32_t( plan.cols );
  a.ktype = plan.ktype;
  a.e8m0 = plan.dtype_scale == ETIR_E8M0;
  bool const l_e5m2 = plan.dtype_q == ETIR_F8E5M2;
  if( plan.dtype == ETIR_BF16 ) return l_e5m2 ? launch_type< uint16_t, true >( plan, a, stream ) : launch_type< uint16_t, false >( plan, a, stream );
  return l_e5m2 ? launch_type< float, true >( plan, a, stream ) : launch_type< float, false >( plan, a, stream );
}

}  // namespace etir
