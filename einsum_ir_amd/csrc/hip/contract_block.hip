// gfx950 product of 8-bit floating point blocks, or of bf16, with or without
// groups, any strides:
//
//   out[c][m][n] = last( sum_kb sa[c][m][kb] sb[c][n][kb] sum_(k in kb) A[c][m][k] B[c][n][k] + bias[c][n] )
//
// One workgroup of 4 waves computes a 64 x 64 tile with
// v_mfma_f32_32x32x16_bf16 (a wave a 32 x 32 block), 64 k at a time through LDS.
// 8-bit numbers become bf16 on their way into LDS, which holds all of them
// exactly, so products are exact and sums are fp32.  Both 64-k halves of a block
// of 128 are summed before its scales are applied.  An operand that is
// unit-stride along k, or along its rows, is read in 16-byte pieces at any
// address, any other element by element with neighbouring lanes on neighbouring
// rows.  It is the kernel for layouts that the others do not take; the waits of
// its single buffer bound it.
#include "block_internal.h"
#include "contract_kernel.h"

namespace etir {
namespace {

typedef float    f32x16 __attribute__( ( ext_vector_type( 16 ) ) );
typedef __bf16   bf16x8 __attribute__( ( ext_vector_type( 8 ) ) );
typedef __bf16   bf16x2 __attribute__( ( ext_vector_type( 2 ) ) );
typedef uint32_t u32x4 __attribute__( ( ext_vector_type( 4 ) ) );
typedef u32x4    u32x4_u __attribute__( ( aligned( 1 ) ) );

constexpr int kTile  = 64;
constexpr int kBk    = 64;
constexpr int kPitch = kBk + 8;    // bf16 elements a row: 144 bytes, 16-byte reads of 16 rows over all banks

// how an operand lies
enum Lie : int { ALONG_K, ALONG_ROWS, APART };

// 16 elements as bf16 bits, two a dword
struct Piece { uint32_t w[8]; };

__device__ inline void put( Piece & p, int i, uint32_t bits ) { p.w[i / 2] |= bits << ( 16 * ( i % 2 ) ); }

// four 8-bit numbers to bf16
template< bool E5M2 >
__device__ inline void widen4( uint32_t v, uint32_t * to ) {
  bf16x2 l_lo, l_hi;
  if constexpr( E5M2 ) {
    l_lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8( int( v ), 1.0f, false );
    l_hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8( int( v ), 1.0f, true );
  }
  else {
    l_lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8( int( v ), 1.0f, false );
    l_hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8( int( v ), 1.0f, true );
  }
  to[0] = __builtin_bit_cast( uint32_t, l_lo );
  to[1] = __builtin_bit_cast( uint32_t, l_hi );
}

// 16 elements from p on with the given stride, of which the first n exist
template< bool F8, bool E5M2 >
__device__ inline Piece load16( uint8_t const * p, int64_t stride, int n ) {
  Piece l_p = {};
  if constexpr( F8 ) {
    uint32_t l_v[4] = { 0, 0, 0, 0 };
    if( stride == 1 && n >= 16 ) {
      u32x4 const l_r = *reinterpret_cast< u32x4_u const * >( p );
#pragma unroll
      for( int l_i = 0; l_i < 4; l_i++ ) l_v[l_i] = l_r[l_i];
    }
    else {
#pragma unroll
      for( int l_i = 0; l_i < 16; l_i++ ) if( l_i < n ) l_v[l_i / 4] |= uint32_t( p[l_i * stride] ) << ( 8 * ( l_i % 4 ) );
    }
#pragma unroll
    for( int l_i = 0; l_i < 4; l_i++ ) widen4< E5M2 >( l_v[l_i], l_p.w + 2 * l_i );
  }
  else {
    uint16_t const * l_q = reinterpret_cast< uint16_t const * >( p );
    if( stride == 1 && n >= 16 ) {
#pragma unroll
      for( int l_h = 0; l_h < 2; l_h++ ) {
        u32x4 const l_r = *reinterpret_cast< u32x4_u const * >( p + 16 * l_h );
#pragma unroll
        for( int l_i = 0; l_i < 4; l_i++ ) l_p.w[4 * l_h + l_i] = l_r[l_i];
      }
    }
    else {
#pragma unroll
      for( int l_i = 0; l_i < 16; l_i++ ) if( l_i < n ) put( l_p, l_i, l_q[l_i * stride] );
    }
  }
  return l_p;
}

// One operand's 64 rows x 64 k of a step into LDS as [row][k] of bf16, 16
// elements a thread.  base: the tile's first row at k = 0; rows and k past the
// tensor's count as zeros.
template< bool F8, bool E5M2 >
__device__ inline void stage( uint16_t * lds, uint8_t const * base, int64_t row, int64_t k, int rows, int32_t k0, int32_t K ) {
  constexpr int ITEM = F8 ? 1 : 2;
  int const l_t = threadIdx.x;
  Lie const l_lie = k == 1 ? ALONG_K : row == 1 ? ALONG_ROWS : APART;
  if( l_lie != ALONG_ROWS ) {
    int const l_r = l_lie == ALONG_K ? l_t / 4 : l_t % 64;
    int const l_k = 16 * ( l_lie == ALONG_K ? l_t % 4 : l_t / 64 );
    int const l_n = l_r < rows ? max( min( K - k0 - l_k, 16 ), 0 ) : 0;
    Piece l_p = {};
    if( l_n > 0 ) l_p = load16< F8, E5M2 >( base + ( l_r * row + int64_t( k0 + l_k ) * k ) * ITEM, k, l_n );
    u32x4 * const l_to = reinterpret_cast< u32x4 * >( lds + l_r * kPitch + l_k );
    l_to[0] = u32x4{ l_p.w[0], l_p.w[1], l_p.w[2], l_p.w[3] };
    l_to[1] = u32x4{ l_p.w[4], l_p.w[5], l_p.w[6], l_p.w[7] };
  }
  else {
    int const l_k = l_t / 4, l_r = 16 * ( l_t % 4 );
    int const l_n = k0 + l_k < K ? max( min( rows - l_r, 16 ), 0 ) : 0;
    Piece l_p = {};
    if( l_n > 0 ) l_p = load16< F8, E5M2 >( base + ( l_r + int64_t( k0 + l_k ) * k ) * ITEM, 1, l_n );
#pragma unroll
    for( int l_i = 0; l_i < 16; l_i++ ) lds[( l_r + l_i ) * kPitch + l_k] = uint16_t( l_p.w[l_i / 2] >> ( 16 * ( l_i % 2 ) ) );
  }
}

__device__ inline float scale_at( void const * s, bool e8m0, int64_t at ) {
  return e8m0 ? e8m0_to_f32( static_cast< uint8_t const * >( s )[at] ) : static_cast< float const * >( s )[at];
}

template< bool F8, bool A_E5M2 >
__global__ __launch_bounds__( 256 )
void contract_block_general_kernel( BlockArgs a ) {
  constexpr int ITEM = F8 ? 1 : 2;
  constexpr int PITCH_OUT = kTile + 1;
  __shared__ __align__( 16 ) char l_lds[kTile * PITCH_OUT * 4 > 4 * kTile * kPitch ? kTile * PITCH_OUT * 4 : 4 * kTile * kPitch];
  __shared__ float l_sa[kTile], l_sb[kTile];
  uint16_t * const l_lds_a = reinterpret_cast< uint16_t * >( l_lds );
  uint16_t * const l_lds_b = l_lds_a + kTile * kPitch;

  int const l_t = threadIdx.x;
  int32_t const l_tiles_n = ( a.N + kTile - 1 ) / kTile;
  int64_t const l_id = blockIdx.x;
  int32_t const l_n0 = int32_t( l_id % l_tiles_n ) * kTile;
  int32_t l_c, l_m0, l_m_end = a.M, l_k_begin = 0, l_K = a.K;
  if( a.has( BlockArgs::GROUP_ROWS ) ) {
    BlockRows const l_r = block_rows< kTile >( a.offsets, a.C, a.M, int32_t( l_id / l_tiles_n ) );
    if( l_r.group < 0 ) return;
    l_c = l_r.group;
    l_m0 = l_r.m0;
    l_m_end = l_r.end;
  }
  else {
    int32_t const l_tiles_m = ( a.M + kTile - 1 ) / kTile;
    int64_t const l_cm = l_id / l_tiles_n;
    l_m0 = int32_t( l_cm % l_tiles_m ) * kTile;
    l_c = int32_t( l_cm / l_tiles_m );
    if( a.has( BlockArgs::GROUP_K ) ) {
      BlockGroup const l_g = block_group( a.offsets, l_c, a.K );
      l_k_begin = l_g.begin;
      l_K = l_g.end - l_g.begin;
    }
  }
  int const l_rows = min( kTile, l_m_end - l_m0 ), l_cols = min( kTile, a.N - l_n0 );
  uint8_t const * const l_a = static_cast< uint8_t const * >( a.a ) + ( l_c * a.a_c + l_m0 * a.a_row + l_k_begin * a.a_k ) * ITEM;
  uint8_t const * const l_b = static_cast< uint8_t const * >( a.b ) + ( l_c * a.b_c + l_n0 * a.b_row + l_k_begin * a.b_k ) * ITEM;

  int const l_wave = l_t / 64, l_lane = l_t % 64;
  int const l_wm = 32 * ( l_wave / 2 ), l_wn = 32 * ( l_wave % 2 );
  f32x16 l_acc = { 0 }, l_part = { 0 };
  for( int32_t l_k0 = 0; l_k0 < l_K; l_k0 += kBk ) {
    stage< F8, A_E5M2 >( l_lds_a, l_a, a.a_row, a.a_k, l_rows, l_k0, l_K );
    stage< F8, false >( l_lds_b, l_b, a.b_row, a.b_k, l_cols, l_k0, l_K );
    bool const l_first = l_k0 % kScaleBlock == 0;
    if( F8 && l_first && l_t < 2 * kTile ) {
      // rows past the tensor take the last one's scale and are not stored
      int32_t const l_kb = l_k0 / kScaleBlock;
      if( l_t < kTile ) {
        int64_t const l_m = l_m0 + min( l_t, l_rows - 1 );
        l_sa[l_t] = a.sa == nullptr ? 1.0f : scale_at( a.sa, a.has( BlockArgs::E8M0 ), l_c * a.sa_c + l_kb * a.sa_k
                                       + ( a.has( BlockArgs::SA_BLOCKS ) ? l_m / kScaleBlock : l_m ) * a.sa_row );
      }
      else {
        int64_t const l_n = l_n0 + min( l_t - kTile, l_cols - 1 );
        l_sb[l_t - kTile] = a.sb == nullptr ? 1.0f : scale_at( a.sb, a.has( BlockArgs::E8M0 ), l_c * a.sb_c + l_kb * a.sb_k
                                       + ( a.has( BlockArgs::SB_BLOCKS ) ? l_n / kScaleBlock : l_n ) * a.sb_row );
      }
    }
    __syncthreads();
    // the columns' side first: a lane holds one row m and 16 columns
    f32x16 l_sum = { 0 };
    if( !F8 ) l_sum = l_acc;
    else if( !l_first ) l_sum = l_part;
#pragma unroll
    for( int l_s = 0; l_s < kBk / 16; l_s++ ) {
      int const l_k = 16 * l_s + 8 * ( l_lane / 32 );
      bf16x8 const l_fa = *reinterpret_cast< bf16x8 const * >( l_lds_a + ( l_wm + l_lane % 32 ) * kPitch + l_k );
      bf16x8 const l_fb = *reinterpret_cast< bf16x8 const * >( l_lds_b + ( l_wn + l_lane % 32 ) * kPitch + l_k );
      l_sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16( l_fb, l_fa, l_sum, 0, 0, 0 );
    }
    if( !F8 ) l_acc = l_sum;
    else {
      l_part = l_sum;
      if( !l_first || l_k0 + kBk >= l_K ) {
        float const l_s = l_sa[l_wm + l_lane % 32];
#pragma unroll
        for( int l_i = 0; l_i < 16; l_i++ ) {
          l_acc[l_i] += l_part[l_i] * ( l_s * l_sb[l_wn + 8 * ( l_i / 4 ) + 4 * ( l_lane / 32 ) + l_i % 4] );
        }
      }
    }
    __syncthreads();
  }

  // out through LDS, neighbouring lanes on the output's shorter stride
  float * const l_out = reinterpret_cast< float * >( l_lds );
#pragma unroll
  for( int l_i = 0; l_i < 16; l_i++ ) {
    l_out[( l_wm + l_lane % 32 ) * PITCH_OUT + l_wn + 8 * ( l_i / 4 ) + 4 * ( l_lane / 32 ) + l_i % 4] = l_acc[l_i];
  }
  __syncthreads();
  bool const l_along_n = a.o_col <= a.o_row;
  for( int l_e = l_t; l_e < kTile * kTile; l_e += 256 ) {
    int const l_m = l_along_n ? l_e / kTile : l_e % kTile, l_n = l_along_n ? l_e % kTile : l_e / kTile;
    if( l_m >= l_rows || l_n >= l_cols ) continue;
    float l_v = l_out[l_m * PITCH_OUT + l_n];
    if( a.bias ) l_v += a.bias[l_c * a.bias_c + ( l_n0 + l_n ) * a.bias_col];
    if( a.has( BlockArgs::RELU ) && l_v < 0.0f ) l_v = 0.0f;         // a NaN stays
    int64_t const l_o = l_c * a.o_c + ( l_m0 + l_m ) * a.o_row + ( l_n0 + l_n ) * a.o_col;
    if( a.has( BlockArgs::OUT_BF16 ) ) static_cast< uint16_t * >( a.out )[l_o] = kern::f32_to_bf16_rne( l_v );
    else                               static_cast< float * >( a.out )[l_o] = l_v;
  }
}

}  // namespace

int launch_block_general( BlockArgs const & a, hipStream_t stream ) {
  int64_t const l_tiles_n = ( int64_t( a.N ) + kTile - 1 ) / kTile;
  int64_t const l_tiles_m = a.has( BlockArgs::GROUP_ROWS ) ? block_most_tiles( a.M, a.C, kTile )
                                                           : ( int64_t( a.M ) + kTile - 1 ) / kTile * a.C;
  dim3 const l_grid( uint32_t( l_tiles_m * l_tiles_n ) );
  if( !a.has( BlockArgs::F8 ) )         hipLaunchKernelGGL( ( contract_block_general_kernel< false, false > ), l_grid, dim3( 256 ), 0, stream, a );
  else if( a.has( BlockArgs::A_E5M2 ) ) hipLaunchKernelGGL( ( contract_block_general_kernel< true, true > ), l_grid, dim3( 256 ), 0, stream, a );
  else                                  hipLaunchKernelGGL( ( contract_block_general_kernel< true, false > ), l_grid, dim3( 256 ), 0, stream, a );
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "contraction launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

}  // namespace etir
