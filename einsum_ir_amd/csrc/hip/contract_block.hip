// gfx950 product of 8-bit floating point blocks, or of bf16, with or without
// groups, any strides:
//
//   out[c][m][n] = last( sum_kb sa[c][m][kb] sb[c][n][kb] sum_(k in kb) A[c][m][k] B[c][n][k] + bias[c][n] )
//
// One workgroup of 4 waves computes a 64 x 64 tile with
// v_mfma_f32_32x32x16_bf16 (a wave a 32 x 32 block), 128 k at a time through LDS,
// the next 128 on their way in registers meanwhile (509 x 1001 x 333 in 5 groups
// 19.5 -> 18.9 us).  8-bit numbers become bf16 on their way into LDS, which holds
// all of them exactly, so products are exact and sums are fp32.  An operand that is
// unit-stride along k, or along its rows, is read in 16-byte pieces at any
// address, any other element by element with neighbouring lanes on neighbouring
// rows.  It is the kernel for layouts that the others do not take.
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
constexpr int kBk    = 128;        // of 8-bit numbers: one block
constexpr int kPitch = kBk + 8;    // bf16 elements a row: 272 bytes, 16-byte reads of 16 rows over all banks

// how an operand lies
enum Lie : int { ALONG_K, ALONG_ROWS, APART };

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

// 16 elements as they lie in memory
template< bool F8 > struct Piece { uint32_t w[F8 ? 4 : 8]; };

// 16 elements from p on with the given stride, of which the first n exist
template< bool F8 >
__device__ inline Piece< F8 > load16( uint8_t const * p, int64_t stride, int n ) {
  constexpr int WORDS = F8 ? 4 : 8;
  Piece< F8 > l_p = {};
  if( stride == 1 && n >= 16 ) {
#pragma unroll
    for( int l_h = 0; l_h < WORDS / 4; l_h++ ) {
      u32x4 const l_r = *reinterpret_cast< u32x4_u const * >( p + 16 * l_h );
#pragma unroll
      for( int l_i = 0; l_i < 4; l_i++ ) l_p.w[4 * l_h + l_i] = l_r[l_i];
    }
    return l_p;
  }
#pragma unroll
  for( int l_i = 0; l_i < 16; l_i++ ) {
    if( l_i >= n ) continue;
    if constexpr( F8 ) l_p.w[l_i / 4] |= uint32_t( p[l_i * stride] ) << ( 8 * ( l_i % 4 ) );
    else l_p.w[l_i / 2] |= uint32_t( reinterpret_cast< uint16_t const * >( p )[l_i * stride] ) << ( 16 * ( l_i % 2 ) );
  }
  return l_p;
}

// One operand's 64 rows x 128 k of a step: 32 elements a thread, from global
// memory into registers and from there into LDS as [row][k] of bf16.  Rows and k
// past the tensor's count as zeros.
template< bool F8, bool E5M2 >
struct Side {
  static constexpr int ITEM = F8 ? 1 : 2;
  uint8_t const * m_base;      // the tile's first row at k = 0
  int64_t m_row, m_k;
  int     m_rows;
  Lie     m_lie;
  Piece< F8 > m_p[2];

  __device__ inline void init( uint8_t const * base, int64_t row, int64_t k, int rows ) {
    m_base = base;
    m_row = row;
    m_k = k;
    m_rows = rows;
    m_lie = k == 1 ? ALONG_K : row == 1 ? ALONG_ROWS : APART;
  }
  __device__ inline void load( int32_t k0, int32_t K ) {
    int const l_t = threadIdx.x;
#pragma unroll
    for( int l_h = 0; l_h < 2; l_h++ ) {
      int l_r, l_k, l_n;
      if( m_lie == ALONG_ROWS ) {
        l_k = l_t / 2;
        l_r = 32 * ( l_t % 2 ) + 16 * l_h;
        l_n = k0 + l_k < K ? min( m_rows - l_r, 16 ) : 0;
      }
      else {
        l_r = m_lie == ALONG_K ? l_t / 4 : l_t % 64;
        l_k = 32 * ( m_lie == ALONG_K ? l_t % 4 : l_t / 64 ) + 16 * l_h;
        l_n = l_r < m_rows ? min( K - k0 - l_k, 16 ) : 0;
      }
      m_p[l_h] = Piece< F8 >{};
      if( l_n > 0 ) {
        m_p[l_h] = load16< F8 >( m_base + ( l_r * m_row + int64_t( k0 + l_k ) * m_k ) * ITEM, m_lie == ALONG_ROWS ? 1 : m_k, l_n );
      }
    }
  }
  __device__ inline void store( uint16_t * lds ) const {
    int const l_t = threadIdx.x;
#pragma unroll
    for( int l_h = 0; l_h < 2; l_h++ ) {
      uint32_t l_w[8];
#pragma unroll
      for( int l_i = 0; l_i < ( F8 ? 4 : 8 ); l_i++ ) {
        if constexpr( F8 ) widen4< E5M2 >( m_p[l_h].w[l_i], l_w + 2 * l_i );
        else               l_w[l_i] = m_p[l_h].w[l_i];
      }
      if( m_lie == ALONG_ROWS ) {
        int const l_k = l_t / 2, l_r = 32 * ( l_t % 2 ) + 16 * l_h;
#pragma unroll
        for( int l_i = 0; l_i < 16; l_i++ ) lds[( l_r + l_i ) * kPitch + l_k] = uint16_t( l_w[l_i / 2] >> ( 16 * ( l_i % 2 ) ) );
      }
      else {
        int const l_r = m_lie == ALONG_K ? l_t / 4 : l_t % 64;
        int const l_k = 32 * ( m_lie == ALONG_K ? l_t % 4 : l_t / 64 ) + 16 * l_h;
        u32x4 * const l_to = reinterpret_cast< u32x4 * >( lds + l_r * kPitch + l_k );
        l_to[0] = u32x4{ l_w[0], l_w[1], l_w[2], l_w[3] };
        l_to[1] = u32x4{ l_w[4], l_w[5], l_w[6], l_w[7] };
      }
    }
  }
};

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
  uint32_t const l_id = blockIdx.x;
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
  Side< F8, A_E5M2 > l_side_a;
  Side< F8, false > l_side_b;
  l_side_a.init( l_a, a.a_row, a.a_k, l_rows );
  l_side_b.init( l_b, a.b_row, a.b_k, l_cols );
  // the scale of a row or column of the tile, by a thread of its own
  float l_scale = 1.0f;
  auto load = [&]( int32_t k0 ) {
    l_side_a.load( k0, l_K );
    l_side_b.load( k0, l_K );
    if( !F8 || l_t >= 2 * kTile ) return;
    // rows past the tensor take the last one's scale and are not stored
    int32_t const l_kb = k0 / kScaleBlock;
    if( l_t < kTile ) {
      int64_t const l_m = l_m0 + min( l_t, l_rows - 1 );
      if( a.sa != nullptr ) l_scale = scale_at( a.sa, a.has( BlockArgs::E8M0 ), l_c * a.sa_c + l_kb * a.sa_k
                                               + ( a.has( BlockArgs::SA_BLOCKS ) ? l_m / kScaleBlock : l_m ) * a.sa_row );
    }
    else {
      int64_t const l_n = l_n0 + min( l_t - kTile, l_cols - 1 );
      if( a.sb != nullptr ) l_scale = scale_at( a.sb, a.has( BlockArgs::E8M0 ), l_c * a.sb_c + l_kb * a.sb_k
                                               + ( a.has( BlockArgs::SB_BLOCKS ) ? l_n / kScaleBlock : l_n ) * a.sb_row );
    }
  };
  f32x16 l_acc = { 0 };
  if( l_K > 0 ) load( 0 );
  for( int32_t l_k0 = 0; l_k0 < l_K; l_k0 += kBk ) {
    __syncthreads();         // the last step's fragments are read
    l_side_a.store( l_lds_a );
    l_side_b.store( l_lds_b );
    if( F8 && l_t < 2 * kTile ) ( l_t < kTile ? l_sa : l_sb - kTile )[l_t] = l_scale;
    __syncthreads();
    if( l_K - l_k0 > kBk ) load( l_k0 + kBk );
    // the columns' side first: a lane holds one row m and 16 columns
    f32x16 l_sum = { 0 };
    if( !F8 ) l_sum = l_acc;
#pragma unroll
    for( int l_s = 0; l_s < kBk / 16; l_s++ ) {
      int const l_k = 16 * l_s + 8 * ( l_lane / 32 );
      bf16x8 const l_fa = *reinterpret_cast< bf16x8 const * >( l_lds_a + ( l_wm + l_lane % 32 ) * kPitch + l_k );
      bf16x8 const l_fb = *reinterpret_cast< bf16x8 const * >( l_lds_b + ( l_wn + l_lane % 32 ) * kPitch + l_k );
      l_sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16( l_fb, l_fa, l_sum, 0, 0, 0 );
    }
    if( !F8 ) l_acc = l_sum;
    else {
      float const l_s = l_sa[l_wm + l_lane % 32];
#pragma unroll
      for( int l_i = 0; l_i < 16; l_i++ ) {
        l_acc[l_i] += l_sum[l_i] * ( l_s * l_sb[l_wn + 8 * ( l_i / 4 ) + 4 * ( l_lane / 32 ) + l_i % 4] );
      }
    }
  }
  __syncthreads();

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
