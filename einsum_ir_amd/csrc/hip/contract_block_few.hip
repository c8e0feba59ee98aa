// gfx950 product of 8-bit floating point blocks, or of bf16, where the rows are
// few (tokens that are answered one at a time, groups of a few rows):
//
//   out[c][m][n] = last( sum_kb sa[c][m][kb] sb[c][n][kb] sum_(k in kb) A[c][m][k] B[c][n][k] + bias[c][n] )
//
// Bound by the bytes of B, each read once.  A workgroup takes 16 FB rows of A
// (of one group) and 16 / PARTS rows of B, and its waves split K.  PARTS 4 puts a
// quarter of K each into the 16 rows of a fragment, A's rows in fragments of 4, of
// which those products count whose quarters are the same: four times the
// workgroups where B has few rows.  Operands, unit-stride along k and at any
// address, go from global memory straight into the fragments of
// v_mfma_f32_16x16x32_bf16; 8-bit numbers become bf16 there, so that products are
// exact and sums fp32 (the conversions are hidden behind the loads).  A block's
// sum is scaled before the next begins.  The waves' sums meet in LDS and are
// added in their order.  Rows past a side's end read its last row and are not
// stored.  24 rows of 16 groups times 2048 x 2048 in bf16 take 15.4 us (20 with B not in
// the cache: the used groups' bytes at 4.6 TB/s), 1 row times 2048 x 2048 in 8 bits
// 3.8 (4.2), nearly all of it the launch.
#include "block_internal.h"
#include "contract_kernel.h"

namespace etir {
namespace {

typedef float    f32x4 __attribute__( ( ext_vector_type( 4 ) ) );
typedef uint32_t u32x4 __attribute__( ( ext_vector_type( 4 ) ) );
typedef u32x4    u32x4_dword __attribute__( ( aligned( 4 ) ) );
typedef __bf16   bf16x2 __attribute__( ( ext_vector_type( 2 ) ) );
typedef __bf16   bf16x8 __attribute__( ( ext_vector_type( 8 ) ) );

constexpr int kWaves = 8;       // of a workgroup, over K
constexpr int kLoads = 4;       // of 64 bytes of a row, in flight together
constexpr int kPiece = 64 * kLoads;

// 16 bytes of a row on their way.  OFF: at any address, read as the five aligned
// dwords that hold them (of which only those with a byte of the 16 are read) and
// shifted into place: 16-byte loads off a 4-byte boundary run at a third of the
// rate.  Else: at a multiple of 4.
// MASKED: K may end inside or before them; the row's last 16 bytes are then loaded
// in their place, and those that belong to an earlier piece, or to none, count as
// zeros.  bytes: of the row, at least 16.
template< bool OFF >
struct Load {
  u32x4    m_v;
  uint32_t m_w;
  int      m_shift, m_skip;

  template< bool MASKED >
  __device__ __attribute__( ( always_inline ) ) inline void load( uint8_t const * row, int64_t at, int64_t bytes ) {
    int64_t const l_at = MASKED ? min( at, bytes - 16 ) : at;
    m_skip = MASKED ? int( min( at - l_at, int64_t( 16 ) ) ) : 0;      // leading bytes that do not count
    uintptr_t const l_p = reinterpret_cast< uintptr_t >( row + l_at );
    if constexpr( OFF ) {
      m_v = *reinterpret_cast< u32x4_dword const * >( l_p & ~uintptr_t( 3 ) );
      m_w = *reinterpret_cast< uint32_t const * >( ( l_p + 15 ) & ~uintptr_t( 3 ) );
      m_shift = int( l_p & 3 );
    }
    else m_v = *reinterpret_cast< u32x4_dword const * >( l_p );
  }
  template< bool MASKED >
  __device__ __attribute__( ( always_inline ) ) inline u32x4 value() const {
    u32x4 l_v = m_v;
    if constexpr( OFF ) {
      l_v = u32x4{ __builtin_amdgcn_alignbyte( m_v[1], m_v[0], m_shift ), __builtin_amdgcn_alignbyte( m_v[2], m_v[1], m_shift ),
                   __builtin_amdgcn_alignbyte( m_v[3], m_v[2], m_shift ), __builtin_amdgcn_alignbyte( m_w, m_v[3], m_shift ) };
    }
    if constexpr( MASKED ) {
#pragma unroll
      for( int l_d = 0; l_d < 4; l_d++ ) {
        int const l_z = m_skip - 4 * l_d;
        l_v[l_d] &= l_z <= 0 ? 0xffffffffu : l_z >= 4 ? 0u : 0xffffffffu << ( 8 * l_z );
      }
    }
    return l_v;
  }
};

// half H of 16 8-bit numbers as bf16
template< bool E5M2, int H >
__device__ __attribute__( ( always_inline ) ) inline bf16x8 widen( u32x4 v ) {
  bf16x8 l_w;
#pragma unroll
  for( int l_i = 0; l_i < 2; l_i++ ) {
    int const l_d = int( v[2 * H + l_i] );
    bf16x2 l_lo, l_hi;
    if constexpr( E5M2 ) {
      l_lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8( l_d, 1.0f, false );
      l_hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8( l_d, 1.0f, true );
    }
    else {
      l_lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8( l_d, 1.0f, false );
      l_hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8( l_d, 1.0f, true );
    }
    l_w[4 * l_i] = l_lo[0];
    l_w[4 * l_i + 1] = l_lo[1];
    l_w[4 * l_i + 2] = l_hi[0];
    l_w[4 * l_i + 3] = l_hi[1];
  }
  return l_w;
}

__device__ inline float scale_at( void const * s, bool e8m0, int64_t at ) {
  return e8m0 ? e8m0_to_f32( static_cast< uint8_t const * >( s )[at] ) : static_cast< float const * >( s )[at];
}

template< bool F8, bool A_E5M2, int FB, int PARTS, bool OFF >
__global__ __launch_bounds__( 64 * kWaves )
void contract_block_few_kernel( BlockFast a ) {
  constexpr int ITEM = F8 ? 1 : 2;
  constexpr int MANY = 16 / PARTS, EACH = 16 / PARTS, FEW = EACH * FB;      // rows of B, of a fragment of A, of A
  constexpr int PITCH = MANY + 4;
  __shared__ __align__( 16 ) float l_part[kWaves * PARTS][FEW * PITCH];

  int const l_lane = threadIdx.x % 64;
  int const l_wave = __builtin_amdgcn_readfirstlane( threadIdx.x / 64 );
  int32_t const l_tiles_n = ( a.N + MANY - 1 ) / MANY;
  int64_t const l_cm = blockIdx.x / uint32_t( l_tiles_n );
  int32_t const l_n0 = int32_t( blockIdx.x % uint32_t( l_tiles_n ) ) * MANY;
  int32_t l_c, l_m0, l_m_end = a.M;
  if( a.has( BlockArgs::GROUP_ROWS ) ) {
    BlockRows const l_r = block_rows< FEW >( a.offsets(), a.groups(), a.M, int32_t( l_cm ) );
    if( l_r.group < 0 ) return;
    l_c = l_r.group;
    l_m0 = l_r.m0;
    l_m_end = l_r.end;
  }
  else {
    int32_t const l_tiles_m = ( a.M + FEW - 1 ) / FEW;
    l_m0 = int32_t( l_cm % l_tiles_m ) * FEW;
    l_c = int32_t( l_cm / l_tiles_m );
  }

  int const l_row = l_lane % EACH, l_of = l_lane % 16 / EACH;      // row of a fragment, part of K
  int64_t const l_bytes = int64_t( a.K ) * ITEM;
  int32_t const l_pieces = int32_t( ( l_bytes + kPiece * PARTS - 1 ) / ( kPiece * PARTS ) );      // of a part of K
  int32_t const l_n = min( l_n0 + l_row, a.N - 1 );
  uint8_t const * const l_b = static_cast< uint8_t const * >( a.b ) + ( l_c * int64_t( a.b_c ) + l_n * int64_t( a.b_ld ) ) * ITEM;
  uint8_t const * l_a[FB];
  int32_t l_m[FB];
#pragma unroll
  for( int l_i = 0; l_i < FB; l_i++ ) {
    l_m[l_i] = min( l_m0 + EACH * l_i + l_row, l_m_end - 1 );
    l_a[l_i] = static_cast< uint8_t const * >( a.a ) + ( l_c * a.a_batch() + l_m[l_i] * int64_t( a.a_ld ) ) * ITEM;
  }

  f32x4 l_acc[FB];
#pragma unroll
  for( int l_i = 0; l_i < FB; l_i++ ) l_acc[l_i] = f32x4{ 0.0f, 0.0f, 0.0f, 0.0f };
  bool const l_e8m0 = a.has( BlockArgs::E8M0 );

  auto step = [&]( int32_t piece, auto masked ) __attribute__( ( always_inline ) ) {
    // the lane's first byte: its part of K, its 16 of 64 bytes
    int64_t const l_at = ( int64_t( l_of ) * l_pieces + piece ) * kPiece + 16 * ( l_lane / 16 );
    constexpr bool MASKED = decltype( masked )::value;
    Load< OFF > l_lb[kLoads], l_la[kLoads][FB];
#pragma unroll
    for( int l_s = 0; l_s < kLoads; l_s++ ) {
      l_lb[l_s].template load< MASKED >( l_b, l_at + 64 * l_s, l_bytes );
#pragma unroll
      for( int l_i = 0; l_i < FB; l_i++ ) l_la[l_s][l_i].template load< MASKED >( l_a[l_i], l_at + 64 * l_s, l_bytes );
    }
    u32x4 l_vb[kLoads], l_va[kLoads][FB];
    auto values = [&]() __attribute__( ( always_inline ) ) {
#pragma unroll
      for( int l_s = 0; l_s < kLoads; l_s++ ) {
        l_vb[l_s] = l_lb[l_s].template value< MASKED >();
#pragma unroll
        for( int l_i = 0; l_i < FB; l_i++ ) l_va[l_s][l_i] = l_la[l_s][l_i].template value< MASKED >();
      }
    };
    if constexpr( !F8 ) {
      values();
#pragma unroll
      for( int l_s = 0; l_s < kLoads; l_s++ ) {
#pragma unroll
        for( int l_i = 0; l_i < FB; l_i++ ) {
          l_acc[l_i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16( __builtin_bit_cast( bf16x8, l_vb[l_s] ),
                                                                __builtin_bit_cast( bf16x8, l_va[l_s][l_i] ), l_acc[l_i], 0, 0, 0 );
        }
      }
    }
    else {
      // Blocks past the last have sums of 0 and scales of 0.  An accumulator holds rows 4 (lane / 16) + 0..3
      // of B, with parts those of one part, against row lane % 16 of A.
      float l_sb[kPiece / kScaleBlock][4], l_sa[kPiece / kScaleBlock][FB];
      int32_t const l_last = ( a.K - 1 ) / kScaleBlock;
      int64_t const l_first = ( int64_t( l_of ) * l_pieces + piece ) * ( kPiece / kScaleBlock );
#pragma unroll
      for( int l_k = 0; l_k < kPiece / kScaleBlock; l_k++ ) {
        int64_t const l_kb = min( l_first + l_k, int64_t( l_last ) );
        bool const l_past = MASKED && l_first + l_k > l_last;
#pragma unroll
        for( int l_i = 0; l_i < FB; l_i++ ) {
          l_sa[l_k][l_i] = a.sa == nullptr ? 1.0f : scale_at( a.sa, l_e8m0, l_c * int64_t( a.sa_c ) + l_kb * a.sa_k
                                                  + int64_t( a.has( BlockArgs::SA_BLOCKS ) ? l_m[l_i] / kScaleBlock : l_m[l_i] ) * a.sa_row );
        }
        if( a.sb == nullptr || a.has( BlockArgs::SB_BLOCKS ) ) {
          // a workgroup's rows of B are in one block
          l_sb[l_k][0] = a.sb == nullptr ? 1.0f : scale_at( a.sb, l_e8m0, l_c * int64_t( a.sb_c ) + l_kb * a.sb_k + int64_t( l_n0 / kScaleBlock ) * a.sb_row );
          l_sb[l_k][1] = l_sb[l_k][2] = l_sb[l_k][3] = l_sb[l_k][0];
        }
        else {
#pragma unroll
          for( int l_e = 0; l_e < 4; l_e++ ) {
            int32_t const l_r = min( l_n0 + ( PARTS > 1 ? l_e : 4 * ( l_lane / 16 ) + l_e ), a.N - 1 );
            l_sb[l_k][l_e] = scale_at( a.sb, l_e8m0, l_c * int64_t( a.sb_c ) + l_kb * a.sb_k + l_r * int64_t( a.sb_row ) );
          }
        }
        if( l_past ) {
#pragma unroll
          for( int l_i = 0; l_i < FB; l_i++ ) l_sa[l_k][l_i] = 0.0f;
#pragma unroll
          for( int l_e = 0; l_e < 4; l_e++ ) l_sb[l_k][l_e] = 0.0f;
        }
      }
      values();
#pragma unroll
      for( int l_k = 0; l_k < kPiece / kScaleBlock; l_k++ ) {
#pragma unroll
        for( int l_i = 0; l_i < FB; l_i++ ) {
          f32x4 l_p = { 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
          for( int l_s = 2 * l_k; l_s < 2 * l_k + 2; l_s++ ) {
            l_p = __builtin_amdgcn_mfma_f32_16x16x32_bf16( widen< false, 0 >( l_vb[l_s] ), widen< A_E5M2, 0 >( l_va[l_s][l_i] ), l_p, 0, 0, 0 );
            l_p = __builtin_amdgcn_mfma_f32_16x16x32_bf16( widen< false, 1 >( l_vb[l_s] ), widen< A_E5M2, 1 >( l_va[l_s][l_i] ), l_p, 0, 0, 0 );
          }
#pragma unroll
          for( int l_e = 0; l_e < 4; l_e++ ) l_acc[l_i][l_e] = fmaf( l_p[l_e], l_sa[l_k][l_i] * l_sb[l_k][l_e], l_acc[l_i][l_e] );
        }
      }
    }
  };
  // The waves take the pieces in turn, each workgroup from another one on, so
  // that workgroups in step do not all read the same part of their rows, which
  // lies in the same memory channels.
  int32_t const l_rot = l_pieces > 0 ? int32_t( blockIdx.x % uint32_t( l_pieces ) ) : 0;
  for( int32_t l_i = l_wave; l_i < l_pieces; l_i += kWaves ) {
    int32_t const l_p = l_i + l_rot < l_pieces ? l_i + l_rot : l_i + l_rot - l_pieces;
    if( ( l_p + 1 + ( PARTS - 1 ) * int64_t( l_pieces ) ) * kPiece <= l_bytes ) step( l_p, std::false_type() );
    else                                                                      step( l_p, std::true_type() );
  }

  // with parts those products count whose parts are the same
  if( PARTS == 1 || l_lane / 16 == l_of ) {
#pragma unroll
    for( int l_j = 0; l_j < FB; l_j++ ) {
      *reinterpret_cast< f32x4 * >( &l_part[l_wave * PARTS + ( PARTS > 1 ? l_of : 0 )]
                                           [( EACH * l_j + l_row ) * PITCH + ( PARTS > 1 ? 0 : 4 * ( l_lane / 16 ) )] ) = l_acc[l_j];
    }
  }
  __syncthreads();

  for( int l_e = threadIdx.x; l_e < MANY * FEW; l_e += 64 * kWaves ) {
    int const l_i = l_e % MANY, l_f = l_e / MANY;
    int32_t const l_ng = l_n0 + l_i, l_mg = l_m0 + l_f;
    if( l_ng >= a.N || l_mg >= l_m_end ) continue;
    float l_v = 0.0f;
#pragma unroll
    for( int l_w = 0; l_w < kWaves * PARTS; l_w++ ) l_v += l_part[l_w][l_f * PITCH + l_i];
    if( a.bias() ) l_v += a.bias()[l_ng];
    if( a.has( BlockArgs::RELU ) && l_v < 0.0f ) l_v = 0.0f;         // a NaN stays
    int64_t const l_o = l_c * int64_t( a.o_c ) + l_mg * int64_t( a.o_row ) + l_ng;
    if( a.has( BlockArgs::OUT_BF16 ) ) static_cast< uint16_t * >( a.out )[l_o] = kern::f32_to_bf16_rne( l_v );
    else                               static_cast< float * >( a.out )[l_o] = l_v;
  }
}

template< bool F8, bool A_E5M2, int FB, int PARTS, bool OFF >
void launch_shape( BlockArgs const & a, hipStream_t stream ) {
  constexpr int MANY = 16 / PARTS, FEW = MANY * FB;
  int64_t const l_tiles_n = ( int64_t( a.N ) + MANY - 1 ) / MANY;
  int64_t const l_tiles_m = a.has( BlockArgs::GROUP_ROWS ) ? block_most_tiles( a.M, a.C, FEW ) : ( int64_t( a.M ) + FEW - 1 ) / FEW * a.C;
  hipLaunchKernelGGL( ( contract_block_few_kernel< F8, A_E5M2, FB, PARTS, OFF > ), dim3( uint32_t( l_tiles_m * l_tiles_n ) ),
                      dim3( 64 * kWaves ), 0, stream, BlockFast::of( a, false, false ) );
}

template< bool F8, bool A_E5M2, bool OFF >
int launch_type( BlockArgs const & a, BlockKernel kernel, hipStream_t stream ) {
  switch( kernel ) {
    case BlockKernel::FEW_4:       launch_shape< F8, A_E5M2, 1, 4, OFF >( a, stream ); break;
    case BlockKernel::FEW_8_PARTS: launch_shape< F8, A_E5M2, 2, 4, OFF >( a, stream ); break;
    case BlockKernel::FEW_16:      launch_shape< F8, A_E5M2, 1, 1, OFF >( a, stream ); break;
    default:                       launch_shape< F8, A_E5M2, 2, 1, OFF >( a, stream ); break;
  }
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "contraction launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

}  // namespace

int launch_block_few( BlockArgs const & a, BlockKernel kernel, hipStream_t stream ) {
  int64_t const l_item = a.has( BlockArgs::F8 ) ? 1 : 2;
  auto off = [&]( void const * p, int64_t c, int64_t row ) { return ( uintptr_t( p ) | uintptr_t( c * l_item ) | uintptr_t( row * l_item ) ) % 4 != 0; };
  if( off( a.a, a.a_c, a.a_row ) || off( a.b, a.b_c, a.b_row ) || a.K * l_item % 4 != 0 ) {
    if( !a.has( BlockArgs::F8 ) ) return launch_type< false, false, true >( a, kernel, stream );
    return a.has( BlockArgs::A_E5M2 ) ? launch_type< true, true, true >( a, kernel, stream ) : launch_type< true, false, true >( a, kernel, stream );
  }
  if( !a.has( BlockArgs::F8 ) ) return launch_type< false, false, false >( a, kernel, stream );
  return a.has( BlockArgs::A_E5M2 ) ? launch_type< true, true, false >( a, kernel, stream ) : launch_type< true, false, false >( a, kernel, stream );
}

}  // namespace etir
