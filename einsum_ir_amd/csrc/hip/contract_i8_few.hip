// gfx950 product of 8-bit integers where one side has few rows (tokens that are
// answered one at a time, or a handful of channels):
//
//   out[c][many][few] = last( s s sum_k MANY[c][many][k] FEW[c][few][k] + bias )
//
// Bound by the bytes of the many side, each read once.  A workgroup takes
// 16 rows of it and all of the few side (16 FB rows), and its waves split K;
// with up to 16 few rows it may take 4 rows of it instead and put a quarter of K
// each into the 16 rows of a fragment, the few side in fragments of 4 rows, of
// which those products count whose quarters are the same (PARTS 4: four times
// the workgroups for a short many side): that keeps all of a workgroup's bytes
// in flight at once where there are few workgroups, and needs no memory between
// workgroups.  Operands go from global
// memory straight into the fragments of v_mfma_i32_16x16x64_i8 (16 k of a row a
// lane, 4 lanes a row), at any byte address; the partial sums meet in LDS,
// where their order cannot change an integer sum.  Rows past a side's end read
// its last row and are not stored.
#include "i8_internal.h"
#include "contract_kernel.h"
#include <utility>

namespace etir {
namespace {

typedef int32_t i32x4 __attribute__( ( ext_vector_type( 4 ) ) );

constexpr int kSteps = 4;      // steps of 64 k whose loads are in flight together
constexpr int kPiece = 64 * kSteps;
constexpr int kWaves = 8;      // of a workgroup, over K

template< int FB, int PARTS, bool BYTES >
__global__ __launch_bounds__( 64 * kWaves )
void contract_i8_few_kernel( I8Args a ) {     // A: the many side
  constexpr int MANY = 16 / PARTS, FEW = 16 * FB / PARTS;   // rows of a workgroup
  constexpr int PITCH = MANY + 4;                           // 16-byte writes of the few rows over all banks
  __shared__ __align__( 16 ) int32_t l_part[kWaves * PARTS][FEW * PITCH];

  int const l_lane = threadIdx.x % 64;
  int const l_wave = __builtin_amdgcn_readfirstlane( threadIdx.x / 64 );
  int32_t const l_k = a.K();
  int32_t const l_tiles = ( a.M + MANY - 1 ) / MANY;
  int32_t const l_pieces = ( l_k + kPiece * PARTS - 1 ) / ( kPiece * PARTS );      // of a part of K
  int64_t const l_c = blockIdx.x / l_tiles;
  int32_t const l_m0 = ( blockIdx.x % l_tiles ) * MANY;
  int const l_row = l_lane % MANY, l_part_k = l_lane % 16 / MANY;
  int32_t const l_kl = 16 * ( l_lane / 16 ) + l_part_k * l_pieces * kPiece;

  int8_t const * const l_pm = a.a + l_c * a.c[I8_A] + int64_t( min( l_m0 + l_row, a.M - 1 ) ) * a.a_row;
  int8_t const * l_pf[FB];
#pragma unroll
  for( int l_i = 0; l_i < FB; l_i++ ) {
    l_pf[l_i] = a.b + l_c * a.c[I8_B] + int64_t( min( MANY * l_i + l_row, a.N - 1 ) ) * a.b_col;
  }

  i32x4 l_acc[FB];
#pragma unroll
  for( int l_i = 0; l_i < FB; l_i++ ) l_acc[l_i] = i32x4{ 0, 0, 0, 0 };

  auto step = [&]( int32_t k0, auto masked ) __attribute__( ( always_inline ) ) {
    I8Vec< BYTES > l_fm[kSteps], l_ff[kSteps][FB];
#pragma unroll
    for( int l_s = 0; l_s < kSteps; l_s++ ) {
      int32_t const l_ks = k0 + 64 * l_s + l_kl;
      int32_t const l_at = decltype( masked )::value ? i8_piece( l_ks, l_k ).at : l_ks;
      l_fm[l_s].load( l_pm + l_at );
#pragma unroll
      for( int l_i = 0; l_i < FB; l_i++ ) l_ff[l_s][l_i].load( l_pf[l_i] + l_at );
    }
#pragma unroll
    for( int l_s = 0; l_s < kSteps; l_s++ ) {
      i32x4 l_m = l_fm[l_s].value();
      if constexpr( decltype( masked )::value ) {
        int32_t const l_skip = i8_piece( k0 + 64 * l_s + l_kl, l_k ).skip;
#pragma unroll
        for( int l_d = 0; l_d < 4; l_d++ ) l_m[l_d] &= int32_t( i8_mask( l_skip, l_d ) );
      }
#pragma unroll
      for( int l_i = 0; l_i < FB; l_i++ ) {
        l_acc[l_i] = __builtin_amdgcn_mfma_i32_16x16x64_i8( l_m, l_ff[l_s][l_i].value(), l_acc[l_i], 0, 0, 0 );
      }
    }
  };
  // The waves take the pieces of kPiece k in turn, each workgroup from another
  // one on, so that workgroups in step do not all read the same part of their
  // rows, which lies in the same memory channels: 4096 x 4096 by one token
  // 5.8 us, without 6.3.
  int32_t const l_rot = int32_t( blockIdx.x % uint32_t( l_pieces ) );
  for( int32_t l_i = l_wave; l_i < l_pieces; l_i += kWaves ) {
    int32_t const l_p = l_i + l_rot < l_pieces ? l_i + l_rot : l_i + l_rot - l_pieces;
    if( ( l_p + 1 + ( PARTS - 1 ) * l_pieces ) * kPiece <= l_k ) step( l_p * kPiece, std::false_type() );
    else                              step( l_p * kPiece, std::true_type() );
  }

  // the accumulators hold rows 4 (lane / 16) + 0..3 of A against row lane % 16
  // of B; with parts those of the same part count
  if( PARTS == 1 || l_lane / 16 == l_part_k ) {
#pragma unroll
    for( int l_j = 0; l_j < FB; l_j++ ) {
      *reinterpret_cast< i32x4 * >( &l_part[l_wave * PARTS + ( PARTS > 1 ? l_part_k : 0 )]
                                           [( MANY * l_j + l_row ) * PITCH + ( PARTS > 1 ? 0 : 4 * ( l_lane / 16 ) )] ) = l_acc[l_j];
    }
  }
  __syncthreads();

  bool const l_along_many = a.o_row <= a.o_col;     // neighbouring lanes on neighbouring outputs
  for( int l_e = threadIdx.x; l_e < MANY * FEW; l_e += 64 * kWaves ) {
    int const l_m = l_along_many ? l_e % MANY : l_e / FEW;
    int const l_f = l_along_many ? l_e / MANY : l_e % FEW;
    int32_t const l_mg = l_m0 + l_m;
    if( l_mg >= a.M || l_f >= a.N ) continue;
    int32_t l_sum = 0;
#pragma unroll
    for( int l_w = 0; l_w < kWaves * PARTS; l_w++ ) l_sum += l_part[l_w][l_f * PITCH + l_m];
    float const l_sm = a.sa ? a.sa[l_c * a.c[I8_SA] + int64_t( l_mg ) * a.sa_row] : 1.0f;
    float const l_sf = a.sb ? a.sb[l_c * a.c[I8_SB] + int64_t( l_f ) * a.sb_col] : 1.0f;
    float const l_b = a.bias ? a.bias[l_c * a.c[I8_BIAS] + int64_t( a.has( I8Args::BIAS_ROWS ) ? l_mg : l_f ) * a.bias_step] : 0.0f;
    float const l_v = i8_finish( l_sum, l_sf, l_sm, l_b, a.has( I8Args::RELU ) );
    int64_t const l_o = l_c * a.c[I8_OUT] + int64_t( l_mg ) * a.o_row + int64_t( l_f ) * a.o_col;
    if( a.has( I8Args::OUT_BF16 ) ) static_cast< uint16_t * >( a.out )[l_o] = kern::f32_to_bf16_rne( l_v );
    else                            static_cast< float * >( a.out )[l_o] = l_v;
  }
}

template< int FB, int PARTS, bool BYTES >
int launch_shape( I8Args const & a, int64_t C, hipStream_t stream ) {
  constexpr int MANY = 16 / PARTS;
  hipLaunchKernelGGL( ( contract_i8_few_kernel< FB, PARTS, BYTES > ), dim3( uint32_t( ( a.M + MANY - 1 ) / MANY * C ) ),
                      dim3( 64 * kWaves ), 0, stream, a );
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "contraction_i8 launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

}  // namespace

int launch_i8_few( I8Args const & args, int64_t C, I8Kernel kernel, hipStream_t stream ) {
  I8Args a = args;
  if( a.M <= a.N ) {
    // the few side is A: A and B change places
    std::swap( a.a, a.b );
    std::swap( a.sa, a.sb );
    std::swap( a.M, a.N );
    std::swap( a.a_row, a.b_col );
    std::swap( a.o_row, a.o_col );
    std::swap( a.sa_row, a.sb_col );
    std::swap( a.c[I8_A], a.c[I8_B] );
    std::swap( a.c[I8_SA], a.c[I8_SB] );
    a.k_flags ^= I8Args::BIAS_ROWS;
  }
  bool const l_bytes = !i8_aligned( a, 4 );
  switch( kernel ) {
    case I8Kernel::FEW_4:
      return l_bytes ? launch_shape< 1, 4, true >( a, C, stream ) : launch_shape< 1, 4, false >( a, C, stream );
    case I8Kernel::FEW_8_PARTS:
      return l_bytes ? launch_shape< 2, 4, true >( a, C, stream ) : launch_shape< 2, 4, false >( a, C, stream );
    case I8Kernel::FEW_16_PARTS:
      return l_bytes ? launch_shape< 4, 4, true >( a, C, stream ) : launch_shape< 4, 4, false >( a, C, stream );
    case I8Kernel::FEW_16:
      return l_bytes ? launch_shape< 1, 1, true >( a, C, stream ) : launch_shape< 1, 1, false >( a, C, stream );
    default:
      return l_bytes ? launch_shape< 2, 1, true >( a, C, stream ) : launch_shape< 2, 1, false >( a, C, stream );
  }
}

}  // namespace etir
