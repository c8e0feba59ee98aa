// gfx950 product of 8-bit integers where one side has few rows (tokens that are
// answered one at a time, or a handful of channels):
//
//   out[c][many][few] = last( s s sum_k MANY[c][many][k] FEW[c][few][k] + bias )
//
// Bound by the bytes of the many side, each read once.  A workgroup takes
// 16 rows of it and all of the few side (16 FB rows), and its waves split K:
// that keeps all of a workgroup's bytes in flight at once where there are few
// workgroups, and needs no memory between workgroups.  Operands go from global
// memory straight into the fragments of v_mfma_i32_16x16x64_i8 (16 k of a row a
// lane, 4 lanes a row), at any byte address; the partial sums meet in LDS,
// where their order cannot change an integer sum.  Rows past a side's end read
// its last row and are not stored.
#include "i8_internal.h"
#include "contract_kernel.h"

namespace etir {
namespace {

typedef int32_t i32x4 __attribute__( ( ext_vector_type( 4 ) ) );

struct FewArgs {
  int8_t const * many;
  int8_t const * few;
  float const  * s_many;
  float const  * s_few;
  float const  * bias;
  void         * out;
  int32_t n_many, n_few, K, pieces, tiles;
  int64_t many_row, few_row, o_many, o_few, sm_row, sf_row, bias_many, bias_few;
  int64_t c_many, c_few, c_out, c_sm, c_sf, c_bias;
  int32_t out_bf16, relu;
};

constexpr int kSteps = 4;      // steps of 64 k whose loads are in flight together
constexpr int kPiece = 64 * kSteps;
constexpr int kWaves = 8;      // of a workgroup, over K
constexpr int kMany  = 16;     // rows of the many side a workgroup

template< int FB, bool BYTES >
__global__ __launch_bounds__( 64 * kWaves )
void contract_i8_few_kernel( FewArgs a ) {
  constexpr int FEW = 16 * FB;
  constexpr int PITCH = kMany + 4;                       // 16-byte writes of 16 few rows over all banks
  __shared__ __align__( 16 ) int32_t l_part[kWaves][FEW * PITCH];

  int const l_lane = threadIdx.x % 64;
  int const l_wave = __builtin_amdgcn_readfirstlane( threadIdx.x / 64 );
  int const l_c = blockIdx.x / a.tiles;
  int const l_m0 = ( blockIdx.x % a.tiles ) * kMany;
  int const l_kl = 16 * ( l_lane / 16 );

  int8_t const * const l_pm = a.many + l_c * a.c_many + min( l_m0 + l_lane % 16, a.n_many - 1 ) * a.many_row;
  int8_t const * l_pf[FB];
#pragma unroll
  for( int l_i = 0; l_i < FB; l_i++ ) {
    l_pf[l_i] = a.few + l_c * a.c_few + min( 16 * l_i + l_lane % 16, a.n_few - 1 ) * a.few_row;
  }

  i32x4 l_acc[FB];
#pragma unroll
  for( int l_i = 0; l_i < FB; l_i++ ) l_acc[l_i] = i32x4{ 0, 0, 0, 0 };

  auto step = [&]( int32_t k0, auto masked ) __attribute__( ( always_inline ) ) {
    I8Vec< BYTES > l_fm[kSteps], l_ff[kSteps][FB];
#pragma unroll
    for( int l_s = 0; l_s < kSteps; l_s++ ) {
      int32_t const l_k = k0 + 64 * l_s + l_kl;
      int32_t const l_at = decltype( masked )::value ? i8_piece( l_k, a.K ).at : l_k;
      l_fm[l_s].load( l_pm + l_at );
#pragma unroll
      for( int l_i = 0; l_i < FB; l_i++ ) l_ff[l_s][l_i].load( l_pf[l_i] + l_at );
    }
#pragma unroll
    for( int l_s = 0; l_s < kSteps; l_s++ ) {
      i32x4 l_m = l_fm[l_s].value();
      if constexpr( decltype( masked )::value ) {
        int32_t const l_skip = i8_piece( k0 + 64 * l_s + l_kl, a.K ).skip;
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
  int32_t const l_rot = int32_t( blockIdx.x % uint32_t( a.pieces ) );
  for( int32_t l_i = l_wave; l_i < a.pieces; l_i += kWaves ) {
    int32_t const l_p = l_i + l_rot < a.pieces ? l_i + l_rot : l_i + l_rot - a.pieces;
    if( ( l_p + 1 ) * kPiece <= a.K ) step( l_p * kPiece, std::false_type() );
    else                              step( l_p * kPiece, std::true_type() );
  }

  // the accumulators hold many rows 4 (lane / 16) + 0..3 of few row lane % 16
#pragma unroll
  for( int l_j = 0; l_j < FB; l_j++ ) {
    *reinterpret_cast< i32x4 * >( &l_part[l_wave][( 16 * l_j + l_lane % 16 ) * PITCH + 4 * ( l_lane / 16 )] ) = l_acc[l_j];
  }
  __syncthreads();

  int const l_rows = min( kMany, a.n_many - l_m0 );
  bool const l_along_many = a.o_many <= a.o_few;     // neighbouring lanes on neighbouring outputs
  for( int l_e = threadIdx.x; l_e < kMany * FEW; l_e += 64 * kWaves ) {
    int const l_m = l_along_many ? l_e % kMany : l_e / FEW;
    int const l_f = l_along_many ? l_e / kMany : l_e % FEW;
    if( l_m >= l_rows || l_f >= a.n_few ) continue;
    int32_t l_sum = 0;
#pragma unroll
    for( int l_w = 0; l_w < kWaves; l_w++ ) l_sum += l_part[l_w][l_f * PITCH + l_m];
    int64_t const l_mg = l_m0 + l_m;
    float const l_sm = a.s_many ? a.s_many[l_c * a.c_sm + l_mg * a.sm_row] : 1.0f;
    float const l_sf = a.s_few ? a.s_few[l_c * a.c_sf + l_f * a.sf_row] : 1.0f;
    float const l_b = a.bias ? a.bias[l_c * a.c_bias + l_mg * a.bias_many + l_f * a.bias_few] : 0.0f;
    float const l_v = i8_finish( l_sum, l_sf, l_sm, l_b, a.relu );
    int64_t const l_o = l_c * a.c_out + l_mg * a.o_many + l_f * a.o_few;
    if( a.out_bf16 ) static_cast< uint16_t * >( a.out )[l_o] = kern::f32_to_bf16_rne( l_v );
    else             static_cast< float * >( a.out )[l_o] = l_v;
  }
}

template< int FB, bool BYTES >
int launch_shape( FewArgs const & a, int32_t C, hipStream_t stream ) {
  hipLaunchKernelGGL( ( contract_i8_few_kernel< FB, BYTES > ), dim3( uint32_t( int64_t( a.tiles ) * C ) ),
                      dim3( 64 * kWaves ), 0, stream, a );
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "contraction_i8 launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

}  // namespace

int launch_i8_few( I8Args const & a, hipStream_t stream ) {
  FewArgs f{};
  bool const l_rows_few = a.M <= a.N;       // the few side is A
  f.many = l_rows_few ? a.b : a.a;
  f.few = l_rows_few ? a.a : a.b;
  f.s_many = l_rows_few ? a.sb : a.sa;
  f.s_few = l_rows_few ? a.sa : a.sb;
  f.bias = a.bias;
  f.out = a.out;
  f.n_many = l_rows_few ? a.N : a.M;
  f.n_few = l_rows_few ? a.M : a.N;
  f.K = a.K;
  f.many_row = l_rows_few ? a.b_col : a.a_row;
  f.few_row = l_rows_few ? a.a_row : a.b_col;
  f.o_many = l_rows_few ? a.o_col : a.o_row;
  f.o_few = l_rows_few ? a.o_row : a.o_col;
  f.sm_row = l_rows_few ? a.sb_col : a.sa_row;
  f.sf_row = l_rows_few ? a.sa_row : a.sb_col;
  f.bias_many = l_rows_few ? a.bias_col : a.bias_row;
  f.bias_few = l_rows_few ? a.bias_row : a.bias_col;
  f.c_many = a.c[l_rows_few ? I8_B : I8_A];
  f.c_few = a.c[l_rows_few ? I8_A : I8_B];
  f.c_sm = a.c[l_rows_few ? I8_SB : I8_SA];
  f.c_sf = a.c[l_rows_few ? I8_SA : I8_SB];
  f.c_out = a.c[I8_OUT];
  f.c_bias = a.c[I8_BIAS];
  f.out_bf16 = a.out_bf16;
  f.relu = a.relu;
  f.tiles = ( f.n_many + kMany - 1 ) / kMany;
  f.pieces = ( a.K + kPiece - 1 ) / kPiece;
  bool const l_bytes = !i8_aligned( a, 4 );
  if( f.n_few <= 16 ) return l_bytes ? launch_shape< 1, true >( f, a.C, stream ) : launch_shape< 1, false >( f, a.C, stream );
  return l_bytes ? launch_shape< 2, true >( f, a.C, stream ) : launch_shape< 2, false >( f, a.C, stream );
}

}  // namespace etir
