// gfx950 product of 8-bit integers, any strides.
//
//   out[c][m][n] = last( sa[c][m] sb[c][n] sum_k A[c][m][k] B[c][n][k] + bias )
//
// One workgroup of 4 waves computes a 64 x 64 tile with
// v_mfma_i32_32x32x32_i8 (a wave a 32 x 32 block), 64 k at a time through LDS.
// Every index is decoded from the fused loops with 64-bit offsets: once a tile
// for rows and columns, once a step for k.  An operand that is unit-stride
// along a single K loop is read in 16-byte pieces at any byte address, any
// other byte by byte with neighbouring lanes on neighbouring rows.  It is the
// kernel for layouts that the others do not take; the byte loads bound it.
#include "i8_internal.h"
#include "contract_kernel.h"

namespace etir {
namespace {

typedef int32_t i32x4 __attribute__( ( ext_vector_type( 4 ) ) );
typedef int32_t i32x16 __attribute__( ( ext_vector_type( 16 ) ) );
// 16 bytes at any address
typedef i32x4 i32x4_u __attribute__( ( aligned( 1 ) ) );

constexpr int kTile  = 64;
constexpr int kBk    = 64;
constexpr int kPitch = kBk + 16;   // 80 bytes a row: 16 rows of 16-byte reads touch each of the 64 banks once

__device__ inline int64_t offset_of( I8Loops const & l, int64_t index, int tensor ) {
  int64_t l_off = 0;
  for( int l_d = l.n - 1; l_d >= 0; l_d-- ) {
    int64_t const l_s = l.size[l_d];
    l_off += ( index % l_s ) * l.stride[l_d][tensor];
    index /= l_s;
  }
  return l_off;
}

// 16 k from k0 of one row, zeros from K on and outside the tensor
__device__ inline i32x4 load_along_k( int8_t const * row, bool ok, int64_t k0, int64_t K ) {
  i32x4 l_v = { 0, 0, 0, 0 };
  if( !ok || k0 >= K ) return l_v;
  if( k0 + 16 <= K ) return *reinterpret_cast< i32x4_u const * >( row + k0 );
  for( int l_i = 0; k0 + l_i < K; l_i++ ) {
    reinterpret_cast< int8_t * >( &l_v )[l_i] = row[k0 + l_i];
  }
  return l_v;
}

__device__ inline i32x4 load_bytes( int8_t const * row, bool ok, int64_t k0, int64_t K, I8Loops const & loops, int tensor ) {
  uint32_t l_w[4] = { 0, 0, 0, 0 };
#pragma unroll
  for( int l_i = 0; l_i < 16; l_i++ ) {
    int64_t const l_k = k0 + l_i;
    if( ok && l_k < K ) {
      l_w[l_i / 4] |= uint32_t( uint8_t( row[offset_of( loops, l_k, tensor )] ) ) << ( 8 * ( l_i % 4 ) );
    }
  }
  return i32x4{ int32_t( l_w[0] ), int32_t( l_w[1] ), int32_t( l_w[2] ), int32_t( l_w[3] ) };
}

// an operand's side of a tile: 64 rows x 64 k, 16 bytes a thread
template< int TENSOR >
__device__ inline void stage( char * lds, int8_t const * base, I8Loops const & loops_k, bool along_k,
                              int64_t const * row_off, int rows, int64_t k0, int64_t K ) {
  int const l_t = threadIdx.x;
  int const l_row = along_k ? l_t / 4 : l_t % 64;
  int const l_kc = along_k ? l_t % 4 : l_t / 64;
  int8_t const * l_p = base + row_off[l_row];
  bool const l_ok = l_row < rows;
  i32x4 const l_v = along_k ? load_along_k( l_p, l_ok, k0 + 16 * l_kc, K )
                            : load_bytes( l_p, l_ok, k0 + 16 * l_kc, K, loops_k, TENSOR );
  *reinterpret_cast< i32x4 * >( lds + l_row * kPitch + 16 * l_kc ) = l_v;
}

__device__ inline bool unit_k( I8Loops const & k, int tensor ) {
  return k.n == 0 || ( k.n == 1 && k.stride[0][tensor] == 1 );
}

__global__ __launch_bounds__( 256 )
void contract_i8_general_kernel( I8GeneralArgs a ) {
  __shared__ __align__( 16 ) char l_lds_a[kTile * kPitch];
  __shared__ __align__( 16 ) char l_lds_b[kTile * kPitch];
  __shared__ int64_t l_off_a[kTile], l_off_b[kTile], l_out_m[kTile], l_out_n[kTile];
  __shared__ float   l_sa[kTile], l_sb[kTile], l_bias_m[kTile], l_bias_n[kTile];

  int const l_t = threadIdx.x;
  int64_t l_id = blockIdx.x;
  int64_t const l_n0 = ( l_id % a.tiles_n ) * kTile;
  l_id /= a.tiles_n;
  int64_t const l_m0 = ( l_id % a.tiles_m ) * kTile;
  int64_t const l_c  = l_id / a.tiles_m;
  int const l_rows = int( min( int64_t( kTile ), a.M - l_m0 ) );
  int const l_cols = int( min( int64_t( kTile ), a.N - l_n0 ) );

  // rows and columns past the tensor take the last one's offsets and are not stored
  if( l_t < kTile ) {
    int64_t const l_m = min( l_m0 + l_t, a.M - 1 );
    int64_t const l_bias = offset_of( a.c, l_c, I8_BIAS );
    l_off_a[l_t] = offset_of( a.c, l_c, I8_A ) + offset_of( a.m, l_m, I8_A );
    l_out_m[l_t] = offset_of( a.c, l_c, I8_OUT ) + offset_of( a.m, l_m, I8_OUT );
    l_sa[l_t] = a.sa ? a.sa[offset_of( a.c, l_c, I8_SA ) + offset_of( a.m, l_m, I8_SA )] : 1.0f;
    l_bias_m[l_t] = 0.0f;
    // the bias runs over rows where left and right have changed places
    if( a.bias && a.bias_rows ) l_bias_m[l_t] = a.bias[l_bias + offset_of( a.m, l_m, I8_BIAS )];
  }
  else if( l_t < 2 * kTile ) {
    int const l_i = l_t - kTile;
    int64_t const l_n = min( l_n0 + l_i, a.N - 1 );
    int64_t const l_bias = offset_of( a.c, l_c, I8_BIAS );
    l_off_b[l_i] = offset_of( a.c, l_c, I8_B ) + offset_of( a.n, l_n, I8_B );
    l_out_n[l_i] = offset_of( a.n, l_n, I8_OUT );
    l_sb[l_i] = a.sb ? a.sb[offset_of( a.c, l_c, I8_SB ) + offset_of( a.n, l_n, I8_SB )] : 1.0f;
    l_bias_n[l_i] = 0.0f;
    if( a.bias && !a.bias_rows ) l_bias_n[l_i] = a.bias[l_bias + offset_of( a.n, l_n, I8_BIAS )];
  }
  __syncthreads();

  bool const l_ka = unit_k( a.k, I8_A ), l_kb = unit_k( a.k, I8_B );
  int const l_wave = l_t / 64, l_lane = l_t % 64;
  int const l_wm = 32 * ( l_wave / 2 ), l_wn = 32 * ( l_wave % 2 );
  i32x16 l_acc = { 0 };
  for( int64_t l_k0 = 0; l_k0 < a.K; l_k0 += kBk ) {
    stage< I8_A >( l_lds_a, a.a, a.k, l_ka, l_off_a, l_rows, l_k0, a.K );
    stage< I8_B >( l_lds_b, a.b, a.k, l_kb, l_off_b, l_cols, l_k0, a.K );
    __syncthreads();
#pragma unroll
    for( int l_s = 0; l_s < kBk / 32; l_s++ ) {
      int const l_k = 32 * l_s + 16 * ( l_lane / 32 );
      i32x4 const l_fa = *reinterpret_cast< i32x4 const * >( l_lds_a + ( l_wm + l_lane % 32 ) * kPitch + l_k );
      i32x4 const l_fb = *reinterpret_cast< i32x4 const * >( l_lds_b + ( l_wn + l_lane % 32 ) * kPitch + l_k );
      l_acc = __builtin_amdgcn_mfma_i32_32x32x32_i8( l_fa, l_fb, l_acc, 0, 0, 0 );
    }
    __syncthreads();
  }

  int const l_n = l_wn + l_lane % 32;
  if( l_n >= l_cols ) return;
#pragma unroll
  for( int l_i = 0; l_i < 16; l_i++ ) {
    int const l_m = l_wm + 8 * ( l_i / 4 ) + 4 * ( l_lane / 32 ) + l_i % 4;
    if( l_m >= l_rows ) continue;
    float const l_v = i8_finish( l_acc[l_i], l_sa[l_m], l_sb[l_n], l_bias_m[l_m] + l_bias_n[l_n], a.relu );
    int64_t const l_o = l_out_m[l_m] + l_out_n[l_n];
    if( a.out_bf16 ) static_cast< uint16_t * >( a.out )[l_o] = kern::f32_to_bf16_rne( l_v );
    else             static_cast< float * >( a.out )[l_o] = l_v;
  }
}

}  // namespace

int launch_i8_general( I8GeneralArgs const & a, hipStream_t stream ) {
  uint32_t const l_grid = uint32_t( int64_t( a.tiles_m ) * a.tiles_n * a.C );
  hipLaunchKernelGGL( contract_i8_general_kernel, dim3( l_grid ), dim3( 256 ), 0, stream, a );
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "contraction_i8 launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

}  // namespace etir
