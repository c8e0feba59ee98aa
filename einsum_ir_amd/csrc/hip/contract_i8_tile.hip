// gfx950 product of 8-bit integers, tiles staged through LDS:
//
//   out[c][m][n] = last( sa[c][m] sb[c][n] sum_k A[c][m][k] B[c][n][k] + bias )
//
// A workgroup computes a BM x BN tile with v_mfma_i32_32x32x32_i8, WM x WN waves
// a K group and KG groups, which take the blocks of 128 k in turn and add their
// sums in LDS at the end (integers: in any order the same).
//
// Operands go from global memory into LDS directly (buffer_load ... lds).  Rows
// at multiples of 16 bytes: 128 k of a row in 128 bytes, 16-byte piece g of row r
// at place g ^ swz(r), so that the fragment reads (16 bytes a lane, 32 rows)
// touch every bank equally.  Rows anywhere (SHIFT): the dwords that hold the 128
// k, in 144 bytes; a fragment is read with the dword after it and shifted by its
// row's first byte, and k from K on count as zeros on one side (2048 a side with
// K = 2050: 22 us, byte-wise through registers 30, K = 2048 15).  Two to four
// buffers, one barrier a block.
//
// The channels' side is the first operand of the matrix instruction, so a lane
// holds 4 neighbouring columns of the output; the tile goes out through LDS in
// rows of 16-byte stores.
#include "i8_internal.h"
#include "contract_dma.h"

namespace etir {
namespace {

using kern::i32x4;
typedef int32_t i32x16 __attribute__( ( ext_vector_type( 16 ) ) );
typedef float f32x4 __attribute__( ( ext_vector_type( 4 ) ) );

constexpr int kBk = 128;      // k of a block

// ROWS rows of an operand by WAVES waves, one K group's side of the tile, loaded
// 64 pieces of 16 bytes at a time.
// Rows (and K) at multiples of 16 bytes: 8 pieces a row, piece g of row r at
// place g ^ swz(r).  SHIFT, rows anywhere: the 9 pieces that hold a row's 128 k
// from the dword on that the row's first byte lies in, one after the other; the
// pitch of 144 bytes spreads 16 rows over all banks.
template< int ROWS, int WAVES, bool SHIFT >
struct Side {
  static constexpr int PER_ROW = SHIFT ? 9 : 8;
  static constexpr int PITCH   = 16 * PER_ROW;
  static constexpr int LOADS   = ( ROWS * PER_ROW + 63 ) / 64;
  static constexpr int EACH    = ( LOADS + WAVES - 1 ) / WAVES;      // a wave's loads
  static constexpr int BYTES   = EACH * WAVES * 1024;
  static_assert( SHIFT || LOADS % WAVES == 0, "loads have to divide over the waves" );

  uint32_t m_off[EACH];       // bytes from the tile's first row to the lane's piece of block 0
  i32x4    m_rsrc;
  int      m_k[2];            // the lane's k of a block in even and odd loads (not SHIFT)
  uint32_t m_first;           // the wave's first load

  __device__ inline void init( int8_t const * tile, int32_t stride, int32_t rows, int32_t K, int wave, int lane ) {
    m_first = wave * EACH;
    if constexpr( SHIFT ) {
      // up to the dword of the last k of the tile's last row
      uint32_t const l_off = uint32_t( reinterpret_cast< uintptr_t >( tile ) & 3 );
      m_rsrc = kern::make_rsrc( tile - l_off, ( l_off + uint32_t( min( rows, ROWS ) - 1 ) * uint32_t( stride ) + uint32_t( K ) + 3 ) & ~3u );
#pragma unroll
      for( int l_i = 0; l_i < EACH; l_i++ ) {
        uint32_t const l_piece = ( m_first + l_i ) * 64 + lane, l_r = l_piece / PER_ROW;
        m_off[l_i] = ( ( l_off + min( l_r, uint32_t( rows - 1 ) ) * uint32_t( stride ) ) & ~3u ) + 16 * ( l_piece % PER_ROW );
        if( l_r >= ROWS ) m_off[l_i] = kern::kDmaOob;
      }
    }
    else {
      m_rsrc = kern::make_rsrc( tile, kern::kDmaOob );
#pragma unroll
      for( int l_i = 0; l_i < 2; l_i++ ) m_k[l_i] = 16 * ( ( lane % 8 ) ^ int( kern::swz_k( 8 * l_i + lane / 8 ) ) );
#pragma unroll
      for( int l_i = 0; l_i < EACH; l_i++ ) {
        // rows past the tensor read its last one and are not stored
        int32_t const l_r = min( int32_t( 8 * ( m_first + l_i ) + lane / 8 ), rows - 1 );
        m_off[l_i] = uint32_t( l_r * stride + k_of( l_i ) );
      }
    }
  }
  __device__ inline int k_of( int i ) const { return m_k[( m_first + i ) % 2]; }

  // starts the wave's load I of the block at k0 into lds
  template< int I >
  __device__ __attribute__( ( always_inline ) ) inline void issue( uint32_t lds, int32_t k0, int32_t K ) {
    uint32_t l_off = m_off[I], l_k0 = uint32_t( k0 );
    if constexpr( SHIFT ) {
      // where the pieces may leave the tensor, the k go into the offset that
      // the buffer's range check sees
      if( k0 + PITCH > K ) {
        l_off += l_k0;
        l_k0 = 0;
      }
    }
    // K is a multiple of 16, so a lane's k are inside or outside; outside: zeros
    else if( k0 + kBk > K && k0 + k_of( I ) >= K ) l_off = kern::kDmaOob;
    kern::set_m0( lds + ( m_first + I ) * 1024 );
    kern::dma16_so< 0 >( m_rsrc, l_off, l_k0 );
  }
};

// 16 k of a row as read from LDS; SHIFT: the dwords they lie in
template< bool SHIFT > struct Raw { i32x4 v; };
template<> struct Raw< true > { i32x4 v; int32_t w; };

// elements from row to row of a wave's output slab in LDS
template< class T, int COLS > constexpr int kPitch = COLS + 16 / int( sizeof( T ) );

// Stores ROWS rows x COLS columns of a wave's slab from row m1, column n1 of
// the output on: 16 bytes a lane where the columns are adjacent, else an element
// a lane; non-temporal, the output is not read here again (4072 x 2048 x 2048:
// 23.2 -> 21.2 us).  bf16 rows of an odd stride start between two dwords, where
// these stores are slow but better than an element a lane (2395 x 80 x 7693:
// 23.3 us against 27.7; vectors shifted by one element to lie on dwords, with
// single stores at the slab's edges, 27.7).
template< int ROWS, int COLS, class T >
__device__ inline void store_slab( I8Args const & a, T const * slab, int64_t out0, int32_t m1, int32_t n1, int lane ) {
  constexpr int V = 16 / sizeof( T );
  constexpr int LANES = COLS / V;            // lanes a row
  constexpr int PITCH = kPitch< T, COLS >;
  typedef T v __attribute__( ( ext_vector_type( V ) ) );
  typedef v v_any __attribute__( ( aligned( sizeof( T ) ) ) );
  T * const l_out = static_cast< T * >( a.out ) + out0;
  if( a.has( I8Args::VEC_OUT ) ) {
#pragma unroll
    for( int l_p = 0; l_p < ROWS * LANES / 64; l_p++ ) {
      int const l_r = l_p * ( 64 / LANES ) + lane / LANES, l_c = lane % LANES * V;
      v const l_v = *reinterpret_cast< v const * >( slab + l_r * PITCH + l_c );
      if( m1 + l_r >= a.M ) continue;
      T * const l_o = l_out + int64_t( m1 + l_r ) * a.o_row + n1 + l_c;
      int32_t const l_left = a.N - n1 - l_c;       // columns from this lane's first on
      if( l_left >= V ) __builtin_nontemporal_store( l_v, reinterpret_cast< v_any * >( l_o ) );
      else {
#pragma unroll
        for( int l_e = 0; l_e < V; l_e++ ) if( l_e < l_left ) l_o[l_e] = l_v[l_e];
      }
    }
  }
  else {
#pragma unroll 4
    for( int l_p = 0; l_p < ROWS * COLS / 64; l_p++ ) {
      int const l_r = ( l_p * 64 + lane ) / COLS, l_c = ( l_p * 64 + lane ) % COLS;
      T const l_v = slab[l_r * PITCH + l_c];
      if( m1 + l_r < a.M && n1 + l_c < a.N ) l_out[int64_t( m1 + l_r ) * a.o_row + int64_t( n1 + l_c ) * a.o_col] = l_v;
    }
  }
}

template< int BM, int BN, int WM, int WN, int KG, int STAGES, bool DEEP, bool SHIFT >
__global__ __launch_bounds__( 64 * WM * WN * KG )
void contract_i8_tile_kernel( I8Args a ) {
  constexpr int WAVES = WM * WN;                       // of a K group
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;  // 32 x 32 blocks a wave
  typedef Side< BM, WAVES, SHIFT > SideA;
  typedef Side< BN, WAVES, SHIFT > SideB;
  constexpr int STAGE = SideA::BYTES + SideB::BYTES;
  constexpr int COLS = BN / WN;
  // a wave's output slab: fp32 32 rows, bf16 all of its rows
  constexpr int SLAB_F32 = 32 * kPitch< float, COLS > * 4, SLAB_BF16 = 32 * TM * kPitch< __bf16, COLS > * 2;
  constexpr int SLAB = SLAB_F32 > SLAB_BF16 ? SLAB_F32 : SLAB_BF16;
  constexpr int SLABS = WAVES * SLAB;
  constexpr int PARTS = KG > 1 ? ( KG - 1 ) * BM * BN * 4 : 0;
  constexpr int BYTES = STAGES * KG * STAGE > SLABS + PARTS ? STAGES * KG * STAGE : SLABS + PARTS;
  __shared__ __align__( 16 ) char l_lds[BYTES];
  __shared__ __align__( 16 ) float l_sb[BN], l_bias[BN];

  int32_t const l_k = a.K();
  int32_t const l_blocks = ( l_k + kBk - 1 ) / kBk;
  int32_t const l_tiles_m = ( a.M + BM - 1 ) / BM, l_tiles_n = ( a.N + BN - 1 ) / BN;
  int const l_lane = threadIdx.x % 64;
  int const l_w = __builtin_amdgcn_readfirstlane( threadIdx.x / 64 );
  int const l_group = l_w / WAVES, l_wave = l_w % WAVES;
  int const l_wm = l_wave / WN * ( BM / WM ), l_wn = l_wave % WN * ( BN / WN );

  // Neighbouring tiles on one XCD (workgroups go to the 8 XCDs in turn), and
  // there in bands of 8 tile rows, so that its cache serves both operands.
  int32_t const l_per_c = l_tiles_m * l_tiles_n, l_each = l_per_c / 8;
  int64_t const l_c = blockIdx.x / l_per_c;
  int32_t l_r = blockIdx.x % l_per_c;
  if( l_r < 8 * l_each ) l_r = l_r % 8 * l_each + l_r / 8;
  int32_t const l_band = l_r / ( 8 * l_tiles_n ) * 8;
  int32_t const l_high = min( 8, l_tiles_m - l_band );
  int32_t const l_m0 = ( l_band + l_r % ( 8 * l_tiles_n ) % l_high ) * BM;
  int32_t const l_n0 = ( l_r % ( 8 * l_tiles_n ) / l_high ) * BN;

  int8_t const * const l_at_a = a.a + l_c * a.c[I8_A] + int64_t( l_m0 ) * a.a_row;
  int8_t const * const l_at_b = a.b + l_c * a.c[I8_B] + int64_t( l_n0 ) * a.b_col;
  SideA l_a;
  SideB l_b;
  l_a.init( l_at_a, a.a_row, a.M - l_m0, l_k, l_wave, l_lane );
  l_b.init( l_at_b, a.b_col, a.N - l_n0, l_k, l_wave, l_lane );

  // scales and bias, needed after the loop
  bool const l_bias_rows = a.has( I8Args::BIAS_ROWS );
  constexpr int CH = ( BN + 64 * WAVES * KG - 1 ) / ( 64 * WAVES * KG );
  float l_sb_r[CH], l_bias_r[CH], l_sa[TM], l_bias_m[TM];
#pragma unroll
  for( int l_i = 0; l_i < CH; l_i++ ) {
    int32_t const l_n = min( l_n0 + l_i * 64 * WAVES * KG + int( threadIdx.x ), a.N - 1 );
    l_sb_r[l_i] = a.sb ? a.sb[l_c * a.c[I8_SB] + int64_t( l_n ) * a.sb_col] : 1.0f;
    l_bias_r[l_i] = a.bias && !l_bias_rows ? a.bias[l_c * a.c[I8_BIAS] + int64_t( l_n ) * a.bias_step] : 0.0f;
  }
  int const l_row = l_lane % 32;
#pragma unroll
  for( int l_j = 0; l_j < TM; l_j++ ) {
    int32_t const l_m = min( l_m0 + l_wm + 32 * l_j + l_row, a.M - 1 );
    l_sa[l_j] = a.sa ? a.sa[l_c * a.c[I8_SA] + int64_t( l_m ) * a.sa_row] : 1.0f;
    l_bias_m[l_j] = a.bias && l_bias_rows ? a.bias[l_c * a.c[I8_BIAS] + int64_t( l_m ) * a.bias_step] : 0.0f;
  }

  // this group's buffers
  char * const l_buf = l_lds + l_group * STAGES * STAGE;
  uint32_t const l_buf_at = kern::lds_addr( l_buf );
  int const l_steps = ( l_blocks + KG - 1 ) / KG;
  // first k of the group's step s; past the last block nothing is in range and
  // zeros are loaded
  auto k_of_step = [&]( int s ) -> int32_t { return min( s * KG + l_group, l_blocks ) * kBk; };
  // the wave's load i, those of both sides counted through
  constexpr int EACH = SideA::EACH + SideB::EACH;
  auto issue = [&]( auto ic, int stage, int32_t k0 ) __attribute__( ( always_inline ) ) {
    constexpr int l_i = decltype( ic )::value;
    uint32_t const l_to = l_buf_at + stage * STAGE;
    if constexpr( l_i < SideA::EACH ) l_a.template issue< l_i >( l_to, k0, l_k );
    else                              l_b.template issue< l_i - SideA::EACH >( l_to + SideA::BYTES, k0, l_k );
  };
  // loads of block 1 (two buffers) that are issued in front of the loop
  constexpr int EARLY = ( EACH + 1 ) / 2;
  kern::static_for< EACH >( [&]( auto ic ) __attribute__( ( always_inline ) ) { issue( ic, 0, k_of_step( 0 ) ); } );
  if constexpr( STAGES > 2 ) {
    kern::static_for< STAGES - 2 >( [&]( auto sc ) __attribute__( ( always_inline ) ) {
      constexpr int l_s = decltype( sc )::value + 1;
      kern::static_for< EACH >( [&]( auto ic ) __attribute__( ( always_inline ) ) { issue( ic, l_s, k_of_step( l_s ) ); } );
    } );
    if constexpr( !DEEP ) {
      kern::wait_vmcnt< ( STAGES - 2 ) * EACH >();
      kern::barrier_lds();
    }
  }
  else {
    kern::static_for< EARLY >( [&]( auto ic ) __attribute__( ( always_inline ) ) { issue( ic, 1, k_of_step( 1 ) ); } );
    kern::wait_vmcnt< EARLY >();
    kern::barrier_lds();
  }

  // Fragments of 32 k: TM of rows, then TN of columns.
  constexpr int FRAGS = TM + TN, MFMAS = TM * TN;
  constexpr int HELD = DEEP ? 4 : 2;
  Raw< SHIFT > l_f[HELD][FRAGS];
  uint32_t const l_swz = kern::swz_k( l_row );       // of 32-row blocks: the same
  auto read = [&]( auto fc, Raw< SHIFT > * f, int stage, int q ) __attribute__( ( always_inline ) ) {
    constexpr int l_i = decltype( fc )::value;
    int const l_first = l_i < TM ? ( l_wm + 32 * l_i ) * SideA::PITCH : SideA::BYTES + ( l_wn + 32 * ( l_i - TM ) ) * SideB::PITCH;
    char const * const l_p = l_buf + stage * STAGE + l_first + l_row * SideA::PITCH;
    if constexpr( SHIFT ) {
      f[l_i].v = *reinterpret_cast< i32x4 const * >( l_p + 16 * ( 2 * q + l_lane / 32 ) );
      f[l_i].w = *reinterpret_cast< int32_t const * >( l_p + 16 * ( 2 * q + l_lane / 32 ) + 16 );
    }
    else f[l_i].v = *reinterpret_cast< i32x4 const * >( l_p + ( ( ( 2 * q + l_lane / 32 ) ^ l_swz ) << 4 ) );
  };
  // SHIFT: the first byte of a row in its dword (of rows 32 apart the same), and
  // from K on zeros on A's side
  int const l_shift_a = int( ( reinterpret_cast< uintptr_t >( l_at_a ) + uint32_t( l_row ) * uint32_t( a.a_row ) ) & 3 );
  int const l_shift_b = int( ( reinterpret_cast< uintptr_t >( l_at_b ) + uint32_t( l_row ) * uint32_t( a.b_col ) ) & 3 );
  auto ready = [&]( auto fc, Raw< SHIFT > const * f, int32_t k0, int q ) __attribute__( ( always_inline ) ) -> i32x4 {
    constexpr int l_i = decltype( fc )::value;
    i32x4 l_v = f[l_i].v;
    if constexpr( SHIFT ) {
      int const l_s = l_i < TM ? l_shift_a : l_shift_b;
      l_v = i32x4{ int32_t( __builtin_amdgcn_alignbyte( l_v[1], l_v[0], l_s ) ), int32_t( __builtin_amdgcn_alignbyte( l_v[2], l_v[1], l_s ) ),
                   int32_t( __builtin_amdgcn_alignbyte( l_v[3], l_v[2], l_s ) ), int32_t( __builtin_amdgcn_alignbyte( f[l_i].w, l_v[3], l_s ) ) };
      if( l_i < TM && k0 + kBk > l_k ) {
        int32_t const l_n = l_k - ( k0 + 32 * q + 16 * ( l_lane / 32 ) );      // bytes that count
#pragma unroll
        for( int l_d = 0; l_d < 4; l_d++ ) {
          int32_t const l_left = l_n - 4 * l_d;
          l_v[l_d] &= l_left >= 4 ? -1 : l_left <= 0 ? 0 : int32_t( ( 1u << ( 8 * l_left ) ) - 1 );
        }
      }
    }
    return l_v;
  };
  i32x16 l_acc[TN][TM];
#pragma unroll
  for( int l_i = 0; l_i < TN * TM; l_i++ ) l_acc[l_i / TM][l_i % TM] = i32x16{ 0 };
  auto multiply = [&]( auto mc, i32x4 const * f ) __attribute__( ( always_inline ) ) {
    constexpr int l_i = decltype( mc )::value / TM, l_j = decltype( mc )::value % TM;
    l_acc[l_i][l_j] = __builtin_amdgcn_mfma_i32_32x32x32_i8( f[TM + l_i], f[l_j], l_acc[l_i][l_j], 0, 0, 0 );
  };

  // One block of 128 k in 4 parts of 32.  During a part's matrix instructions the
  // next part's fragments are read; the barrier stands in front of the last part,
  // when every wave has read all of this block and the next one has landed.  Two
  // buffers: the block after that is loaded over this one from there on, half of
  // it in the last part, half in the next block's first.  More: the block
  // STAGES - 1 ahead is loaded over the last one, spread over the first three
  // parts.
  auto step = [&]( int l_st, int l_next, int l_free, int s ) __attribute__( ( always_inline ) ) {
    kern::static_for< 4 >( [&]( auto qc ) __attribute__( ( always_inline ) ) {
      constexpr int l_q = decltype( qc )::value;
      if constexpr( l_q == 3 ) {
        kern::wait_vmcnt< ( STAGES - 2 ) * EACH >();
        kern::wait_lgkmcnt0();
        kern::barrier_lds();
      }
      int32_t const l_k0 = k_of_step( s + ( STAGES > 2 ? STAGES - 1 : l_q == 3 ? 2 : 1 ) );
      i32x4 l_g[FRAGS];
      kern::static_for< FRAGS >( [&]( auto fc ) __attribute__( ( always_inline ) ) {
        l_g[decltype( fc )::value] = ready( fc, l_f[l_q % 2], k_of_step( s ), l_q );
      } );
      kern::static_for< MFMAS >( [&]( auto mc ) __attribute__( ( always_inline ) ) {
        constexpr int l_m = decltype( mc )::value;
        multiply( mc, l_g );
        // the next part's fragments over the first half of the instructions
        constexpr int l_slots = ( MFMAS + 1 ) / 2;
        if constexpr( l_m < l_slots ) {
          constexpr int l_from = FRAGS * l_m / l_slots, l_to = FRAGS * ( l_m + 1 ) / l_slots;
          kern::static_for< l_to - l_from >( [&]( auto fc ) __attribute__( ( always_inline ) ) {
            read( std::integral_constant< int, l_from + decltype( fc )::value >(), l_f[( l_q + 1 ) % 2],
                  l_q == 3 ? l_next : l_st, ( l_q + 1 ) % 4 );
          } );
        }
        if constexpr( STAGES > 2 && l_q < 3 ) {
          constexpr int l_at = l_q * MFMAS + l_m, l_from = EACH * l_at / ( 3 * MFMAS ), l_to = EACH * ( l_at + 1 ) / ( 3 * MFMAS );
          kern::static_for< l_to - l_from >( [&]( auto ic ) __attribute__( ( always_inline ) ) {
            issue( std::integral_constant< int, l_from + decltype( ic )::value >(), l_free, l_k0 );
          } );
        }
        if constexpr( STAGES == 2 && ( l_q == 3 || l_q == 0 ) ) {
          constexpr int l_p0 = l_q == 3 ? 0 : EARLY, l_n = l_q == 3 ? EARLY : EACH - EARLY;
          constexpr int l_from = l_p0 + l_n * l_m / MFMAS, l_to = l_p0 + l_n * ( l_m + 1 ) / MFMAS;
          kern::static_for< l_to - l_from >( [&]( auto ic ) __attribute__( ( always_inline ) ) {
            issue( std::integral_constant< int, l_from + decltype( ic )::value >(), l_q == 3 ? l_st : l_next, l_k0 );
          } );
        }
        __builtin_amdgcn_sched_barrier( 0 );
      } );
    } );
  };
  // DEEP, for small tiles, which wait for memory and not for the matrix
  // cores: blocks are issued STAGES - 1 ahead, also past the last one, so that
  // a wave's loads in flight are the same number in every step.
  auto deep = [&]( auto stage_c, int s ) __attribute__( ( always_inline ) ) {
    constexpr int l_st = decltype( stage_c )::value;
    // this block is in LDS, and every wave has read the last one
    kern::wait_vmcnt< ( STAGES - 2 ) * EACH >();
    kern::wait_lgkmcnt0();
    kern::barrier_lds();
    kern::static_for< 4 >( [&]( auto qc ) __attribute__( ( always_inline ) ) {
      constexpr int l_q = decltype( qc )::value;
      kern::static_for< FRAGS >( [&]( auto fc ) __attribute__( ( always_inline ) ) { read( fc, l_f[l_q % HELD], l_st, l_q ); } );
    } );
    __builtin_amdgcn_sched_barrier( 0 );
    int32_t const l_k0 = k_of_step( s + STAGES - 1 );
    kern::static_for< EACH >( [&]( auto ic ) __attribute__( ( always_inline ) ) {
      issue( ic, ( l_st + STAGES - 1 ) % STAGES, l_k0 );
    } );
    __builtin_amdgcn_sched_barrier( 0 );
    kern::static_for< 4 >( [&]( auto qc ) __attribute__( ( always_inline ) ) {
      constexpr int l_q = decltype( qc )::value;
      i32x4 l_g[FRAGS];
      kern::static_for< FRAGS >( [&]( auto fc ) __attribute__( ( always_inline ) ) {
        l_g[decltype( fc )::value] = ready( fc, l_f[l_q % HELD], k_of_step( s ), l_q );
      } );
      kern::static_for< MFMAS >( [&]( auto mc ) __attribute__( ( always_inline ) ) { multiply( mc, l_g ); } );
    } );
  };
  if constexpr( !DEEP ) {
    kern::static_for< FRAGS >( [&]( auto fc ) __attribute__( ( always_inline ) ) { read( fc, l_f[0], 0, 0 ); } );
    int l_st = 0, l_free = STAGES - 1;
    for( int l_s = 0; l_s < l_steps; l_s++ ) {
      int const l_next = l_st == STAGES - 1 ? 0 : l_st + 1;
      step( l_st, l_next, l_free, l_s );
      l_free = l_st;
      l_st = l_next;
    }
  }
  else {
    for( int l_s = 0; l_s < l_steps; l_s += STAGES ) {
      kern::static_for< STAGES >( [&]( auto sc ) __attribute__( ( always_inline ) ) {
        constexpr int l_st = decltype( sc )::value;
        if( l_s + l_st < l_steps ) deep( sc, l_s + l_st );
      } );
    }
  }
  kern::wait_vmcnt< 0 >();
#pragma unroll
  for( int l_i = 0; l_i < CH; l_i++ ) {
    int const l_n = l_i * 64 * WAVES * KG + threadIdx.x;
    if( l_n < BN ) {
      l_sb[l_n] = l_sb_r[l_i];
      l_bias[l_n] = l_bias_r[l_i];
    }
  }
  __syncthreads();           // nothing is on its way into LDS, all fragments are read, the scales are there

  // the other groups' sums to the first one
  if constexpr( KG > 1 ) {
    i32x4 * const l_part = reinterpret_cast< i32x4 * >( l_lds + SLABS );
    if( l_group > 0 ) {
#pragma unroll
      for( int l_i = 0; l_i < TN * TM * 4; l_i++ ) {
        i32x16 const & l_v = l_acc[l_i / 4 / TM][l_i / 4 % TM];
        int const l_e = 4 * ( l_i % 4 );
        l_part[( ( ( l_group - 1 ) * WAVES + l_wave ) * TN * TM * 4 + l_i ) * 64 + l_lane]
            = i32x4{ l_v[l_e], l_v[l_e + 1], l_v[l_e + 2], l_v[l_e + 3] };
      }
    }
    __syncthreads();
    if( l_group > 0 ) return;
    for( int l_g = 0; l_g < KG - 1; l_g++ ) {
#pragma unroll
      for( int l_i = 0; l_i < TN * TM * 4; l_i++ ) {
        i32x4 const l_v = l_part[( ( l_g * WAVES + l_wave ) * TN * TM * 4 + l_i ) * 64 + l_lane];
#pragma unroll
        for( int l_e = 0; l_e < 4; l_e++ ) l_acc[l_i / 4 / TM][l_i / 4 % TM][4 * ( l_i % 4 ) + l_e] += l_v[l_e];
      }
    }
  }

  // PASS blocks of 32 rows at a time through this wave's slab
  int64_t const l_out0 = l_c * a.c[I8_OUT];
  auto finish = [&]( auto zero, auto pass ) __attribute__( ( always_inline ) ) {
    typedef decltype( zero ) T;
    typedef T t4 __attribute__( ( ext_vector_type( 4 ) ) );
    constexpr int PASS = decltype( pass )::value;
    T * const l_slab = reinterpret_cast< T * >( l_lds + l_wave * SLAB );
#pragma unroll
    for( int l_j0 = 0; l_j0 < TM; l_j0 += PASS ) {
#pragma unroll
      for( int l_i = 0; l_i < TN; l_i++ ) {
#pragma unroll
        for( int l_q = 0; l_q < 4; l_q++ ) {
          int const l_n = 32 * l_i + 8 * l_q + 4 * ( l_lane / 32 );
          f32x4 const l_sb4 = *reinterpret_cast< f32x4 const * >( l_sb + l_wn + l_n );
          f32x4 l_b4 = { 0.0f, 0.0f, 0.0f, 0.0f };
          if( a.bias && !l_bias_rows ) l_b4 = *reinterpret_cast< f32x4 const * >( l_bias + l_wn + l_n );
#pragma unroll
          for( int l_j = l_j0; l_j < l_j0 + PASS; l_j++ ) {
            float l_v[4];
#pragma unroll
            for( int l_e = 0; l_e < 4; l_e++ ) {
              l_v[l_e] = i8_finish( l_acc[l_i][l_j][4 * l_q + l_e], l_sa[l_j], l_sb4[l_e],
                                    l_bias_rows ? l_bias_m[l_j] : l_b4[l_e], 0 );
            }
            if( a.has( I8Args::RELU ) ) {
#pragma unroll
              for( int l_e = 0; l_e < 4; l_e++ ) l_v[l_e] = l_v[l_e] < 0.0f ? 0.0f : l_v[l_e];
            }
            *reinterpret_cast< t4 * >( l_slab + ( 32 * ( l_j - l_j0 ) + l_row ) * kPitch< T, COLS > + l_n )
                = t4{ static_cast< T >( l_v[0] ), static_cast< T >( l_v[1] ), static_cast< T >( l_v[2] ), static_cast< T >( l_v[3] ) };
          }
        }
      }
      // the slab is this wave's own, and its LDS operations are in order
      __builtin_amdgcn_fence( __ATOMIC_ACQ_REL, "wavefront" );
      store_slab< 32 * PASS, COLS, T >( a, l_slab, l_out0, l_m0 + l_wm + 32 * l_j0, l_n0 + l_wn, l_lane );
      __builtin_amdgcn_fence( __ATOMIC_ACQ_REL, "wavefront" );
    }
  };
  if( a.has( I8Args::OUT_BF16 ) ) finish( __bf16( 0.0f ), std::integral_constant< int, TM >() );
  else             finish( 0.0f, std::integral_constant< int, 1 >() );
}

template< int BM, int BN, int WM, int WN, int KG, int STAGES, bool DEEP, bool SHIFT >
int launch_shape( I8Args const & a, int64_t C, hipStream_t stream ) {
  uint32_t const l_grid = uint32_t( ( int64_t( a.M ) + BM - 1 ) / BM * ( ( int64_t( a.N ) + BN - 1 ) / BN ) * C );
  hipLaunchKernelGGL( ( contract_i8_tile_kernel< BM, BN, WM, WN, KG, STAGES, DEEP, SHIFT > ), dim3( l_grid ), dim3( 64 * WM * WN * KG ),
                      0, stream, a );
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "contraction_i8 launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

}  // namespace

int launch_i8_tile( I8Args const & args, int64_t C, I8Kernel kernel, hipStream_t stream ) {
  I8Args a = args;
  if( a.o_col == 1 ) a.k_flags |= I8Args::VEC_OUT;
  switch( kernel ) {
    case I8Kernel::TILE_32x32:   return launch_shape< 32, 32, 1, 1, 4, 3, true, false >( a, C, stream );
    case I8Kernel::TILE_64x32:   return launch_shape< 64, 32, 2, 1, 2, 4, true, false >( a, C, stream );
    case I8Kernel::TILE_64x64:   return launch_shape< 64, 64, 2, 2, 1, 4, true, false >( a, C, stream );
    case I8Kernel::TILE_128x64:  return launch_shape< 128, 64, 2, 2, 1, 3, false, false >( a, C, stream );
    case I8Kernel::TILE_128x128: return launch_shape< 128, 128, 2, 4, 1, 4, false, false >( a, C, stream );
    case I8Kernel::TILE_256x128: return launch_shape< 256, 128, 4, 2, 1, 3, false, false >( a, C, stream );
    case I8Kernel::TILE_256x256: return launch_shape< 256, 256, 4, 2, 1, 2, false, false >( a, C, stream );
    case I8Kernel::SHIFT_32x32:   return launch_shape< 32, 32, 1, 1, 4, 3, true, true >( a, C, stream );
    case I8Kernel::SHIFT_64x64:   return launch_shape< 64, 64, 2, 2, 1, 3, true, true >( a, C, stream );
    case I8Kernel::SHIFT_128x128: return launch_shape< 128, 128, 2, 4, 1, 3, false, true >( a, C, stream );
    case I8Kernel::SHIFT_256x128: return launch_shape< 256, 128, 4, 2, 1, 2, false, true >( a, C, stream );
    default: return fail( ETIR_COMPILATION_FAILED, "contraction_i8: unknown tile" );
  }
}

}  // namespace etir
