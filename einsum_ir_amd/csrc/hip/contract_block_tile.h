// gfx950 product of 8-bit floating point blocks, or of bf16, with or without
// groups, tiles staged through LDS:
//
//   out[c][m][n] = last( sum_kb sa[c][m][kb] sb[c][n][kb] sum_(k in kb) A[c][m][k] B[c][n][k] + bias[c][n] )
//
// A workgroup computes a BM x BN tile, a wave a block of TM x TN fragments of
// 16 x 16.  A step takes 128 bytes of k of every row: one block of 128 8-bit
// numbers or 64 bf16.
//
// Operands go from global memory into LDS directly (buffer_load ... lds), STAGES
// steps deep, one barrier a step.  An operand that is unit-stride along k lies
// there as [row][128 bytes], 16-byte piece g of row r at place g ^ swz(r), and a
// fragment is two 16-byte reads a lane.  One that is unit-stride along its rows
// lies as [k][row], the pieces of a k likewise exchanged, and a fragment is four
// transposing reads (ds_read_b64_tr_b8 / _tr_b16).  A lane of either holds row
// lane % 16 and two pieces of its k; which these are does not matter as long as
// both operands agree.
//
// The columns' side is the first operand of the matrix instruction, so a lane
// holds one row m and 4 neighbouring columns; the tile goes out through LDS in
// rows of 16-byte stores.
//
// How a block's sum is made (KIND):
//   BF16    v_mfma_f32_16x16x32_bf16 onto the accumulators.
//   F8      v_mfma_f32_16x16x128_f8f6f4 from zero, then one fused multiply-add
//           with the product of the block's scales: 4 for each matrix
//           instruction of 32 cycles.  The matrix cores add 8-bit products in
//           groups of 8, cut 13 binary places below the largest (measured), a
//           relative error of 2^-16 of a sum of normal numbers, which bf16
//           outputs (2^-9) do not show.
//   EXACT   fp32 outputs: the 8-bit numbers become bf16 between LDS and the
//           matrix cores, where products are exact and sums fp32, at half the
//           rate.  EXACT_E8M0: with scales of a byte, become fp32 where they
//           are read (a branch on their type in the loop let the compiler put
//           all scaling behind the last of them, past the matrix instructions:
//           gradient of weights 8192 x 4096 x 2048 164 -> 134 us without it).
//   E8M0    as F8, the scales applied by the matrix instruction itself.
//
// Bound by the matrix cores' power where the tiles are many: 8192^3 with inputs
// that change from call to call takes 446 us with E8M0 (2.5 PFLOP/s, matrix cores
// busy 61 % at 1.9 of 2.4 GHz), 487 with F8, 972 with EXACT; bf16, 16384 rows in 8
// groups times 4096 x 4096, 491 us (1.12 PFLOP/s).  With the same inputs again and
// again: 428, 462, 949 and 470.  Large tiles read LDS least for a product, small ones fill the
// compute units: 4072 x 2048 x 2048 takes 39 us with 64 x 64, 24 with 128 x 128, 21
// with 256 x 128 (one round of 256 tiles) and 29 with 256 x 256 (half of one).
#ifndef ETIR_CONTRACT_BLOCK_TILE_H
#define ETIR_CONTRACT_BLOCK_TILE_H

#include "block_internal.h"
#include "contract_dma.h"

namespace etir {
namespace block {

using kern::i32x4;
typedef int32_t i32x2 __attribute__( ( ext_vector_type( 2 ) ) );
typedef int32_t i32x8 __attribute__( ( ext_vector_type( 8 ) ) );
typedef float   f32x4 __attribute__( ( ext_vector_type( 4 ) ) );
typedef __bf16  bf16x2 __attribute__( ( ext_vector_type( 2 ) ) );
typedef __bf16  bf16x8 __attribute__( ( ext_vector_type( 8 ) ) );

enum Kind : int { BF16, F8, EXACT, E8M0, EXACT_E8M0 };

constexpr int kStep = 128;      // bytes of k of a step

// Slots of 16 bytes of one k of an operand that lies along its rows, and by what
// they are exchanged: the 8-byte (f8: of 8 k, bf16: of 4) transposing reads of 16
// lanes, and of the 16 beside them, touch every bank once.
template< int ROWS, int ITEM >
__device__ inline uint32_t swz_rows( int k ) {
  constexpr int SLOTS = ROWS * ITEM / 16;
  if constexpr( ITEM == 1 ) {
    constexpr int P = 16 / SLOTS;                  // k in 256 bytes
    return uint32_t( k / P % ( 8 / P ) + ( k >> 5 & 1 ) * ( 8 / P ) );
  }
  else if constexpr( SLOTS >= 16 ) return uint32_t( 2 * ( k & 3 ) + 8 * ( k >> 4 & 1 ) );
  else if constexpr( SLOTS == 8 ) return uint32_t( 2 * ( k >> 1 & 1 ) + 4 * ( k >> 4 & 1 ) );
  else return uint32_t( 2 * ( k >> 4 & 1 ) );
}

// One operand's ROWS rows of a step, loaded directly by WAVES waves, 64 pieces of 16
// bytes at a time.
template< int ROWS, int WAVES, bool ALONG_ROWS, int ITEM >
struct Side {
  static constexpr int LOADS = ROWS / 8;
  static constexpr int EACH  = LOADS / WAVES;      // a wave's
  static constexpr int BYTES = ROWS * kStep;
  static constexpr int K     = kStep / ITEM;       // k of a step
  static_assert( LOADS % WAVES == 0, "loads have to divide over the waves" );

  uint32_t     m_off[EACH];      // bytes from the step's first to the lane's piece
  int          m_k[2];           // along k: the lane's byte of the step in even and odd loads
  uint32_t     m_first;          // the wave's first load
  uint8_t const * m_base;
  int64_t      m_stride;         // along rows: bytes from k to k
  int32_t      m_extent;         // along rows: bytes of a k from the tile's first row to the tensor's last
  i32x4        m_rsrc;

  // tile: the first row at k = 0; stride: bytes from row to row, or (along rows)
  // from k to k; rows: of the tensor from there on
  __device__ inline void init( uint8_t const * tile, int64_t stride, int32_t rows, int wave, int lane ) {
    m_first = wave * EACH;
    m_base = tile;
    m_stride = stride;
    if constexpr( ALONG_ROWS ) {
      constexpr int SLOTS = ROWS * ITEM / 16, PER = 64 / SLOTS;      // k of a load
      // to the last dword: its bytes past the tensor are in the same dword as the last row
      m_extent = ( rows * ITEM + 3 ) & ~3;
#pragma unroll
      for( int l_i = 0; l_i < EACH; l_i++ ) {
        int const l_k = ( int( m_first ) + l_i ) * PER + lane / SLOTS;
        m_off[l_i] = uint32_t( l_k * int32_t( stride ) ) + 16u * ( uint32_t( lane % SLOTS ) ^ swz_rows< ROWS, ITEM >( l_k ) );
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
        m_off[l_i] = uint32_t( l_r * int32_t( stride ) + m_k[( m_first + l_i ) % 2] );
      }
    }
  }
  // the step of which the next loads are; k: all of the sum's
  __device__ __attribute__( ( always_inline ) ) inline void at_step( int32_t step, int32_t k ) {
    if constexpr( ALONG_ROWS ) {
      // k past the end lie past the buffer's last byte: they load zeros
      int32_t const l_left = min( k - step * K, K );
      uint32_t const l_bytes = l_left > 0 ? uint32_t( l_left - 1 ) * uint32_t( m_stride ) + uint32_t( m_extent ) : 0u;
      m_rsrc = kern::make_rsrc( m_base + int64_t( step ) * K * m_stride, l_bytes );
    }
  }
  // starts the wave's load I of a step into lds
  template< int I >
  __device__ __attribute__( ( always_inline ) ) inline void issue( uint32_t lds, int32_t step, int32_t k ) {
    uint32_t l_off = m_off[I], l_soff = 0;
    if constexpr( !ALONG_ROWS ) {
      // k is a multiple of 16 bytes, so a lane's piece is inside or outside; outside: zeros
      int32_t const l_at = step * kStep, l_bytes = k * ITEM;
      if( l_at + kStep > l_bytes && l_at + m_k[( m_first + I ) % 2] >= l_bytes ) l_off = kern::kDmaOob;
      l_soff = uint32_t( l_at );
    }
    kern::set_m0( lds + ( m_first + I ) * 1024 );
    kern::dma16_so< 0 >( m_rsrc, l_off, l_soff );
  }
};

// The first of the two pieces (the other is 4 further) of a lane.  16-byte reads
// take lanes 0-3, 12-15 and 20-27 together, then 4-11, 16-19 and 28-31: pieces 0
// and 2 of lanes next to each other then touch every bank once, pieces 0 and 1
// half of them twice.
__device__ inline int first_piece( int lane ) { return ( lane >> 5 & 1 ) + 2 * ( lane >> 4 & 1 ); }

// 16 rows x 128 bytes of k: a lane's two pieces of 16 bytes
struct Frag { i32x4 v[2]; };

// Reads fragments of an operand's side.
template< int ROWS, bool ALONG_ROWS, int ITEM >
struct Reader {
  typedef short v4i16 __attribute__( ( ext_vector_type( 4 ) ) );
  typedef __attribute__( ( address_space( 3 ) ) ) v4i16 lds_v4i16;
  typedef __attribute__( ( address_space( 3 ) ) ) i32x2 lds_v2i32;
  int      m_lane;
  uint32_t m_k[4];          // along rows: bytes to the k of the lane's four reads
  uint32_t m_swz[4];

  __device__ inline void init( int lane ) {
    m_lane = lane;
    if constexpr( ALONG_ROWS ) {
#pragma unroll
      for( int l_i = 0; l_i < 4; l_i++ ) {
        // a piece has 16 / ITEM k, read 8 / ITEM at a time
        int const l_piece = first_piece( lane ) + 4 * ( l_i / 2 );
        int const l_k = l_piece * ( 16 / ITEM ) + ( l_i % 2 ) * ( 8 / ITEM ) + lane % 16 / ( ITEM == 1 ? 2 : 4 );
        m_k[l_i] = uint32_t( l_k * ROWS * ITEM );
        m_swz[l_i] = swz_rows< ROWS, ITEM >( l_k );
      }
    }
  }
  // the fragment of rows row .. row + 15 (a multiple of 16)
  __device__ __attribute__( ( always_inline ) ) inline Frag read( char const * lds, int row ) const {
    Frag l_f;
    if constexpr( !ALONG_ROWS ) {
      int const l_r = row + m_lane % 16;
      uint32_t const l_swz = kern::swz_k( m_lane % 16 );      // of rows 16 apart: the same
#pragma unroll
      for( int l_i = 0; l_i < 2; l_i++ ) {
        l_f.v[l_i] = *reinterpret_cast< i32x4 const * >( lds + l_r * kStep + ( ( uint32_t( first_piece( m_lane ) + 4 * l_i ) ^ l_swz ) << 4 ) );
      }
    }
    else {
#pragma unroll
      for( int l_i = 0; l_i < 4; l_i++ ) {
        // f8: lanes 2 j and 2 j + 1 read the 16 rows of k j; bf16: lanes 4 j to 4 j + 3
        i32x2 l_v;
        if constexpr( ITEM == 1 ) {
          char const * l_p = lds + m_k[l_i] + ( ( uint32_t( row / 16 ) ^ m_swz[l_i] ) << 4 ) + 8 * ( m_lane & 1 );
          l_v = __builtin_amdgcn_ds_read_tr8_b64_v2i32( (lds_v2i32 *) l_p );
        }
        else {
          char const * l_p = lds + m_k[l_i] + ( ( uint32_t( row / 8 + ( m_lane >> 1 & 1 ) ) ^ m_swz[l_i] ) << 4 ) + 8 * ( m_lane & 1 );
          l_v = __builtin_bit_cast( i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16( (lds_v4i16 *) l_p ) );
        }
        l_f.v[l_i / 2][2 * ( l_i % 2 )] = l_v[0];
        l_f.v[l_i / 2][2 * ( l_i % 2 ) + 1] = l_v[1];
      }
    }
    return l_f;
  }
};

// 32 8-bit numbers as four operands of 8 bf16
struct Wide { bf16x8 v[4]; };
template< bool E5M2 >
__device__ __attribute__( ( always_inline ) ) inline Wide widen( Frag const & f ) {
  Wide l_w;
#pragma unroll
  for( int l_i = 0; l_i < 8; l_i++ ) {
    int const l_d = f.v[l_i / 4][l_i % 4];
    bf16x2 l_lo, l_hi;
    if constexpr( E5M2 ) {
      l_lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8( l_d, 1.0f, false );
      l_hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8( l_d, 1.0f, true );
    }
    else {
      l_lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8( l_d, 1.0f, false );
      l_hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8( l_d, 1.0f, true );
    }
    l_w.v[l_i / 2][4 * ( l_i % 2 )] = l_lo[0];
    l_w.v[l_i / 2][4 * ( l_i % 2 ) + 1] = l_lo[1];
    l_w.v[l_i / 2][4 * ( l_i % 2 ) + 2] = l_hi[0];
    l_w.v[l_i / 2][4 * ( l_i % 2 ) + 3] = l_hi[1];
  }
  return l_w;
}

// What a workgroup computes: tile of BM x BN of batch or group c.
struct Where {
  int32_t c, m0, m_end, n0;
  int32_t k_begin, K;
  bool    any;
};

// Neighbouring tiles on one XCD (workgroups go to the 8 XCDs in turn), and there
// in bands of 8 tile rows, so that its cache serves both operands.
template< int BM, int BN >
__device__ inline Where where( BlockFast const & a ) {
  bool const l_grouped = a.has( BlockArgs::GROUP_ROWS );
  int32_t const l_tiles_n = ( a.N + BN - 1 ) / BN;
  // rows of tiles: the groups may have fewer than the grid, whose last ones
  // would else all be missing on the same XCD (with offsets that do not rise
  // they may have more, which are left out)
  int32_t const l_tiles_m = l_grouped ? min( block_tiles< BM >( a.offsets(), a.groups(), a.M ), a.M / BM + min( a.M, a.groups() ) )
                                      : ( a.M + BM - 1 ) / BM;
  int32_t const l_per_c = l_tiles_m * l_tiles_n, l_each = l_per_c / 8;
  Where l_w;
  l_w.any = !l_grouped || int64_t( blockIdx.x ) < l_per_c;
  if( !l_w.any ) return l_w;
  l_w.c = int32_t( blockIdx.x / uint32_t( l_per_c ) );
  int32_t l_r = int32_t( blockIdx.x % uint32_t( l_per_c ) );
  if( l_r < 8 * l_each ) l_r = l_r % 8 * l_each + l_r / 8;
  int32_t const l_band = l_r / ( 8 * l_tiles_n ) * 8;
  int32_t const l_high = min( 8, l_tiles_m - l_band );
  int32_t const l_tile_m = l_band + l_r % ( 8 * l_tiles_n ) % l_high;
  l_w.n0 = ( l_r % ( 8 * l_tiles_n ) / l_high ) * BN;
  l_w.m0 = l_tile_m * BM;
  l_w.m_end = a.M;
  l_w.k_begin = 0;
  l_w.K = a.K;
  if( l_grouped ) {
    BlockRows const l_rows = block_rows< BM >( a.offsets(), a.groups(), a.M, l_tile_m );
    l_w.any = l_rows.group >= 0;
    l_w.c = l_rows.group;
    l_w.m0 = l_rows.m0;
    l_w.m_end = l_rows.end;
  }
  else if( a.has( BlockArgs::GROUP_K ) ) {
    // The longest groups first, so that none is begun last (16 groups of 8192 rows,
    // 2048 x 2048 each 98 -> 94 us).  Every workgroup ranks the groups, so for large
    // tiles and up to 32 groups only: more of them are short against a launch (64:
    // 65.7 -> 66.2 us), and small tiles lose more than they gain (64 x 64 of 32 groups
    // 269 -> 337 us).
    if( BM * BN >= 256 * 256 && a.groups() <= 32 ) l_w.c = block_nth_longest( a.offsets(), a.groups(), a.K, l_w.c );
    BlockGroup const l_g = block_group( a.offsets(), l_w.c, a.K );
    l_w.k_begin = l_g.begin;
    l_w.K = l_g.end - l_g.begin;
  }
  return l_w;
}

// The scales of a step: those of A's rows, then of B's, a dword each in LDS
// (E8M0: the byte), 64 a load; a side of 32 rows has a load of its own.  Every
// wave has EACH loads, those past the last one load zeros.
template< int BM, int BN, int WAVES >
struct Scales {
  static constexpr int LOADS_A = ( BM + 63 ) / 64, LOADS_B = ( BN + 63 ) / 64;
  static constexpr int EACH  = ( LOADS_A + LOADS_B + WAVES - 1 ) / WAVES;
  static constexpr int BYTES = EACH * WAVES * 256;
  static constexpr int AT_B  = LOADS_A * 256;
  uint32_t m_off[EACH];      // bytes from block kb = 0 to the lane's scale
  uint32_t m_k[EACH];        // bytes from block to block of k
  i32x4    m_rsrc[EACH];
  uint32_t m_first;

  __device__ inline void init( BlockFast const & a, Where const & w, int wave, int lane ) {
    int const l_item = a.has( BlockArgs::E8M0 ) ? 1 : 4;
    m_first = wave * EACH;
#pragma unroll
    for( int l_i = 0; l_i < EACH; l_i++ ) {
      int const l_load = int( m_first ) + l_i;
      bool const l_a = l_load < LOADS_A;
      int32_t const l_at = 64 * ( l_a ? l_load : l_load - LOADS_A ) + lane;
      // rows past the tensor take the last one's scale and are not stored; the
      // tile's first row or block is in the base
      int32_t const l_first = l_a ? w.m0 : w.n0;
      int32_t const l_row = min( l_first + l_at, ( l_a ? w.m_end : a.N ) - 1 );
      bool const l_blocks = a.has( l_a ? BlockArgs::SA_BLOCKS : BlockArgs::SB_BLOCKS );
      int32_t const l_b0 = l_blocks ? l_first / kScaleBlock : l_first, l_b = l_blocks ? l_row / kScaleBlock : l_row;
      int64_t const l_stride = l_a ? a.sa_row : a.sb_row;
      void const * const l_s = l_a ? a.sa : a.sb;
      m_off[l_i] = l_s != nullptr && l_load < LOADS_A + LOADS_B ? uint32_t( ( l_b - l_b0 ) * int32_t( l_stride ) * l_item ) : kern::kDmaOob;
      m_k[l_i] = uint32_t( ( l_a ? a.sa_k : a.sb_k ) * l_item );
      m_rsrc[l_i] = kern::make_rsrc( static_cast< uint8_t const * >( l_s ) + ( int64_t( w.c ) * ( l_a ? a.sa_c : a.sb_c ) + l_b0 * l_stride ) * l_item,
                                     kern::kDmaOob );
    }
  }
  template< int I >
  __device__ __attribute__( ( always_inline ) ) inline void issue( uint32_t lds, int32_t step, int32_t blocks, bool e8m0 ) {
    uint32_t const l_off = step < blocks ? m_off[I] : kern::kDmaOob;
    uint32_t const l_soff = step < blocks ? uint32_t( step ) * m_k[I] : 0u;
    kern::set_m0( lds + ( m_first + I ) * 256 );
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    if( e8m0 ) asm volatile( "buffer_load_ubyte %0, %1, %2 offen lds" :: "v"( l_off ), "s"( m_rsrc[I] ), "s"( l_soff ) );
    else       asm volatile( "buffer_load_dword %0, %1, %2 offen lds" :: "v"( l_off ), "s"( m_rsrc[I] ), "s"( l_soff ) );
#pragma clang diagnostic pop
  }
};

// The same operand and scales through registers, for rows at any address: a
// step's pieces are loaded while the one in front of it is multiplied, and
// written to the places in LDS that the direct loads would give them.
template< int ROWS, int WAVES, bool ALONG_ROWS, int ITEM >
struct Staged {
  static constexpr int EACH = ROWS / 8 / WAVES, BYTES = ROWS * kStep, K = kStep / ITEM;
  static_assert( ROWS / 8 % WAVES == 0, "loads have to divide over the waves" );
  typedef i32x4 i32x4_any __attribute__( ( aligned( 1 ) ) );

  uint8_t const * m_base;
  int64_t  m_stride;
  int32_t  m_rows;
  int      m_wave, m_lane;
  int64_t  m_at[EACH];           // bytes from the step's first to the lane's piece
  i32x4    m_v[EACH];

  // along rows: the k and the byte of it of the wave's load i; along k: the byte of the step
  __device__ inline int k_of( int i ) const {
    constexpr int SLOTS = ROWS * ITEM / 16;
    return ( m_wave * EACH + i ) * ( 64 / SLOTS ) + m_lane / SLOTS;
  }
  __device__ inline int byte_of( int i ) const {
    if constexpr( ALONG_ROWS ) return 16 * int( uint32_t( m_lane % ( ROWS * ITEM / 16 ) ) ^ swz_rows< ROWS, ITEM >( k_of( i ) ) );
    else return 16 * ( ( m_lane % 8 ) ^ int( kern::swz_k( 8 * ( m_wave * EACH + i ) + m_lane / 8 ) ) );
  }
  __device__ inline void init( uint8_t const * tile, int64_t stride, int32_t rows, int wave, int lane ) {
    m_base = tile;
    m_stride = stride;
    m_rows = rows;
    m_wave = wave;
    m_lane = lane;
#pragma unroll
    for( int l_i = 0; l_i < EACH; l_i++ ) {
      // along k: rows past the tensor read its last one and are not stored
      m_at[l_i] = ( ALONG_ROWS ? k_of( l_i ) : min( 8 * ( wave * EACH + l_i ) + lane / 8, rows - 1 ) ) * stride + byte_of( l_i );
    }
  }
  __device__ __attribute__( ( always_inline ) ) inline void load( int32_t step, int32_t k ) {
    uint8_t const * const l_base = m_base + int64_t( step ) * ( ALONG_ROWS ? K * m_stride : int64_t( kStep ) );
    // Whether all 16 bytes of every piece are there; what follows a k's rows is
    // not stored and may be read, up to the end of the last k's.
    int64_t const l_after = int64_t( k ) - int64_t( step + 1 ) * K;      // k behind this step's
    if( ALONG_ROWS ? l_after >= 0 && l_after * m_stride + int64_t( m_rows ) * ITEM >= ROWS * ITEM : l_after >= 0 ) {
#pragma unroll
      for( int l_i = 0; l_i < EACH; l_i++ ) m_v[l_i] = *reinterpret_cast< i32x4_any const * >( l_base + m_at[l_i] );
      return;
    }
#pragma unroll
    for( int l_i = 0; l_i < EACH; l_i++ ) {
      int64_t l_left;            // bytes that are there
      if constexpr( ALONG_ROWS ) {
        int64_t const l_ks = l_after + K - 1 - k_of( l_i );      // k behind this one
        l_left = l_ks >= 0 ? int64_t( m_rows ) * ITEM - byte_of( l_i ) + l_ks * m_stride : 0;
      }
      else l_left = ( l_after + K ) * ITEM - byte_of( l_i );
      uint8_t const * const l_p = l_base + m_at[l_i];
      m_v[l_i] = i32x4{ 0, 0, 0, 0 };
      if( l_left >= 16 ) m_v[l_i] = *reinterpret_cast< i32x4_any const * >( l_p );
      else if( l_left > 0 ) {
        // the end, byte by byte (bf16: two)
#pragma unroll
        for( int l_e = 0; l_e < 16 / ITEM; l_e++ ) {
          if( l_e * ITEM >= l_left ) continue;
          uint32_t const l_x = ITEM == 1 ? uint32_t( l_p[l_e] ) : uint32_t( reinterpret_cast< uint16_t const * >( l_p )[l_e] );
          m_v[l_i][l_e * ITEM / 4] |= int32_t( l_x << ( 8 * ( l_e * ITEM % 4 ) ) );
        }
      }
    }
  }
  __device__ __attribute__( ( always_inline ) ) inline void store( char * lds ) const {
#pragma unroll
    for( int l_i = 0; l_i < EACH; l_i++ ) {
      *reinterpret_cast< i32x4 * >( lds + ( m_wave * EACH + l_i ) * 1024 + 16 * m_lane ) = m_v[l_i];
    }
  }
};

// elements from row to row of a wave's output slab in LDS
template< class T, int COLS > constexpr int kPitch = COLS + 16 / int( sizeof( T ) );

// Stores 16 rows x COLS columns of a wave's slab, 16 bytes a lane, non-temporal:
// the output is not read here again.
template< int COLS, class T >
__device__ inline void store_slab( BlockFast const & a, T const * slab, T * out, int32_t m1, int32_t m_end, int32_t n1, int lane ) {
  constexpr int V = 16 / sizeof( T ), LANES = COLS / V, PITCH = kPitch< T, COLS >;
  typedef T v __attribute__( ( ext_vector_type( V ) ) );
  typedef v v_any __attribute__( ( aligned( sizeof( T ) ) ) );
#pragma unroll
  for( int l_p = 0; l_p < ( 16 * LANES + 63 ) / 64; l_p++ ) {
    int const l_i = l_p * 64 + lane;
    int const l_r = l_i / LANES, l_c = l_i % LANES * V;
    if( l_r >= 16 || m1 + l_r >= m_end ) continue;
    v const l_v = *reinterpret_cast< v const * >( slab + l_r * PITCH + l_c );
    T * const l_o = out + int64_t( m1 + l_r ) * a.o_row + n1 + l_c;
    int32_t const l_left = a.N - n1 - l_c;       // columns from this lane's first on
    if( l_left >= V ) __builtin_nontemporal_store( l_v, reinterpret_cast< v_any * >( l_o ) );
    else {
#pragma unroll
      for( int l_e = 0; l_e < V; l_e++ ) if( l_e < l_left ) l_o[l_e] = l_v[l_e];
    }
  }
}

// KIND: see above.  RA, RB: A (B) is unit-stride along its rows, else along k.
// SB_ROWS: B has a scale for every row (F8 and EXACT), else one for 128.  KG
// groups of WM x WN waves take the steps in turn, each with STAGES buffers of its
// own, and add their sums in LDS at the end, in the groups' order: few tiles with
// a long K keep more loads and waves on a compute unit.  REG: operands at any
// address, through registers (two buffers).
template< int KIND, int BM, int BN, int WM, int WN, int KG, int STAGES, bool RA, bool RB, bool A_E5M2, bool SB_ROWS, bool REG >
__global__ __launch_bounds__( 64 * WM * WN * KG )
void contract_block_tile_kernel( BlockFast a ) {
  constexpr int  ITEM = KIND == BF16 ? 2 : 1;
  constexpr bool SCALED = KIND != BF16;
  constexpr bool WIDENED = KIND == EXACT || KIND == EXACT_E8M0;
  constexpr int  WAVES = WM * WN;                            // of a group
  constexpr int  TM = BM / WM / 16, TN = BN / WN / 16;       // fragments of a wave
  constexpr int  COLS = BN / WN;
  static_assert( TN % 2 == 0 && ( KIND == BF16 || KIND == E8M0 || SB_ROWS || COLS <= kScaleBlock ), "wave tile" );
  static_assert( !REG || STAGES == 2, "two buffers" );
  typedef std::conditional_t< REG, Staged< BM, WAVES, RA, ITEM >, Side< BM, WAVES, RA, ITEM > > SideA;
  typedef std::conditional_t< REG, Staged< BN, WAVES, RB, ITEM >, Side< BN, WAVES, RB, ITEM > > SideB;
  typedef Scales< BM, BN, WAVES > SideS;
  constexpr int EACH = SideA::EACH + SideB::EACH + ( SCALED ? SideS::EACH : 0 );      // a wave's loads of a step
  constexpr int STAGE = SideA::BYTES + SideB::BYTES + ( SCALED ? SideS::BYTES : 0 );
  constexpr int SLAB = 16 * kPitch< float, COLS > * 4;
  constexpr int SLABS = WAVES * SLAB, PARTS = ( KG - 1 ) * BM * BN * 4;
  constexpr int BYTES = KG * STAGES * STAGE > SLABS + PARTS ? KG * STAGES * STAGE : SLABS + PARTS;
  __shared__ __align__( 16 ) char l_all[BYTES];
  __shared__ __align__( 16 ) float l_bias[BN];
  static_assert( BN <= 64 * WAVES * KG, "a thread a column" );

  int const l_lane = threadIdx.x % 64;
  int const l_w = __builtin_amdgcn_readfirstlane( threadIdx.x / 64 );
  int const l_group = l_w / WAVES, l_wave = l_w % WAVES;
  char * const l_lds = l_all + l_group * ( STAGES * STAGE );      // the group's buffers
  int const l_wm = l_wave / WN * ( BM / WM ), l_wn = l_wave % WN * COLS;
  Where const w = where< BM, BN >( a );
  if( !w.any ) return;

  uint8_t const * const l_at_a = static_cast< uint8_t const * >( a.a ) + ( w.c * a.a_batch() + ( RA ? w.m0 + w.k_begin * int64_t( a.a_ld ) : w.m0 * int64_t( a.a_ld ) + w.k_begin ) ) * ITEM;
  uint8_t const * const l_at_b = static_cast< uint8_t const * >( a.b ) + ( w.c * int64_t( a.b_c ) + ( RB ? w.n0 + w.k_begin * int64_t( a.b_ld ) : w.n0 * int64_t( a.b_ld ) + w.k_begin ) ) * ITEM;
  SideA l_a;
  SideB l_b;
  SideS l_s;
  l_a.init( l_at_a, int64_t( a.a_ld ) * ITEM, w.m_end - w.m0, l_wave, l_lane );
  l_b.init( l_at_b, int64_t( a.b_ld ) * ITEM, a.N - w.n0, l_wave, l_lane );
  if constexpr( SCALED && !REG ) l_s.init( a, w, l_wave, l_lane );
  Reader< BM, RA, ITEM > l_ra;
  Reader< BN, RB, ITEM > l_rb;
  l_ra.init( l_lane );
  l_rb.init( l_lane );

  // the bias, needed after the loop
  float l_bias_r = 0.0f;
  if( a.bias() && threadIdx.x < BN ) l_bias_r = a.bias()[min( w.n0 + int32_t( threadIdx.x ), a.N - 1 )];

  int32_t const l_blocks = int32_t( ( int64_t( w.K ) * ITEM + kStep - 1 ) / kStep );
  // A group's steps; past the last block nothing is in range and zeros are
  // loaded, so that all groups take as many.
  int32_t const l_steps = ( l_blocks + KG - 1 ) / KG;
  uint32_t const l_lds_at = kern::lds_addr( l_lds );

  // REG: the thread's scale (of the first threads of a group) of the step that
  // is on its way, as fp32; without scales 1
  float l_scale_r = 1.0f;
  int const l_gt = l_wave * 64 + l_lane;
  auto load_regs = [&]( int32_t s ) __attribute__( ( always_inline ) ) {
    if constexpr( REG ) {
      int32_t const l_step = s * KG + l_group;
      l_a.load( l_step, w.K );
      l_b.load( l_step, w.K );
      if constexpr( SCALED ) {
        static_assert( BM + BN <= 64 * WAVES, "a thread a scale" );
        bool const l_is_a = l_gt < BM;
        void const * const l_p = l_is_a ? a.sa : a.sb;
        if( l_p != nullptr && l_gt < BM + BN && l_step < l_blocks ) {
          int32_t const l_row = l_is_a ? min( w.m0 + l_gt, w.m_end - 1 ) : min( w.n0 + l_gt - BM, a.N - 1 );
          bool const l_by = a.has( BlockArgs::SA_BLOCKS ) && l_is_a ? true : a.has( BlockArgs::SB_BLOCKS ) && !l_is_a;
          int64_t const l_i = int64_t( w.c ) * ( l_is_a ? a.sa_c : a.sb_c ) + int64_t( l_step ) * ( l_is_a ? a.sa_k : a.sb_k )
                            + int64_t( l_by ? l_row / kScaleBlock : l_row ) * ( l_is_a ? a.sa_row : a.sb_row );
          if( a.has( BlockArgs::E8M0 ) ) l_scale_r = e8m0_to_f32( static_cast< uint8_t const * >( l_p )[l_i] );
          else                           l_scale_r = static_cast< float const * >( l_p )[l_i];
        }
      }
    }
  };
  auto store_regs = [&]( int stage ) __attribute__( ( always_inline ) ) {
    if constexpr( REG ) {
      char * const l_to = l_lds + stage * STAGE;
      l_a.store( l_to );
      l_b.store( l_to + SideA::BYTES );
      if constexpr( SCALED ) {
        if( l_gt < BM + BN ) {
          *reinterpret_cast< float * >( l_to + SideA::BYTES + SideB::BYTES + ( l_gt < BM ? 4 * l_gt : SideS::AT_B + 4 * ( l_gt - BM ) ) ) = l_scale_r;
        }
      }
    }
  };
  // the wave's load i of a step, those of both sides and the scales counted through
  auto issue = [&]( auto ic, int stage, int32_t s ) __attribute__( ( always_inline ) ) {
    if constexpr( !REG ) {
      constexpr int l_i = decltype( ic )::value;
      int32_t const l_step = s * KG + l_group;
      uint32_t const l_to = l_lds_at + stage * STAGE;
      if constexpr( l_i < SideA::EACH ) {
        if constexpr( l_i == 0 ) l_a.at_step( l_step, w.K );
        l_a.template issue< l_i >( l_to, l_step, w.K );
      }
      else if constexpr( l_i < SideA::EACH + SideB::EACH ) {
        if constexpr( l_i == SideA::EACH ) l_b.at_step( l_step, w.K );
        l_b.template issue< l_i - SideA::EACH >( l_to + SideA::BYTES, l_step, w.K );
      }
      else if constexpr( SCALED ) {
        l_s.template issue< l_i - SideA::EACH - SideB::EACH >( l_to + SideA::BYTES + SideB::BYTES, l_step, l_blocks,
                                                               KIND == E8M0 || KIND == EXACT_E8M0 );
      }
    }
  };
  // loads of step 1 (two buffers) that are issued in front of the loop
  constexpr int EARLY = ( EACH + 1 ) / 2;
  if constexpr( REG ) {
    load_regs( 0 );
    store_regs( 0 );
    load_regs( 1 );
    kern::wait_lgkmcnt0();
  }
  else {
    kern::static_for< EACH >( [&]( auto ic ) __attribute__( ( always_inline ) ) { issue( ic, 0, 0 ); } );
    if constexpr( STAGES > 2 ) {
      kern::static_for< STAGES - 2 >( [&]( auto sc ) __attribute__( ( always_inline ) ) {
        constexpr int l_st = decltype( sc )::value + 1;
        kern::static_for< EACH >( [&]( auto ic ) __attribute__( ( always_inline ) ) { issue( ic, l_st, l_st ); } );
      } );
      kern::wait_vmcnt< ( STAGES - 2 ) * EACH >();
    }
    else {
      kern::static_for< EARLY >( [&]( auto ic ) __attribute__( ( always_inline ) ) { issue( ic, 1, 1 ); } );
      kern::wait_vmcnt< EARLY >();
    }
  }
  kern::barrier_lds();

  f32x4 l_acc[TN][TM];
#pragma unroll
  for( int l_i = 0; l_i < TN * TM; l_i++ ) l_acc[l_i / TM][l_i % TM] = f32x4{ 0.0f, 0.0f, 0.0f, 0.0f };
  Frag l_fa[TM], l_fb[2];
  // scales: a row's of each fragment of A, and B's: of the 128 columns, or of a
  // lane's 4 columns (E8M0: of the lane's row) of two fragments
  int32_t l_sa[TM], l_sb1 = 0;
  i32x4 l_sb[2];
  auto scale_value = [&]( int32_t bits ) __attribute__( ( always_inline ) ) -> float {
    return KIND == EXACT_E8M0 ? e8m0_to_f32( uint32_t( bits ) ) : __uint_as_float( uint32_t( bits ) );
  };
  auto read_a = [&]( auto ic, int stage ) __attribute__( ( always_inline ) ) {
    constexpr int l_i = decltype( ic )::value;
    l_fa[l_i] = l_ra.read( l_lds + stage * STAGE, l_wm + 16 * l_i );
  };
  auto read_b = [&]( auto jc, int stage ) __attribute__( ( always_inline ) ) {
    constexpr int l_j = decltype( jc )::value;
    l_fb[l_j % 2] = l_rb.read( l_lds + stage * STAGE + SideA::BYTES, l_wn + 16 * l_j );
    char const * const l_sc = l_lds + stage * STAGE + SideA::BYTES + SideB::BYTES + SideS::AT_B;
    if constexpr( SCALED && KIND != E8M0 && SB_ROWS ) {
      l_sb[l_j % 2] = *reinterpret_cast< i32x4 const * >( l_sc + 4 * ( l_wn + 16 * l_j + 4 * ( l_lane / 16 ) ) );
    }
    if constexpr( KIND == E8M0 ) l_sb[l_j % 2][0] = *reinterpret_cast< int32_t const * >( l_sc + 4 * ( l_wn + 16 * l_j + l_lane % 16 ) );
  };
  // the scales of A's rows (and of the 128 columns) of a step
  auto read_s = [&]( int stage ) __attribute__( ( always_inline ) ) {
    if constexpr( SCALED ) {
      char const * const l_sc = l_lds + stage * STAGE + SideA::BYTES + SideB::BYTES;
#pragma unroll
      for( int l_i = 0; l_i < TM; l_i++ ) l_sa[l_i] = *reinterpret_cast< int32_t const * >( l_sc + 4 * ( l_wm + 16 * l_i + l_lane % 16 ) );
      if constexpr( KIND != E8M0 && !SB_ROWS ) l_sb1 = *reinterpret_cast< int32_t const * >( l_sc + SideS::AT_B + 4 * l_wn );
    }
  };

  // One step in TN parts, each a fragment of B against all of A's.  During a
  // part the next fragment of B is read; the barrier stands in front of the last
  // part, when every wave has read all of this step and the next one has landed,
  // and behind it A's fragments of the next step replace this one's as they
  // fall free.  Two buffers: the step after that is loaded over this one from
  // there on, half of it in the last part, half in the next step's first.  More:
  // the step STAGES - 1 ahead is loaded over the last one, spread over the parts
  // in front of the barrier.
  auto step = [&]( int l_st, int l_next, int l_free, int32_t s ) __attribute__( ( always_inline ) ) {
    float l_scale[TM];
    if constexpr( KIND == F8 || WIDENED ) {
      float const l_b1 = SB_ROWS ? 1.0f : scale_value( l_sb1 );
#pragma unroll
      for( int l_i = 0; l_i < TM; l_i++ ) l_scale[l_i] = scale_value( l_sa[l_i] ) * l_b1;
    }
    // F8, EXACT: the sums of a pair of fragments are added RING - 1 pairs later
    constexpr int RING = WIDENED ? 2 : 3;
    f32x4 l_part[RING];
    f32x4 l_of_b[2];        // SB_ROWS: the scales of the columns of this part and the last
    Wide l_wa[WIDENED ? TM : 1];
    if constexpr( WIDENED ) {
#pragma unroll
      for( int l_i = 0; l_i < TM; l_i++ ) l_wa[l_i] = widen< A_E5M2 >( l_fa[l_i] );
    }
    auto add = [&]( auto mc ) __attribute__( ( always_inline ) ) {
      constexpr int l_j = decltype( mc )::value / TM, l_i = decltype( mc )::value % TM;
      f32x4 const & l_p = l_part[decltype( mc )::value % RING];
#pragma unroll
      for( int l_e = 0; l_e < 4; l_e++ ) {
        float const l_f = SB_ROWS ? l_scale[l_i] * l_of_b[l_j % 2][l_e] : l_scale[l_i];
        l_acc[l_j][l_i][l_e] = fmaf( l_p[l_e], l_f, l_acc[l_j][l_i][l_e] );
      }
    };
    kern::static_for< TN >( [&]( auto jc ) __attribute__( ( always_inline ) ) {
      constexpr int l_j = decltype( jc )::value;
      constexpr bool LAST = l_j == TN - 1;
      // REG: the next step over the last one, which every wave has read
      if constexpr( REG && l_j == 0 ) {
        store_regs( l_next );
        load_regs( s + 2 );
      }
      if constexpr( LAST ) {
        if constexpr( !REG ) kern::wait_vmcnt< ( STAGES - 2 ) * EACH >();
        kern::wait_lgkmcnt0();
        kern::barrier_lds();
      }
      Frag const & l_f = l_fb[l_j % 2];
      int32_t l_bits_b = 0;
      if constexpr( KIND == E8M0 ) l_bits_b = l_sb[l_j % 2][0];
      if constexpr( ( KIND == F8 || WIDENED ) && SB_ROWS ) {
#pragma unroll
        for( int l_e = 0; l_e < 4; l_e++ ) l_of_b[l_j % 2][l_e] = scale_value( l_sb[l_j % 2][l_e] );
      }
      Wide l_wb;
      if constexpr( WIDENED ) l_wb = widen< false >( l_f );
      if constexpr( !LAST ) read_b( std::integral_constant< int, l_j + 1 >(), l_st );
      else                  read_b( std::integral_constant< int, 0 >(), l_next );
      kern::static_for< TM >( [&]( auto ic ) __attribute__( ( always_inline ) ) {
        constexpr int l_i = decltype( ic )::value, l_m = l_j * TM + l_i;
        constexpr f32x4 ZERO = { 0.0f, 0.0f, 0.0f, 0.0f };
        if constexpr( KIND == BF16 ) {
#pragma unroll
          for( int l_q = 0; l_q < 2; l_q++ ) {
            l_acc[l_j][l_i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16( __builtin_bit_cast( bf16x8, l_f.v[l_q] ),
                                                                       __builtin_bit_cast( bf16x8, l_fa[l_i].v[l_q] ), l_acc[l_j][l_i], 0, 0, 0 );
          }
        }
        else if constexpr( WIDENED ) {
          f32x4 l_p = ZERO;
#pragma unroll
          for( int l_q = 0; l_q < 4; l_q++ ) l_p = __builtin_amdgcn_mfma_f32_16x16x32_bf16( l_wb.v[l_q], l_wa[l_i].v[l_q], l_p, 0, 0, 0 );
          l_part[l_m % RING] = l_p;
          if constexpr( l_m >= RING - 1 ) add( std::integral_constant< int, l_m - RING + 1 >() );
        }
        else {
          i32x8 const l_vb = __builtin_shufflevector( l_f.v[0], l_f.v[1], 0, 1, 2, 3, 4, 5, 6, 7 );
          i32x8 const l_va = __builtin_shufflevector( l_fa[l_i].v[0], l_fa[l_i].v[1], 0, 1, 2, 3, 4, 5, 6, 7 );
          constexpr int FORMAT = A_E5M2 ? 1 : 0;
          if constexpr( KIND == E8M0 ) {
            l_acc[l_j][l_i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4( l_vb, l_va, l_acc[l_j][l_i], 0, FORMAT, 0, l_bits_b, 0,
                                                                                l_sa[l_i] );
          }
          else {
            l_part[l_m % RING] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4( l_vb, l_va, ZERO, 0, FORMAT, 0, 0, 0, 0 );
            if constexpr( l_m >= RING - 1 ) add( std::integral_constant< int, l_m - RING + 1 >() );
          }
        }
        if constexpr( LAST ) read_a( ic, l_next );
        if constexpr( !REG && STAGES > 2 && !LAST ) {
          constexpr int l_from = EACH * l_m / ( ( TN - 1 ) * TM ), l_to = EACH * ( l_m + 1 ) / ( ( TN - 1 ) * TM );
          kern::static_for< l_to - l_from >( [&]( auto dc ) __attribute__( ( always_inline ) ) {
            issue( std::integral_constant< int, l_from + decltype( dc )::value >(), l_free, s + STAGES - 1 );
          } );
        }
        if constexpr( !REG && STAGES == 2 && ( LAST || l_j == 0 ) ) {
          constexpr int l_p0 = LAST ? 0 : EARLY, l_n = LAST ? EARLY : EACH - EARLY;
          constexpr int l_from = l_p0 + l_n * l_i / TM, l_to = l_p0 + l_n * ( l_i + 1 ) / TM;
          kern::static_for< l_to - l_from >( [&]( auto dc ) __attribute__( ( always_inline ) ) {
            issue( std::integral_constant< int, l_from + decltype( dc )::value >(), LAST ? l_st : l_next, LAST ? s + 2 : s + 1 );
          } );
        }
        __builtin_amdgcn_sched_barrier( 0 );
      } );
    } );
    if constexpr( KIND == F8 || WIDENED ) {
      kern::static_for< RING - 1 >( [&]( auto rc ) __attribute__( ( always_inline ) ) {
        add( std::integral_constant< int, TN * TM - ( RING - 1 ) + decltype( rc )::value >() );
      } );
    }
    read_s( l_next );
  };
  if( l_steps > 0 ) {
    kern::static_for< TM >( [&]( auto ic ) __attribute__( ( always_inline ) ) { read_a( ic, 0 ); } );
    read_b( std::integral_constant< int, 0 >(), 0 );
    read_s( 0 );
  }
  int l_st = 0, l_free = STAGES - 1;
  for( int32_t l_step = 0; l_step < l_steps; l_step++ ) {
    int const l_next = l_st == STAGES - 1 ? 0 : l_st + 1;
    step( l_st, l_next, l_free, l_step );
    l_free = l_st;
    l_st = l_next;
  }
  kern::wait_vmcnt< 0 >();
  if( threadIdx.x < BN ) l_bias[threadIdx.x] = l_bias_r;
  __syncthreads();           // nothing is on its way into LDS, all fragments are read

  // the other groups' sums to the first one
  if constexpr( KG > 1 ) {
    f32x4 * const l_parts = reinterpret_cast< f32x4 * >( l_all + SLABS );
    if( l_group > 0 ) {
#pragma unroll
      for( int l_i = 0; l_i < TN * TM; l_i++ ) {
        l_parts[( ( ( l_group - 1 ) * WAVES + l_wave ) * TN * TM + l_i ) * 64 + l_lane] = l_acc[l_i / TM][l_i % TM];
      }
    }
    __syncthreads();
    if( l_group > 0 ) return;
    for( int l_g = 0; l_g < KG - 1; l_g++ ) {
#pragma unroll
      for( int l_i = 0; l_i < TN * TM; l_i++ ) l_acc[l_i / TM][l_i % TM] += l_parts[( ( l_g * WAVES + l_wave ) * TN * TM + l_i ) * 64 + l_lane];
    }
  }

  // 16 rows at a time through this wave's slab
  auto finish = [&]( auto zero ) __attribute__( ( always_inline ) ) {
    typedef decltype( zero ) T;
    typedef T t4 __attribute__( ( ext_vector_type( 4 ) ) );
    T * const l_slab = reinterpret_cast< T * >( l_all + l_wave * SLAB );
    T * const l_out = static_cast< T * >( a.out ) + int64_t( w.c ) * a.o_c;
#pragma unroll
    for( int l_i = 0; l_i < TM; l_i++ ) {
#pragma unroll
      for( int l_j = 0; l_j < TN; l_j++ ) {
        int const l_n = 16 * l_j + 4 * ( l_lane / 16 );
        f32x4 l_f = l_acc[l_j][l_i];
        if( a.bias() ) l_f += *reinterpret_cast< f32x4 const * >( l_bias + l_wn + l_n );
        if( a.has( BlockArgs::RELU ) ) {
#pragma unroll
          for( int l_e = 0; l_e < 4; l_e++ ) l_f[l_e] = l_f[l_e] < 0.0f ? 0.0f : l_f[l_e];      // a NaN stays
        }
        *reinterpret_cast< t4 * >( l_slab + ( l_lane % 16 ) * kPitch< T, COLS > + l_n )
            = t4{ static_cast< T >( l_f[0] ), static_cast< T >( l_f[1] ), static_cast< T >( l_f[2] ), static_cast< T >( l_f[3] ) };
      }
      // the slab is this wave's own, and its LDS operations are in order
      __builtin_amdgcn_fence( __ATOMIC_ACQ_REL, "wavefront" );
      store_slab< COLS, T >( a, l_slab, l_out, w.m0 + l_wm + 16 * l_i, w.m_end, w.n0 + l_wn, l_lane );
      __builtin_amdgcn_fence( __ATOMIC_ACQ_REL, "wavefront" );
    }
  };
  if( a.has( BlockArgs::OUT_BF16 ) ) finish( __bf16( 0.0f ) );
  else                               finish( 0.0f );
}

template< int KIND, int BM, int BN, int WM, int WN, int KG, int STAGES, bool RA, bool RB, bool A_E5M2, bool SB_ROWS, bool REG >
int launch_shape( BlockArgs const & a, hipStream_t stream ) {
  int64_t const l_tiles_n = ( int64_t( a.N ) + BN - 1 ) / BN;
  int64_t const l_tiles_m = a.has( BlockArgs::GROUP_ROWS ) ? block_most_tiles( a.M, a.C, BM ) : ( int64_t( a.M ) + BM - 1 ) / BM * a.C;
  hipLaunchKernelGGL( ( contract_block_tile_kernel< KIND, BM, BN, WM, WN, KG, STAGES, RA, RB, A_E5M2, SB_ROWS, REG > ),
                      dim3( uint32_t( l_tiles_m * l_tiles_n ) ), dim3( 64 * WM * WN * KG ), 0, stream,
                      BlockFast::of( a, RA, RB ) );
  hipError_t const l_e = hipGetLastError();
  if( l_e != hipSuccess ) {
    return fail( ETIR_UNDEFINED_ERROR, std::string( "contraction launch failed: " ) + hipGetErrorString( l_e ) );
  }
  return ETIR_SUCCESS;
}

// the tiles of one kind and layout, through LDS directly
template< int KIND, bool RA, bool RB, bool A_E5M2, bool SB_ROWS >
int launch_tiles( BlockArgs const & a, BlockKernel kernel, hipStream_t stream ) {
  switch( kernel ) {
    case BlockKernel::TILE_32x32:   return launch_shape< KIND, 32, 32, 1, 1, 8, 2, RA, RB, A_E5M2, SB_ROWS, false >( a, stream );
    case BlockKernel::TILE_64x64_K: return launch_shape< KIND, 64, 64, 2, 2, 4, 2, RA, RB, A_E5M2, SB_ROWS, false >( a, stream );
    case BlockKernel::TILE_64x64:   return launch_shape< KIND, 64, 64, 2, 2, 1, 4, RA, RB, A_E5M2, SB_ROWS, false >( a, stream );
    case BlockKernel::TILE_128x128: return launch_shape< KIND, 128, 128, 2, 2, 1, 2, RA, RB, A_E5M2, SB_ROWS, false >( a, stream );
    case BlockKernel::TILE_256x128: return launch_shape< KIND, 256, 128, 4, 2, 1, 3, RA, RB, A_E5M2, SB_ROWS, false >( a, stream );
    case BlockKernel::TILE_256x256:
      // the widened operands of EXACT leave no registers for it
      if constexpr( KIND != EXACT && KIND != EXACT_E8M0 ) return launch_shape< KIND, 256, 256, 4, 2, 1, 2, RA, RB, A_E5M2, SB_ROWS, false >( a, stream );
      [[fallthrough]];
    default: return fail( ETIR_COMPILATION_FAILED, "contraction: unknown tile" );
  }
}

// the tiles of one kind and layout, through registers
template< int KIND, bool RA, bool RB, bool A_E5M2, bool SB_ROWS >
int launch_staged( BlockArgs const & a, BlockKernel kernel, hipStream_t stream ) {
  switch( kernel ) {
    case BlockKernel::STAGED_32x32:    return launch_shape< KIND, 32, 32, 1, 1, 8, 2, RA, RB, A_E5M2, SB_ROWS, true >( a, stream );
    case BlockKernel::STAGED_64x64_K:  return launch_shape< KIND, 64, 64, 2, 2, 2, 2, RA, RB, A_E5M2, SB_ROWS, true >( a, stream );
    case BlockKernel::STAGED_64x64:    return launch_shape< KIND, 64, 64, 2, 2, 1, 2, RA, RB, A_E5M2, SB_ROWS, true >( a, stream );
    case BlockKernel::STAGED_128x128:  return launch_shape< KIND, 128, 128, 2, 4, 1, 2, RA, RB, A_E5M2, SB_ROWS, true >( a, stream );
    default: return fail( ETIR_COMPILATION_FAILED, "contraction: unknown tile" );
  }
}

}  // namespace block
}  // namespace etir

#endif
