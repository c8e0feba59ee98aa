// Declarations of the products of 8-bit floating point with a scale for each
// block of 128, of the products whose rows are grouped by expert (block_plan.cpp,
// contract_block*.hip) and of the operator that rounds to such blocks
// (quant_f8.hip).
#ifndef ETIR_BLOCK_INTERNAL_H
#define ETIR_BLOCK_INTERNAL_H

#include "etir_internal.h"
#include <algorithm>

namespace etir {

// k (and, where a side has blocks, rows) that share a scale
constexpr int kScaleBlock = 128;

// ---------------------------------------------------------------------------
// products
//   out[c,m,n] = last( sum_kb sa[c,m,kb] sb[c,n,kb] sum_(k in kb) A[c,m,k] B[c,n,k] + bias[c,n] )
// A: the left, B: the right tensor; one loop of each type.  Groups: rows of A
// (GROUP_ROWS) or indices k (GROUP_K) offsets[g] to offsets[g + 1] belong to
// group g, which is B's or the output's batch index.
// ---------------------------------------------------------------------------
struct BlockArgs {
  void const    * a;
  void const    * b;
  void const    * sa;       // null: 1
  void const    * sb;       // null: 1
  float const   * bias;     // null: 0
  int32_t const * offsets;  // groups only
  void          * out;
  // elements from index to index; scales: from block to block
  int64_t a_c, b_c, o_c, sa_c, sb_c, bias_c;
  int64_t a_row, a_k, b_row, b_k, o_row, o_col, sa_row, sa_k, sb_row, sb_k, bias_col;
  int32_t M, N, K, C;       // C: batches or groups
  uint32_t flags;

  enum : uint32_t { OUT_BF16 = 1u, RELU = 2u, GROUP_ROWS = 4u, GROUP_K = 8u, F8 = 16u, A_E5M2 = 32u, E8M0 = 64u,
                    SA_BLOCKS = 128u, SB_BLOCKS = 256u,     // a scale for 128 rows
                    SCALES = 512u,                          // both operands have scales
                    BIAS = 1024u };
  __host__ __device__ bool has( uint32_t flag ) const { return ( flags & flag ) != 0; }
};

// The same for all kernels but the general one: one stride an operand (the other
// is 1), the output unit-stride along N, the bias adjacent and the same for all
// batches, strides below 2^31.  112 bytes: a launch with up to so many in kernel
// arguments takes 2.7 to 2.9 us of the host, one with 120 to 1024 bytes 3.3 to
// 3.5 us.
struct BlockFast {
  void const * a;
  void const * b;
  void const * sa;
  void const * sb;
  void const * extra;       // offsets (groups) or bias
  void       * out;
  int32_t a_c;              // groups: how many
  int32_t b_c, o_c, sa_c, sb_c;
  int32_t a_ld, b_ld, o_row, sa_row, sa_k, sb_row, sb_k;
  int32_t M, N, K;
  uint32_t flags;           // of BlockArgs

  __host__ __device__ bool has( uint32_t flag ) const { return ( flags & flag ) != 0; }
  __host__ __device__ bool grouped() const { return has( BlockArgs::GROUP_ROWS | BlockArgs::GROUP_K ); }
  __device__ int32_t groups() const { return a_c; }
  __device__ int64_t a_batch() const { return grouped() ? 0 : a_c; }
  __device__ int32_t const * offsets() const { return static_cast< int32_t const * >( extra ); }
  __device__ float const * bias() const { return grouped() ? nullptr : static_cast< float const * >( extra ); }

  static bool fits( BlockArgs const & a ) {
    for( int64_t l_s : { a.a_c, a.b_c, a.o_c, a.sa_c, a.sb_c, a.a_row, a.a_k, a.b_row, a.b_k, a.o_row, a.sa_row, a.sa_k, a.sb_row, a.sb_k } ) {
      if( l_s >= ( int64_t( 1 ) << 31 ) ) return false;
    }
    return a.o_col == 1 && a.bias_c == 0 && ( a.bias_col == 1 || a.N < 2 || !a.has( BlockArgs::BIAS ) );
  }
  // along_rows_*: the operand is unit-stride along its rows
  static BlockFast of( BlockArgs const & a, bool along_rows_a, bool along_rows_b ) {
    BlockFast f;
    f.a = a.a;
    f.b = a.b;
    f.sa = a.sa;
    f.sb = a.sb;
    f.out = a.out;
    f.flags = a.flags;
    f.extra = f.grouped() ? static_cast< void const * >( a.offsets ) : a.bias;
    f.a_c = f.grouped() ? a.C : int32_t( a.a_c );
    f.b_c = int32_t( a.b_c );
    f.o_c = int32_t( a.o_c );
    f.sa_c = int32_t( a.sa_c );
    f.sb_c = int32_t( a.sb_c );
    f.a_ld = int32_t( along_rows_a ? a.a_k : a.a_row );
    f.b_ld = int32_t( along_rows_b ? a.b_k : a.b_row );
    f.o_row = int32_t( a.o_row );
    f.sa_row = int32_t( a.sa_row );
    f.sa_k = int32_t( a.sa_k );
    f.sb_row = int32_t( a.sb_row );
    f.sb_k = int32_t( a.sb_k );
    f.M = a.M;
    f.N = a.N;
    f.K = a.K;
    return f;
  }
};
static_assert( sizeof( BlockFast ) == 112, "kernel arguments" );

enum class BlockKernel : int32_t {
  GENERAL,         // any strides, 64 x 64 tiles (contract_block.hip)
  FEW_4,           // few rows of A, K over the waves and in 4 parts (contract_block_few.hip)
  FEW_8_PARTS,     // the same, 8 rows at a time
  FEW_16,          // the same, 16 rows at a time, K over the waves
  FEW_32,          // 32 rows at a time
  // through LDS directly (contract_block_tile.h), both operands at multiples of 16 bytes
  TILE_32x32,      // K in 8 groups of waves
  TILE_64x64_K,    // K in 4 groups of waves
  TILE_64x64,
  TILE_128x128,
  TILE_256x128,
  TILE_256x256,
  // the same through registers, operands at any address
  STAGED_32x32,    // K in 8 groups of waves
  STAGED_64x64_K,  // K in 2 groups of waves
  STAGED_64x64,
  STAGED_128x128
};

// How the operands lie for the tiles.
enum class BlockLayout : int32_t {
  NONE,            // any other
  K_K,             // both unit-stride along k: the product itself
  K_ROWS,          // B unit-stride along its rows: the gradient of the rows
  ROWS_ROWS        // both unit-stride along their rows: the gradient of the weights
};

struct BlockPlan {
  BlockKernel kernel = BlockKernel::GENERAL;
  BlockKernel kernel_off = BlockKernel::GENERAL;      // for pointers off 16 bytes
  BlockLayout layout = BlockLayout::NONE;
  bool      grouped = false;
  bool      has_sa = false, has_sb = false, has_bias = false;
  BlockArgs args{};                    // pointers set at execution
  int64_t   flops = 0;
  int64_t   bytes = 0;
  std::string desc;
};

int launch_block_general( BlockArgs const & a, hipStream_t stream );
int launch_block_few( BlockArgs const & a, BlockKernel kernel, hipStream_t stream );
int launch_block_staged( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream );
int launch_block_tile_bf16( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream );
int launch_block_tile_f8( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream );
int launch_block_tile_exact( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream );
int launch_block_tile_e8m0( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream );

// ---------------------------------------------------------------------------
// rounding to 8-bit floating point with a scale for each block
// ---------------------------------------------------------------------------
struct QuantF8Plan {
  int64_t batch = 1, rows = 0, cols = 0;
  int64_t ld_in = 0, ld_gate = 0, ld_q = 0, ld_values = 0;
  int32_t block_rows = 1, block_cols = kScaleBlock;
  int32_t dtype = ETIR_BF16, dtype_q = ETIR_F8E4M3, dtype_scale = ETIR_FP32;
  int32_t ktype = ETIR_KTYPE_UNDEFINED;
  int64_t bytes = 0;                   // with every optional tensor
  std::string desc;
};

int launch_quant_f8( QuantF8Plan const & plan, void const * in, void const * gate, void * q, void * scale, void * values,
                     hipStream_t stream );

#ifdef __HIPCC__
// ---------------------------------------------------------------------------
// device helpers
// ---------------------------------------------------------------------------

// the number that an e8m0 byte stands for: 2^(byte - 127), 255: NaN
__device__ __attribute__( ( always_inline ) ) inline float e8m0_to_f32( uint32_t v ) {
  uint32_t l_bits = v << 23;
  l_bits |= v == 0 ? 0x00400000u : 0u;          // 2^-127
  l_bits |= v == 255 ? 0x00400000u : 0u;        // the infinity's bits so far
  return __uint_as_float( l_bits );
}

// Rows (or k) of a group, inside [0, rows] whatever the offsets are.
struct BlockGroup { int32_t begin, end; };
__device__ inline BlockGroup block_group( int32_t const * offsets, int32_t g, int32_t rows ) {
  BlockGroup l_g;
  l_g.begin = min( max( offsets[g], 0 ), rows );
  l_g.end   = min( max( offsets[g + 1], l_g.begin ), rows );
  return l_g;
}

// tiles of BM rows in all groups
template< int BM >
__device__ inline int32_t block_tiles( int32_t const * offsets, int32_t groups, int32_t rows ) {
  int32_t l_sum = 0;
  for( int32_t l_g = threadIdx.x % 64; l_g < groups; l_g += 64 ) {
    BlockGroup const l_in = block_group( offsets, l_g, rows );
    l_sum += ( l_in.end - l_in.begin + BM - 1 ) / BM;
  }
#pragma unroll
  for( int l_d = 32; l_d > 0; l_d /= 2 ) l_sum += __shfl_xor( l_sum, l_d );
  return __builtin_amdgcn_readfirstlane( l_sum );
}

// Where a workgroup's rows lie: tile `tile` of BM rows, counted through the
// groups, none of which a tile crosses.
struct BlockRows { int32_t group, m0, end; };      // group < 0: no such tile
template< int BM >
__device__ inline BlockRows block_rows( int32_t const * offsets, int32_t groups, int32_t rows, int32_t tile ) {
  // every wave looks for itself: 64 groups at a time, the tiles of the groups
  // up to each lane's by a running sum over the lanes
  int const l_lane = threadIdx.x % 64;
  for( int32_t l_g0 = 0; l_g0 < groups; l_g0 += 64 ) {
    int32_t const l_g = l_g0 + l_lane;
    BlockGroup l_in = { 0, 0 };
    if( l_g < groups ) l_in = block_group( offsets, l_g, rows );
    int32_t const l_tiles = ( l_in.end - l_in.begin + BM - 1 ) / BM;
    int32_t l_sum = l_tiles;
#pragma unroll
    for( int l_d = 1; l_d < 64; l_d *= 2 ) {
      int32_t const l_v = __shfl_up( l_sum, l_d );
      if( l_lane >= l_d ) l_sum += l_v;
    }
    uint64_t const l_past = __ballot( l_sum > tile );
    if( l_past != 0 ) {
      int const l_at = __builtin_ctzll( l_past );
      int32_t const l_first = __builtin_amdgcn_readlane( l_sum - l_tiles, l_at );
      BlockRows l_r;
      l_r.group = l_g0 + l_at;
      l_r.m0 = __builtin_amdgcn_readlane( l_in.begin, l_at ) + ( tile - l_first ) * BM;
      l_r.end = __builtin_amdgcn_readlane( l_in.end, l_at );
      return l_r;
    }
    tile -= __builtin_amdgcn_readlane( l_sum, 63 );
  }
  return { -1, 0, 0 };
}

// The nth-longest group, the first of equal ones first; up to 64 groups, nth one of
// them.  A lane holds a group's length and counts those in front of it.
__device__ inline int32_t block_nth_longest( int32_t const * offsets, int32_t groups, int32_t rows, int32_t nth ) {
  int32_t const l_lane = threadIdx.x % 64;
  BlockGroup const l_in = block_group( offsets, min( l_lane, groups - 1 ), rows );
  int32_t const l_length = l_lane < groups ? l_in.end - l_in.begin : -1;
  int32_t l_front = 0;
  for( int32_t l_g = 0; l_g < groups; l_g++ ) {
    int32_t const l_other = __builtin_amdgcn_readlane( l_length, l_g );
    l_front += l_other > l_length || ( l_other == l_length && l_g < l_lane ) ? 1 : 0;
  }
  // the places of the groups are 0 to groups - 1, each once; lanes past them come after
  return __builtin_ctzll( __ballot( l_front == nth ) );
}
#endif

// tiles of bm rows that `rows` rows in `groups` groups have at most
inline int64_t block_most_tiles( int64_t rows, int64_t groups, int64_t bm ) {
  return rows / bm + std::min( rows, groups );
}

}  // namespace etir

#endif
