// Planner and C entry points of the products of 8-bit floating point blocks, of
// the products grouped by expert and of the rounding to such blocks
// (etir_hip_contraction_f8_*, etir_hip_contraction_grouped_*,
// etir_hip_quant_f8_*, include/einsum_ir_hip.h).
//
// A product's loops are sorted by type and fused where they are contiguous in
// every tensor; one loop of each type has to be left.
#include "block_internal.h"
#include <cmath>
#include <cstdlib>
#include <limits>
#include <vector>

namespace etir {

namespace {

constexpr int64_t kMaxIndex = std::numeric_limits< int32_t >::max();

// The tensors of a product.  Strides are elements, those of scales from block to block.
enum Tensor : int32_t { T_A = 0, T_B = 1, T_OUT = 2, T_SA = 3, T_SB = 4, T_BIAS = 5, T_TENSORS = 6 };
char const * const kTensorNames[T_TENSORS] = { "left", "right", "out", "scale_left", "scale_right", "bias" };

struct Loop {
  int64_t size;
  int64_t s[T_TENSORS];
};

// Everything that a caller says about a product.
struct Given {
  char const    * what;
  int64_t         num_loops;
  int32_t const * dim_types;
  int64_t const * sizes;
  int64_t const * strides[T_TENSORS];      // null: the tensor is not read
  int64_t         ragged;                  // index of the ragged loop, -1: no groups
  int32_t         block_left, block_right;
  int32_t         dtype_left, dtype_right, dtype_scale, dtype_out;
  int32_t         ktype_last_touch;
};

bool is_f8( int32_t dtype ) { return dtype == ETIR_F8E4M3 || dtype == ETIR_F8E5M2; }

// sorts by the stride in `slot` (outermost first) and fuses
void order_and_fuse( std::vector< Loop > & loops, int slot ) {
  std::stable_sort( loops.begin(), loops.end(),
                    [slot]( Loop const & x, Loop const & y ) { return x.s[slot] > y.s[slot]; } );
  std::vector< Loop > l_out;
  for( Loop const & l_l : loops ) {
    bool l_fits = !l_out.empty();
    for( int l_t = 0; l_fits && l_t < T_TENSORS; l_t++ ) l_fits = l_out.back().s[l_t] == l_l.s[l_t] * l_l.size;
    if( l_fits ) {
      int64_t const l_size = l_out.back().size * l_l.size;
      l_out.back() = l_l;
      l_out.back().size = l_size;
    }
    else l_out.push_back( l_l );
  }
  loops = l_out;
}

// which tensors a loop of a type may move in
bool moves( int32_t type, bool ragged_k, bool grouped, int tensor ) {
  switch( type ) {
    case ETIR_DIM_C: return true;
    case ETIR_DIM_M: return tensor == T_A || tensor == T_OUT || tensor == T_SA;
    case ETIR_DIM_N: return tensor == T_B || tensor == T_OUT || tensor == T_SB || tensor == T_BIAS;
    case ETIR_DIM_K: return tensor == T_A || tensor == T_B || tensor == T_SA || tensor == T_SB;
    default:         return grouped && ( ragged_k ? tensor == T_OUT : tensor == T_B || tensor == T_SB );
  }
}

int check_types( Given const & g ) {
  std::string const l_w( g.what );
  bool const l_f8 = is_f8( g.dtype_left );
  bool const l_grouped = g.ragged >= 0;
  if( l_f8 ? g.dtype_right != ETIR_F8E4M3 : !l_grouped || g.dtype_left != ETIR_BF16 || g.dtype_right != ETIR_BF16 ) {
    return fail( ETIR_INVALID_DTYPE, l_w + ( l_grouped ? ": left is F8E4M3 or F8E5M2 and right F8E4M3, or both BF16"
                                                       : ": left is F8E4M3 or F8E5M2, right F8E4M3" ) );
  }
  if( g.dtype_out != ETIR_FP32 && g.dtype_out != ETIR_BF16 ) {
    return fail( ETIR_INVALID_DTYPE, l_w + ": the output is FP32 or BF16" );
  }
  if( l_f8 && g.dtype_scale != ETIR_FP32 && g.dtype_scale != ETIR_E8M0 ) {
    return fail( ETIR_INVALID_DTYPE, l_w + ": scales are FP32 or E8M0" );
  }
  if( !l_f8 && ( g.strides[T_SA] != nullptr || g.strides[T_SB] != nullptr ) ) {
    return fail( ETIR_INVALID_DTYPE, l_w + ": scales belong to 8-bit operands" );
  }
  if( ( g.block_left != 1 && g.block_left != kScaleBlock ) || ( g.block_right != 1 && g.block_right != kScaleBlock ) ) {
    return fail( ETIR_COMPILATION_FAILED, l_w + ": 1 or 128 rows share a scale" );
  }
  if( g.ktype_last_touch != ETIR_KTYPE_UNDEFINED && g.ktype_last_touch != ETIR_KTYPE_RELU ) {
    return fail( ETIR_INVALID_KTYPE, l_w + ": the last touch is RELU or UNDEFINED" );
  }
  return ETIR_SUCCESS;
}

// How the tiles see the operands.
BlockLayout layout_of( BlockArgs const & a ) {
  bool const l_ra = a.a_k != 1, l_rb = a.b_k != 1;
  if( a.o_col != 1 || a.K == 0 || ( l_ra && ( a.a_row != 1 || a.M < 2 ) ) || ( l_rb && ( a.b_row != 1 || a.N < 2 ) ) || ( l_ra && !l_rb ) ) {
    return BlockLayout::NONE;
  }
  return l_ra ? BlockLayout::ROWS_ROWS : l_rb ? BlockLayout::K_ROWS : BlockLayout::K_K;
}

// Whether the loads into LDS directly take the operands; pointers count where
// they are known.
bool direct_fits( BlockArgs const & a, BlockLayout layout ) {
  if( layout == BlockLayout::NONE || ( a.has( BlockArgs::F8 ) && !a.has( BlockArgs::SCALES ) ) ) return false;
  int64_t const l_item = a.has( BlockArgs::F8 ) ? 1 : 2, l_step = 128 / l_item;
  bool const l_ra = layout == BlockLayout::ROWS_ROWS, l_rb = layout != BlockLayout::K_K;
  // k (or rows) of 16 bytes start at multiples of 16
  auto aligned = [&]( void const * p, int64_t c, int64_t stride ) {
    return uintptr_t( p ) % 16 == 0 && c * l_item % 16 == 0 && stride * l_item % 16 == 0;
  };
  int64_t const l_sa = l_ra ? a.a_k : a.a_row, l_sb = l_rb ? a.b_k : a.b_row;
  if( !aligned( a.a, a.a_c, l_sa ) || !aligned( a.b, a.b_c, l_sb ) ) return false;
  if( ( !l_ra || !l_rb ) && a.K * l_item % 16 != 0 ) return false;
  // a group's k start and end anywhere: pieces of 16 bytes along k would not, and
  // the last of them would hold the next group's first k
  if( ( !l_ra || !l_rb ) && a.has( BlockArgs::GROUP_K ) ) return false;
  // and a group's rows start at any row, also within 16 bytes along them
  if( l_ra && a.has( BlockArgs::GROUP_ROWS ) ) return false;
  // 31 bits of bytes in a step of a tile, and along k; rows of a k that do not
  // reach into the next k's, so that k past the end lie past the buffer's end
  int64_t const l_max = int64_t( 1 ) << 31;
  if( l_ra ? l_sa * l_item * l_step >= l_max || a.M > l_sa : l_sa * l_item * 256 >= l_max ) return false;
  if( l_rb ? l_sb * l_item * l_step >= l_max || a.N > l_sb : l_sb * l_item * 256 >= l_max ) return false;
  if( int64_t( a.K ) * l_item >= l_max - 2048 ) return false;
  // scales: 31 bits along a tile's rows and along k
  int64_t const l_kb = ( int64_t( a.K ) + kScaleBlock - 1 ) / kScaleBlock;
  return a.sa_row * 4 * 256 < l_max && a.sb_row * 4 * 256 < l_max && a.sa_k * 4 * l_kb < l_max && a.sb_k * 4 * l_kb < l_max;
}

// What choose_kernel knows of a kernel: rows and columns of a workgroup, groups of
// waves (few rows: parts of a fragment) that K is split over, workgroups on a
// compute unit, and microseconds for bf16, 8-bit products on the matrix cores and
// 8-bit numbers multiplied as bf16:
//   fixed, a step of 128 bytes of k alone, a step of each workgroup beside others,
//   a workgroup's beginning and end, factor of rows off 4 bytes (few rows)
// Few rows: fixed, 2 KiB (8 KiB in parts) of k of a workgroup, a workgroup beside
// others, and 1 KiB of k of one beside others.
// Fitted to 1400 products of 1 to 16384 rows, 64 to 12288 columns and k, up to 64
// groups, multiples of 16 and odd (profiles/block_choice.txt): the times that follow
// are off by 7 to 17 % (root mean square), the kernel chosen is 3 % slower than the
// best of all on average (64 x 64 tiles everywhere: 41 %), more than 20 % slower in
// one of 20 and 2.7 times at most (2 rows in 23 groups).
struct Candidate {
  BlockKernel  kernel;
  char const * name;
  int32_t      rows, cols, split, slots;
  float        us[3][5];
};
Candidate const kCandidates[] = {
  { BlockKernel::GENERAL, "general", 64, 64, 1, 4, { { 4.36f, 1.20f, 0.87f, 0.68f, 1.00f }, { 3.74f, 1.55f, 0.78f, 1.22f, 1.00f }, { 3.74f, 1.55f, 0.78f, 1.22f, 1.00f } } },
  { BlockKernel::FEW_4, "few 4", 4, 4, 4, 1, { { 3.94f, 0.37f, 0.67f, 0.13f, 2.63f }, { 3.01f, 1.43f, 1.58f, 0.20f, 1.11f }, { 3.01f, 1.43f, 1.58f, 0.20f, 1.11f } } },
  { BlockKernel::FEW_8_PARTS, "few 8 parts", 8, 4, 4, 1, { { 3.81f, 0.58f, 1.02f, 0.21f, 2.39f }, { 3.28f, 1.34f, 1.81f, 0.33f, 1.56f }, { 3.28f, 1.34f, 1.81f, 0.33f, 1.56f } } },
  { BlockKernel::FEW_16, "few 16", 16, 16, 1, 1, { { 3.32f, 0.81f, 0.46f, 0.75f, 2.68f }, { 2.99f, 1.32f, 1.29f, 0.90f, 1.46f }, { 2.99f, 1.32f, 1.29f, 0.90f, 1.46f } } },
  { BlockKernel::FEW_32, "few 32", 32, 16, 1, 1, { { 2.80f, 1.34f, 0.78f, 1.05f, 2.02f }, { 2.05f, 2.34f, 3.33f, 1.51f, 1.33f }, { 2.05f, 2.34f, 3.33f, 1.51f, 1.33f } } },
  { BlockKernel::TILE_32x32, "tile 32x32", 32, 32, 8, 1, { { 0.74f, 0.52f, 0.98f, 3.48f, 1.00f }, { 0.66f, 0.50f, 0.91f, 3.55f, 1.00f }, { 0.38f, 0.50f, 1.04f, 3.73f, 1.00f } } },
  { BlockKernel::TILE_64x64_K, "tile 64x64 K", 64, 64, 4, 1, { { 0.75f, 0.47f, 0.93f, 4.14f, 1.00f }, { 0.18f, 0.50f, 0.98f, 4.56f, 1.00f }, { 0.44f, 0.50f, 1.37f, 4.52f, 1.00f } } },
  { BlockKernel::TILE_64x64, "tile 64x64", 64, 64, 1, 2, { { 2.80f, 0.28f, 0.23f, 1.14f, 1.00f }, { 2.63f, 0.31f, 0.27f, 1.13f, 1.00f }, { 2.40f, 0.51f, 0.38f, 1.25f, 1.00f } } },
  { BlockKernel::TILE_128x128, "tile 128x128", 128, 128, 1, 2, { { 3.73f, 0.66f, 0.54f, 1.87f, 1.00f }, { 2.25f, 0.77f, 0.56f, 2.34f, 1.00f }, { 2.15f, 1.21f, 0.95f, 2.53f, 1.00f } } },
  { BlockKernel::TILE_256x128, "tile 256x128", 256, 128, 1, 1, { { 0.82f, 0.42f, 0.69f, 4.83f, 1.00f }, { 0.01f, 0.50f, 0.84f, 4.98f, 1.00f }, { 0.03f, 0.50f, 1.69f, 5.59f, 1.00f } } },
  { BlockKernel::TILE_256x256, "tile 256x256", 256, 256, 1, 1, { { 0.35f, 0.71f, 1.31f, 7.30f, 1.00f }, { 0.02f, 0.50f, 1.41f, 7.07f, 1.00f }, { 0.0f } } },
  { BlockKernel::STAGED_32x32, "staged 32x32", 32, 32, 8, 1, { { 0.83f, 0.63f, 1.07f, 5.32f, 1.00f }, { 0.07f, 1.65f, 1.45f, 5.63f, 1.00f }, { 0.31f, 0.50f, 1.88f, 5.25f, 1.00f } } },
  { BlockKernel::STAGED_64x64_K, "staged 64x64 K", 64, 64, 2, 2, { { 3.47f, 0.47f, 0.45f, 2.02f, 1.00f }, { 2.82f, 0.89f, 0.81f, 2.36f, 1.00f }, { 1.24f, 0.50f, 1.15f, 3.88f, 1.00f } } },
  { BlockKernel::STAGED_64x64, "staged 64x64", 64, 64, 1, 4, { { 3.84f, 0.48f, 0.23f, 0.91f, 1.00f }, { 3.86f, 0.68f, 0.35f, 0.94f, 1.00f }, { 3.30f, 0.83f, 0.46f, 1.44f, 1.00f } } },
  { BlockKernel::STAGED_128x128, "staged 128x128", 128, 128, 1, 2, { { 1.88f, 0.67f, 0.67f, 3.83f, 1.00f }, { 0.71f, 0.50f, 0.92f, 5.08f, 1.00f }, { 0.15f, 0.50f, 1.35f, 5.88f, 1.00f } } }
};

// rows of tiles in all batches or groups at most
int64_t most_tiles_m( BlockArgs const & a, int64_t rows ) {
  return a.has( BlockArgs::GROUP_ROWS ) ? block_most_tiles( a.M, a.C, rows ) : ( a.M + rows - 1 ) / rows * a.C;
}

bool exact( BlockArgs const & a ) { return a.has( BlockArgs::F8 ) && !a.has( BlockArgs::OUT_BF16 ); }

// operands that the kernels of few rows read: unit-stride along k, at any address
bool few_fits( BlockArgs const & a ) {
  return a.a_k == 1 && a.b_k == 1 && a.K * ( a.has( BlockArgs::F8 ) ? int64_t( 1 ) : int64_t( 2 ) ) >= 16 && !a.has( BlockArgs::GROUP_K );
}

// threads of a workgroup
int64_t threads( BlockKernel kernel ) {
  switch( kernel ) {
    case BlockKernel::GENERAL:
    case BlockKernel::TILE_64x64:
    case BlockKernel::TILE_128x128:
    case BlockKernel::STAGED_64x64: return 256;
    case BlockKernel::TILE_64x64_K: return 1024;
    default:                        return 512;
  }
}

double tiles_of( BlockArgs const & a, int64_t rows, int64_t cols ) {
  return double( most_tiles_m( a, rows ) ) * double( ( int64_t( a.N ) + cols - 1 ) / cols );
}

// A grid's threads are counted in 32 bits.
bool grid_fits( BlockArgs const & a, int64_t rows, int64_t cols, int64_t threads ) {
  return tiles_of( a, rows, cols ) * double( threads ) < 4294967296.0;
}

// With groups of rows every workgroup looks through the offsets, 64 in about a
// nanosecond of the whole card (65536 groups of one row: 37 ms): 2^36 of them would
// take a second.
bool groups_fit( BlockArgs const & a, int64_t rows, int64_t cols ) {
  return !a.has( BlockArgs::GROUP_ROWS ) || tiles_of( a, rows, cols ) * a.C < 68719476736.0;
}

bool fits( Candidate const & c, BlockArgs const & a, BlockLayout layout ) {
  if( !grid_fits( a, c.rows, c.cols, threads( c.kernel ) ) || !groups_fit( a, c.rows, c.cols ) ) return false;
  if( c.kernel == BlockKernel::GENERAL ) return true;
  if( !BlockFast::fits( a ) ) return false;
  if( c.kernel <= BlockKernel::FEW_32 ) return few_fits( a );
  if( c.kernel >= BlockKernel::STAGED_32x32 ) return layout != BlockLayout::NONE;
  return direct_fits( a, layout ) && !( exact( a ) && c.kernel == BlockKernel::TILE_256x256 );
}

// the time that a kernel should take on 256 compute units
double estimate( Candidate const & c, BlockArgs const & a, BlockLayout layout, double bytes ) {
  float const * const l_us = c.us[exact( a ) ? 2 : a.has( BlockArgs::F8 ) ? 1 : 0];
  bool const l_rows = a.has( BlockArgs::GROUP_ROWS ), l_ragged_k = a.has( BlockArgs::GROUP_K );
  int64_t const l_item = a.has( BlockArgs::F8 ) ? 1 : 2;
  // half of every group's last tile is empty; a group's K is the average one, the longest twice that
  double const l_tiles_m = l_rows ? double( a.M ) / c.rows + 0.5 * std::min( a.M, a.C ) : double( most_tiles_m( a, c.rows ) );
  double const l_groups = std::max( l_tiles_m, 1.0 ) * double( ( int64_t( a.N ) + c.cols - 1 ) / c.cols ), l_each = l_groups / 256;
  double const l_k = double( a.K ) * l_item / ( l_ragged_k ? a.C : 1 );
  double const l_least = bytes / 5.3e6;
  if( c.kernel != BlockKernel::GENERAL && c.kernel <= BlockKernel::FEW_32 ) {
    double const l_off = l_k != std::floor( l_k / 4 ) * 4 ? l_us[4] : 1.0;
    double const l_turns = std::ceil( std::ceil( l_k / ( 256 * c.split ) ) / 8 );
    return std::max( { l_us[0] + l_turns * l_us[1] * l_off, 0.5 * l_us[0] + l_each * ( l_us[2] + l_k / 1024 * l_us[3] * l_off ), l_least + 2 } );
  }
  double const l_layout = layout == BlockLayout::ROWS_ROWS ? 1.3 : layout == BlockLayout::K_ROWS ? 1.2 : 1.0;
  double const l_steps = c.kernel == BlockKernel::GENERAL ? std::ceil( l_k / l_item / 128 ) : std::ceil( std::ceil( l_k / 128 ) / c.split );
  double const l_rounds = l_rows || l_ragged_k ? std::max( 1.0, l_each > c.slots ? l_each / c.slots + 0.4 : 1.0 ) : std::ceil( l_each / c.slots );
  double const l_beside = l_rows || l_ragged_k ? std::max( 1.0, l_each + 0.4 ) : std::ceil( l_each );
  return std::max( { l_us[0] + l_rounds * ( l_steps * ( l_ragged_k ? 2 : 1 ) * l_us[1] * l_layout + l_us[3] ),
                     l_us[0] + l_beside * ( l_steps * l_us[2] * l_layout + l_us[3] ), l_least + 2.5 } );
}

// Whether a kernel loads into LDS directly.
bool direct( BlockKernel kernel ) { return kernel > BlockKernel::FEW_32 && kernel < BlockKernel::STAGED_32x32; }

// The kernel for operands as their strides say, and for a direct one another that
// takes pointers off 16 bytes at a call.  ETIR_BLOCK_KERNEL forces the first, by its
// place in BlockKernel, where it fits.
struct Choice { char const * name, * name_off; };      // name_off: null where it is the same
Choice choose_kernel( BlockArgs const & a, double bytes, BlockPlan & plan ) {
  plan.layout = layout_of( a );
  char const * const l_env = std::getenv( "ETIR_BLOCK_KERNEL" );
  int const l_forced = l_env ? std::atoi( l_env ) : -1;
  Candidate const * l_best = nullptr, * l_off = nullptr;
  double l_least = 0.0, l_least_off = 0.0;
  for( Candidate const & l_c : kCandidates ) {
    if( !fits( l_c, a, plan.layout ) ) continue;
    double const l_us = estimate( l_c, a, plan.layout, bytes );
    if( l_c.kernel >= BlockKernel::STAGED_32x32 && ( l_off == nullptr || l_us < l_least_off ) ) {
      l_off = &l_c;
      l_least_off = l_us;
    }
    bool const l_force = l_forced == int( l_c.kernel );
    if( l_best == nullptr || l_force || l_us < l_least ) {
      l_best = &l_c;
      l_least = l_force ? -1.0 : l_us;
    }
  }
  plan.kernel = plan.kernel_off = l_best->kernel;
  if( !direct( plan.kernel ) ) return { l_best->name, nullptr };
  // where a direct kernel fits, STAGED_64x64 does
  plan.kernel_off = l_off->kernel;
  return { l_best->name, l_off->name };
}

int plan_block( Given const & g, BlockPlan & plan ) {
  std::string const l_w( g.what );
  if( g.num_loops < 0 || ( g.num_loops > 0 && ( g.dim_types == nullptr || g.sizes == nullptr || g.strides[T_A] == nullptr
                                               || g.strides[T_B] == nullptr || g.strides[T_OUT] == nullptr ) ) ) {
    return fail( ETIR_COMPILATION_FAILED, l_w + ": invalid loop arrays" );
  }
  int l_err = check_types( g );
  if( l_err != ETIR_SUCCESS ) return l_err;
  bool const l_grouped = g.ragged >= 0;
  bool const l_f8 = is_f8( g.dtype_left );
  if( l_grouped && g.ragged >= g.num_loops ) return fail( ETIR_COMPILATION_FAILED, l_w + ": there is no such ragged loop" );
  bool const l_ragged_k = l_grouped && g.dim_types[g.ragged] == ETIR_DIM_K;
  if( l_grouped && !l_ragged_k && g.dim_types[g.ragged] != ETIR_DIM_M ) {
    return fail( ETIR_COMPILATION_FAILED, l_w + ": the ragged loop is of type M or K" );
  }
  if( l_ragged_k && l_f8 ) {
    return fail( ETIR_INVALID_DTYPE, l_w + ": a ragged K takes BF16 (blocks of 128 k would cross groups)" );
  }

  // by type; the group loop in the place of C
  std::vector< Loop > l_loops[4];
  int64_t l_total[4] = { 1, 1, 1, 1 };
  int l_groups = 0;
  for( int64_t l_i = 0; l_i < g.num_loops; l_i++ ) {
    int32_t const l_ty = g.dim_types[l_i];
    if( l_ty == ETIR_DIM_I || l_ty == ETIR_DIM_J ) continue;
    bool const l_group = l_ty == ETIR_DIM_G;
    if( !l_group && ( l_ty < ETIR_DIM_C || l_ty > ETIR_DIM_K ) ) {
      return fail( ETIR_COMPILATION_FAILED, l_w + ": unsupported dimension type" );
    }
    if( l_group && !l_grouped ) return fail( ETIR_COMPILATION_FAILED, l_w + ": a loop over groups without a ragged one" );
    if( l_grouped && l_ty == ETIR_DIM_C ) return fail( ETIR_COMPILATION_FAILED, l_w + ": no C loops beside groups" );
    l_groups += l_group;
    int32_t const l_to = l_group ? int32_t( ETIR_DIM_C ) : l_ty;
    int64_t const l_sz = g.sizes[l_i];
    if( l_sz < 0 ) return fail( ETIR_COMPILATION_FAILED, l_w + ": negative loop size" );
    if( l_sz != 0 && l_total[l_to] > kMaxIndex / 2 / l_sz ) {
      return fail( ETIR_COMPILATION_FAILED, l_w + ": 2^30 indices of one type, or more" );
    }
    l_total[l_to] *= l_sz;
    if( l_sz < 2 ) continue;
    Loop l_l{};
    l_l.size = l_sz;
    for( int l_t = 0; l_t < T_TENSORS; l_t++ ) {
      if( g.strides[l_t] == nullptr ) continue;
      int64_t const l_s = g.strides[l_t][l_i];
      if( l_s < 0 ) return fail( ETIR_COMPILATION_FAILED, l_w + ": negative stride" );
      if( moves( l_ty, l_ragged_k, l_grouped, l_t ) ) l_l.s[l_t] = l_s;
      // strides of an operand or the output along a loop that it does not have are not read
      else if( l_t >= T_SA && l_s != 0 ) {
        return fail( ETIR_COMPILATION_FAILED, l_w + ": " + kTensorNames[l_t] + " does not run over this loop" );
      }
    }
    if( moves( l_ty, l_ragged_k, l_grouped, T_OUT ) && l_l.s[T_OUT] == 0 ) {
      return fail( ETIR_COMPILATION_FAILED, l_w + ": output elements have to lie apart" );
    }
    // Offsets are made of 64-bit products of indices up to 2^30.
    for( int64_t l_s : l_l.s ) {
      if( l_s > ( int64_t( 1 ) << 40 ) / std::min< int64_t >( l_sz, 1 << 10 ) ) {
        return fail( ETIR_COMPILATION_FAILED, l_w + ": stride too large" );
      }
    }
    l_loops[l_to].push_back( l_l );
  }
  if( l_grouped && l_groups != 1 ) return fail( ETIR_COMPILATION_FAILED, l_w + ": one loop is over the groups" );
  // one scale a block of 128 is counted along one loop; a side without scales has no blocks
  if( ( g.block_left == kScaleBlock && g.strides[T_SA] != nullptr && l_loops[ETIR_DIM_M].size() > 1 )
      || ( g.block_right == kScaleBlock && g.strides[T_SB] != nullptr && l_loops[ETIR_DIM_N].size() > 1 )
      || ( l_f8 && l_loops[ETIR_DIM_K].size() > 1 ) ) {
    return fail( ETIR_COMPILATION_FAILED, l_w + ": blocks of 128 run along one loop" );
  }
  // the ragged loop is alone, also where it is shorter than 2
  if( l_grouped ) {
    int32_t const l_ty = g.dim_types[g.ragged];
    if( l_total[l_ty] != g.sizes[g.ragged] || l_loops[l_ty].size() > 1 ) {
      return fail( ETIR_COMPILATION_FAILED, l_w + ": the ragged loop is the only one of its type" );
    }
  }

  int64_t l_s[4][T_TENSORS] = {};
  for( int l_ty = 0; l_ty < 4; l_ty++ ) {
    order_and_fuse( l_loops[l_ty], l_ty == ETIR_DIM_K ? int( T_A ) : int( T_OUT ) );
    if( l_loops[l_ty].size() > 1 ) {
      return fail( ETIR_COMPILATION_FAILED, l_w + ": loops of one type have to fuse to one" );
    }
    if( !l_loops[l_ty].empty() ) std::copy_n( l_loops[l_ty][0].s, int( T_TENSORS ), l_s[l_ty] );
  }

  BlockArgs & a = plan.args;
  a.C = int32_t( l_total[ETIR_DIM_C] );
  a.M = int32_t( l_total[ETIR_DIM_M] );
  a.N = int32_t( l_total[ETIR_DIM_N] );
  a.K = int32_t( l_total[ETIR_DIM_K] );
  a.a_c = l_s[ETIR_DIM_C][T_A];
  a.b_c = l_s[ETIR_DIM_C][T_B];
  a.o_c = l_s[ETIR_DIM_C][T_OUT];
  a.sa_c = l_s[ETIR_DIM_C][T_SA];
  a.sb_c = l_s[ETIR_DIM_C][T_SB];
  a.bias_c = l_s[ETIR_DIM_C][T_BIAS];
  // a side of one index lies along k as well as along its rows
  a.a_row = l_s[ETIR_DIM_M][T_A];
  a.a_k = a.K < 2 ? 1 : l_s[ETIR_DIM_K][T_A];
  a.b_row = l_s[ETIR_DIM_N][T_B];
  a.b_k = a.K < 2 ? 1 : l_s[ETIR_DIM_K][T_B];
  a.o_row = l_s[ETIR_DIM_M][T_OUT];
  a.o_col = a.N < 2 ? 1 : l_s[ETIR_DIM_N][T_OUT];
  a.sa_row = l_s[ETIR_DIM_M][T_SA];
  a.sa_k = l_s[ETIR_DIM_K][T_SA];
  a.sb_row = l_s[ETIR_DIM_N][T_SB];
  a.sb_k = l_s[ETIR_DIM_K][T_SB];
  a.bias_col = l_s[ETIR_DIM_N][T_BIAS];
  a.flags = ( g.dtype_out == ETIR_BF16 ? BlockArgs::OUT_BF16 : 0u )
          | ( g.ktype_last_touch == ETIR_KTYPE_RELU ? BlockArgs::RELU : 0u )
          | ( l_grouped ? ( l_ragged_k ? BlockArgs::GROUP_K : BlockArgs::GROUP_ROWS ) : 0u )
          | ( l_f8 ? BlockArgs::F8 : 0u ) | ( g.dtype_left == ETIR_F8E5M2 ? BlockArgs::A_E5M2 : 0u )
          | ( l_f8 && g.dtype_scale == ETIR_E8M0 ? BlockArgs::E8M0 : 0u )
          | ( g.block_left == kScaleBlock ? BlockArgs::SA_BLOCKS : 0u )
          | ( g.block_right == kScaleBlock ? BlockArgs::SB_BLOCKS : 0u )
          | ( g.strides[T_SA] != nullptr && g.strides[T_SB] != nullptr ? BlockArgs::SCALES : 0u )
          | ( g.strides[T_BIAS] != nullptr ? BlockArgs::BIAS : 0u );
  plan.grouped = l_grouped;
  plan.has_sa = g.strides[T_SA] != nullptr;
  plan.has_sb = g.strides[T_SB] != nullptr;
  plan.has_bias = g.strides[T_BIAS] != nullptr;
  // the kernels that take any operands have 64 x 64 tiles: less than 2^24 of them
  if( !grid_fits( a, 64, 64, threads( BlockKernel::GENERAL ) ) ) return fail( ETIR_COMPILATION_FAILED, l_w + ": grid too large" );
  if( !groups_fit( a, 64, 64 ) ) return fail( ETIR_COMPILATION_FAILED, l_w + ": too many groups for as many blocks" );

  // a group of rows: one pass over all of them, and all weights
  int64_t const l_c = l_grouped ? 1 : int64_t( a.C ), l_item = l_f8 ? 1 : 2, l_out = g.dtype_out == ETIR_BF16 ? 2 : 4;
  int64_t const l_scale = g.dtype_scale == ETIR_E8M0 ? 1 : 4, l_kb = ( int64_t( a.K ) + kScaleBlock - 1 ) / kScaleBlock;
  int64_t const l_b_c = a.has( BlockArgs::GROUP_ROWS ) ? int64_t( a.C ) : l_c, l_o_c = l_ragged_k ? int64_t( a.C ) : l_c;
  plan.flops = 2 * l_c * a.M * a.N * a.K;
  plan.bytes = l_item * ( l_c * a.M + l_b_c * a.N ) * a.K + l_out * l_o_c * a.M * a.N;
  if( plan.has_sa ) plan.bytes += l_scale * l_c * l_kb * ( ( int64_t( a.M ) + g.block_left - 1 ) / g.block_left );
  if( plan.has_sb ) plan.bytes += l_scale * l_b_c * l_kb * ( ( int64_t( a.N ) + g.block_right - 1 ) / g.block_right );
  if( plan.has_bias ) plan.bytes += 4 * l_c * a.N;
  if( l_grouped ) plan.bytes += 4 * ( int64_t( a.C ) + 1 );
  char const * const l_left = l_f8 ? ( g.dtype_left == ETIR_F8E5M2 ? "e5m2" : "e4m3" ) : "bf16";
  Choice const l_choice = choose_kernel( a, double( plan.bytes ), plan );
  plan.desc = l_w + " " + l_choice.name + " " + ( l_grouped ? "groups=" : "C=" ) + std::to_string( a.C ) + " M=" + std::to_string( a.M )
            + " N=" + std::to_string( a.N ) + " K=" + std::to_string( a.K )
            + ( l_grouped ? ( l_ragged_k ? " ragged K" : " ragged M" ) : "" ) + " " + l_left
            + ( a.has( BlockArgs::OUT_BF16 ) ? " out=bf16" : " out=fp32" )
            + ( l_choice.name_off ? std::string( " off 16 bytes=" ) + l_choice.name_off : std::string() );
  return ETIR_SUCCESS;
}

int launch_block( BlockPlan const & plan, void const * left, void const * right, void const * scale_left, void const * scale_right,
                  void const * bias, void const * offsets, void * out, hipStream_t stream ) {
  BlockArgs a = plan.args;
  if( a.C == 0 || a.N == 0 || a.M == 0 ) return ETIR_SUCCESS;
  auto l_missing = [&]( char const * what ) {
    return fail( ETIR_NO_DATA_PTR_PROVIDED, std::string( plan.grouped ? "contraction_grouped" : "contraction_f8" ) + what );
  };
  a.a = left;
  a.b = right;
  a.sa = plan.has_sa ? scale_left : nullptr;
  a.sb = plan.has_sb ? scale_right : nullptr;
  a.bias = plan.has_bias ? static_cast< float const * >( bias ) : nullptr;
  a.offsets = static_cast< int32_t const * >( offsets );
  a.out = out;
  if( out == nullptr || ( a.K > 0 && ( left == nullptr || right == nullptr ) ) ) {
    return l_missing( ": null tensor pointer" );
  }
  if( plan.grouped && offsets == nullptr ) return l_missing( ": null offsets" );
  if( ( plan.has_sa && scale_left == nullptr && a.K > 0 ) || ( plan.has_sb && scale_right == nullptr && a.K > 0 )
      || ( plan.has_bias && bias == nullptr ) ) {
    return l_missing( ": null scale or bias, but its strides were given" );
  }
  // pointers may be less aligned than the strides
  BlockKernel const l_kernel = direct( plan.kernel ) && !direct_fits( a, plan.layout ) ? plan.kernel_off : plan.kernel;
  if( l_kernel == BlockKernel::GENERAL ) return launch_block_general( a, stream );
  if( l_kernel <= BlockKernel::FEW_32 )  return launch_block_few( a, l_kernel, stream );
  if( l_kernel >= BlockKernel::STAGED_32x32 ) return launch_block_staged( a, l_kernel, plan.layout, stream );
  if( !a.has( BlockArgs::F8 ) )   return launch_block_tile_bf16( a, l_kernel, plan.layout, stream );
  if( exact( a ) )                return launch_block_tile_exact( a, l_kernel, plan.layout, stream );
  if( a.has( BlockArgs::E8M0 ) )  return launch_block_tile_e8m0( a, l_kernel, plan.layout, stream );
  return launch_block_tile_f8( a, l_kernel, plan.layout, stream );
}

// Runs fn; what it throws (only memory can run out) becomes an error code.
template< class Fn >
int guarded( Fn && fn ) {
  try {
    return fn();
  }
  catch( ... ) {
    return fail( ETIR_UNDEFINED_ERROR, "out of memory" );   // short enough to need none
  }
}

// a new plan of the given kind on the current device
int new_plan( int32_t kind, etir_plan_t * plan ) {
  int l_device = 0;
  ETIR_HIP_CHECK( hipGetDevice( &l_device ) );
  etir_plan_s * l_plan = new etir_plan_s();
  l_plan->kind = kind;
  l_plan->device = l_device;
  *plan = l_plan;
  return ETIR_SUCCESS;
}

int create_block( Given const & g, int32_t kind, etir_plan_t * plan ) {
  return guarded( [&]() -> int {
    if( plan == nullptr ) return fail( ETIR_UNDEFINED_ERROR, "plan output pointer is null" );
    *plan = nullptr;
    auto l_block = std::make_shared< BlockPlan >();
    int l_err = plan_block( g, *l_block );
    if( l_err == ETIR_SUCCESS ) l_err = new_plan( kind, plan );
    if( l_err == ETIR_SUCCESS ) ( *plan )->block = l_block;
    return l_err;
  } );
}

constexpr int32_t kKindF8 = 6, kKindGrouped = 7, kKindQuant = 8;

}  // namespace

}  // namespace etir

using etir::fail;

extern "C" {

int etir_hip_contraction_f8_create( int64_t         num_loops,
                                    int32_t const * dim_types,
                                    int64_t const * sizes,
                                    int64_t const * strides_left,
                                    int64_t const * strides_right,
                                    int64_t const * strides_scale_left,
                                    int64_t const * strides_scale_right,
                                    int64_t const * strides_bias,
                                    int64_t const * strides_out,
                                    int32_t         block_left,
                                    int32_t         block_right,
                                    int32_t         dtype_left,
                                    int32_t         dtype_right,
                                    int32_t         dtype_scale,
                                    int32_t         dtype_out,
                                    int32_t         ktype_last_touch,
                                    etir_plan_t   * plan ) {
  etir::Given const l_g = { "contraction_f8", num_loops, dim_types, sizes,
                            { strides_left, strides_right, strides_out, strides_scale_left, strides_scale_right, strides_bias },
                            -1, block_left, block_right, dtype_left, dtype_right, dtype_scale, dtype_out, ktype_last_touch };
  return etir::create_block( l_g, etir::kKindF8, plan );
}

int etir_hip_contraction_f8_execute( etir_plan_t  plan,
                                     void const * left,
                                     void const * right,
                                     void const * scale_left,
                                     void const * scale_right,
                                     void const * bias,
                                     void       * out,
                                     void       * stream ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr || plan->kind != etir::kKindF8 ) {
      return fail( ETIR_CALLED_BEFORE_COMPILATION, "not a plan of an 8-bit floating point contraction" );
    }
    return etir::launch_block( *plan->block, left, right, scale_left, scale_right, bias, nullptr, out,
                               reinterpret_cast< hipStream_t >( stream ) );
  } );
}

int etir_hip_contraction_grouped_create( int64_t         num_loops,
                                         int32_t const * dim_types,
                                         int64_t const * sizes,
                                         int64_t const * strides_left,
                                         int64_t const * strides_right,
                                         int64_t const * strides_scale_left,
                                         int64_t const * strides_scale_right,
                                         int64_t const * strides_out,
                                         int64_t         ragged,
                                         int32_t         block_left,
                                         int32_t         block_right,
                                         int32_t         dtype_left,
                                         int32_t         dtype_right,
                                         int32_t         dtype_scale,
                                         int32_t         dtype_out,
                                         etir_plan_t   * plan ) {
  if( ragged < 0 ) {
    if( plan != nullptr ) *plan = nullptr;
    return fail( ETIR_COMPILATION_FAILED, "contraction_grouped: there is no such ragged loop" );
  }
  etir::Given const l_g = { "contraction_grouped", num_loops, dim_types, sizes,
                            { strides_left, strides_right, strides_out, strides_scale_left, strides_scale_right, nullptr },
                            ragged, block_left, block_right, dtype_left, dtype_right, dtype_scale, dtype_out,
                            ETIR_KTYPE_UNDEFINED };
  return etir::create_block( l_g, etir::kKindGrouped, plan );
}

int etir_hip_contraction_grouped_execute( etir_plan_t  plan,
                                          void const * left,
                                          void const * right,
                                          void const * scale_left,
                                          void const * scale_right,
                                          void const * offsets,
                                          void       * out,
                                          void       * stream ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr || plan->kind != etir::kKindGrouped ) {
      return fail( ETIR_CALLED_BEFORE_COMPILATION, "not a plan of a grouped contraction" );
    }
    return etir::launch_block( *plan->block, left, right, scale_left, scale_right, nullptr, offsets, out,
                               reinterpret_cast< hipStream_t >( stream ) );
  } );
}

int etir_hip_quant_f8_create( int64_t       batch,
                              int64_t       rows,
                              int64_t       cols,
                              int64_t       ld_in,
                              int64_t       ld_gate,
                              int64_t       ld_q,
                              int64_t       ld_values,
                              int32_t       block_rows,
                              int32_t       block_cols,
                              int32_t       dtype,
                              int32_t       dtype_q,
                              int32_t       dtype_scale,
                              int32_t       ktype,
                              etir_plan_t * plan ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr ) return fail( ETIR_UNDEFINED_ERROR, "plan output pointer is null" );
    *plan = nullptr;
    if( dtype != ETIR_BF16 && dtype != ETIR_FP32 ) return fail( ETIR_INVALID_DTYPE, "quant_f8: the input is BF16 or FP32" );
    if( !etir::is_f8( dtype_q ) ) return fail( ETIR_INVALID_DTYPE, "quant_f8: blocks are F8E4M3 or F8E5M2" );
    if( dtype_scale != ETIR_FP32 && dtype_scale != ETIR_E8M0 ) {
      return fail( ETIR_INVALID_DTYPE, "quant_f8: scales are FP32 or E8M0" );
    }
    if( ktype != ETIR_KTYPE_UNDEFINED && ktype != ETIR_KTYPE_RELU && ktype != ETIR_KTYPE_SILU ) {
      return fail( ETIR_INVALID_KTYPE, "quant_f8: the activation is RELU, SILU or UNDEFINED" );
    }
    bool const l_rows = block_rows == etir::kScaleBlock, l_cols = block_cols == etir::kScaleBlock;
    if( !( l_rows || block_rows == 1 ) || !( l_cols || block_cols == 1 ) || !( l_rows || l_cols ) ) {
      return fail( ETIR_COMPILATION_FAILED, "quant_f8: blocks are 1 x 128, 128 x 1 or 128 x 128" );
    }
    int64_t const l_max = int64_t( 1 ) << 30;
    if( batch < 0 || rows < 0 || cols < 0 || batch > l_max || rows > l_max || cols > l_max ) {
      return fail( ETIR_COMPILATION_FAILED, "quant_f8: batch, rows and cols are 0 to 2^30" );
    }
    int64_t const l_ld_max = int64_t( 1 ) << 40;
    for( int64_t l_ld : { ld_in, ld_gate, ld_q, ld_values } ) {
      if( l_ld < 0 || l_ld > l_ld_max ) return fail( ETIR_COMPILATION_FAILED, "quant_f8: negative row stride, or one over 2^40" );
    }
    if( ( rows > 1 || batch > 1 ) && ( ld_q < cols || ld_values < cols ) ) {
      return fail( ETIR_COMPILATION_FAILED, "quant_f8: rows of an output overlap" );
    }
    // a grid's threads are counted in 32 bits: 2^24 workgroups of 128 x 128, or of 32 blocks of a row
    double const l_groups = l_rows ? double( batch ) * ( ( rows + 127 ) / 128 ) * ( ( cols + 127 ) / 128 )
                                   : double( batch ) * double( rows ) * ( ( cols + 127 ) / 128 ) / 32;
    if( l_groups >= 16777215.0 || double( batch ) * double( rows ) > 2147483647.0 ) {
      return fail( ETIR_COMPILATION_FAILED, "quant_f8: too many blocks" );
    }
    auto l_q = std::make_shared< etir::QuantF8Plan >();
    l_q->batch = batch;
    l_q->rows = rows;
    l_q->cols = cols;
    l_q->ld_in = ld_in;
    l_q->ld_gate = ld_gate;
    l_q->ld_q = ld_q;
    l_q->ld_values = ld_values;
    l_q->block_rows = block_rows;
    l_q->block_cols = block_cols;
    l_q->dtype = dtype;
    l_q->dtype_q = dtype_q;
    l_q->dtype_scale = dtype_scale;
    l_q->ktype = ktype;
    int64_t const l_blocks = batch * ( ( rows + block_rows - 1 ) / block_rows ) * ( ( cols + block_cols - 1 ) / block_cols );
    l_q->bytes = batch * rows * cols * ( 3 * ( dtype == ETIR_BF16 ? 2 : 4 ) + 1 ) + ( dtype_scale == ETIR_FP32 ? 4 : 1 ) * l_blocks;
    l_q->desc = "quant_f8 batch=" + std::to_string( batch ) + " rows=" + std::to_string( rows ) + " cols=" + std::to_string( cols )
              + " block=" + std::to_string( block_rows ) + "x" + std::to_string( block_cols )
              + ( dtype == ETIR_BF16 ? " bf16" : " fp32" ) + ( dtype_q == ETIR_F8E5M2 ? " e5m2" : " e4m3" );
    int const l_err = etir::new_plan( etir::kKindQuant, plan );
    if( l_err == ETIR_SUCCESS ) ( *plan )->quant_f8 = l_q;
    return l_err;
  } );
}

int etir_hip_quant_f8_execute( etir_plan_t  plan,
                               void const * in,
                               void const * gate,
                               void       * q,
                               void       * scale,
                               void       * values,
                               void       * stream ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr || plan->kind != etir::kKindQuant ) return fail( ETIR_CALLED_BEFORE_COMPILATION, "not a quant_f8 plan" );
    return etir::launch_quant_f8( *plan->quant_f8, in, gate, q, scale, values, reinterpret_cast< hipStream_t >( stream ) );
  } );
}

}  // extern "C"
