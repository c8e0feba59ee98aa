// Planner and C entry points of the 8-bit layer operators
// (etir_hip_contraction_i8_*, etir_hip_norm_quant_*, etir_hip_act_quant_*,
// include/einsum_ir_hip.h).
//
// A product's loops are sorted by type and fused where they are contiguous in
// every tensor, as the contraction planner does (contract_plan.cpp); the
// general kernel takes what is left as it is.
#include "i8_internal.h"
#include <algorithm>
#include <limits>
#include <vector>

namespace etir {

namespace {

// largest K: 128 * 128 * K stays below 2^31
constexpr int64_t kI8MaxK = 131071;

struct Loop {
  int64_t size;
  int64_t s[I8_TENSORS];
};

bool contiguous( Loop const & outer, Loop const & inner ) {
  for( int l_t = 0; l_t < I8_TENSORS; l_t++ ) {
    if( outer.s[l_t] != inner.s[l_t] * inner.size ) return false;
  }
  return true;
}

// sorts by the stride in `slot` (outermost first) and fuses
void order_and_fuse( std::vector< Loop > & loops, int slot ) {
  std::stable_sort( loops.begin(), loops.end(),
                    [slot]( Loop const & x, Loop const & y ) { return x.s[slot] > y.s[slot]; } );
  std::vector< Loop > l_out;
  for( Loop const & l_l : loops ) {
    if( !l_out.empty() && contiguous( l_out.back(), l_l ) ) {
      Loop l_f = l_l;
      l_f.size *= l_out.back().size;
      l_out.back() = l_f;
    }
    else l_out.push_back( l_l );
  }
  loops = l_out;
}

int to_loops( std::vector< Loop > const & loops, I8Loops & out ) {
  if( loops.size() > std::size_t( kI8MaxLoops ) ) {
    return fail( ETIR_COMPILATION_FAILED, "contraction_i8: too many loops of one type that cannot be fused" );
  }
  out.n = int32_t( loops.size() );
  for( int l_i = 0; l_i < out.n; l_i++ ) {
    out.size[l_i] = int32_t( loops[l_i].size );
    std::copy_n( loops[l_i].s, int( I8_TENSORS ), out.stride[l_i] );
  }
  return ETIR_SUCCESS;
}

int64_t smallest( std::vector< Loop > const & loops, int slot ) {
  int64_t l_s = std::numeric_limits< int64_t >::max();
  for( Loop const & l_l : loops ) l_s = std::min( l_s, l_l.s[slot] );
  return l_s;
}

std::string sizes_of( I8Loops const & l ) {
  std::string l_s = "[";
  for( int l_i = 0; l_i < l.n; l_i++ ) l_s += ( l_i ? "," : "" ) + std::to_string( l.size[l_i] );
  return l_s + "]";
}

// What choose_kernel knows of a kernel.  Tiles: a workgroup's rows and columns,
// its threads, the k it takes in a step, and the time of a workgroup alone on
// its compute unit, fixed + step * steps.  Few-sided kernels (rows, cols: of the
// few and the many side): fixed + (step + step_few * few rows) * K / 1024 where
// nothing else bounds them, and at least (row + few * few rows) for every 10^6 k
// of all workgroups, which their 64-byte pieces of rows take in the caches, and
// 0.4 ns for each workgroup.
// Fitted to 170 products with rows at multiples of 16 bytes and 150 at others (1
// to 8192 rows, 16 to 16384 columns, K 64 to 12288).  The times that follow are
// off by 7 to 30 % (root mean square; K in parts up to 46 %), but alike for
// neighbours: the kernel chosen is 0.7 % slower than the best of all on average
// over these products, 0.8 % over 150 others (64 x 64 tiles everywhere: 44 and
// 42 %), and 28 % at most (profiles/i8_choice.txt).
struct Candidate {
  I8Kernel     kernel;
  char const * name;
  int32_t      alignment;          // of the rows; tiles: 16 bytes or not (1), few-sided: 4 (or more) or not (1)
  int32_t      rows, cols, threads, step_k;
  float        fixed_us, step_us;
  float        step_few_us, row_us, few_us;      // few-sided kernels
};
Candidate const kCandidates[] = {
  { I8Kernel::FEW_4,        "few 4",         4,  4,   4,   512, 1024, 0.35f, 0.10f, 0.0f,   0.63f, 0.07f },
  { I8Kernel::FEW_8_PARTS,  "few 8 parts",   4,  8,   4,   512, 1024, 0.35f, 0.31f, 0.0f,   0.63f, 0.09f },
  { I8Kernel::FEW_16_PARTS, "few 16 parts",  4,  16,  4,   512, 1024, 0.45f, 0.54f, 0.0f,   0.63f, 0.10f },
  { I8Kernel::FEW_16,       "few 16",        4,  16,  16,  512, 1024, 0.0f,  0.48f, 0.022f, 3.1f,  0.12f },
  { I8Kernel::FEW_32,       "few 32",        4,  32,  16,  512, 1024, 0.0f,  0.48f, 0.022f, 3.1f,  0.12f },
  { I8Kernel::TILE_32x32,   "tile 32x32",    16, 32,  32,  256, 512,  2.1f,  0.34f },
  { I8Kernel::TILE_64x32,   "tile 64x32",    16, 64,  32,  256, 256,  2.0f,  0.28f },
  { I8Kernel::TILE_64x64,   "tile 64x64",    16, 64,  64,  256, 128,  1.4f,  0.23f },
  { I8Kernel::TILE_128x64,  "tile 128x64",   16, 128, 64,  256, 128,  2.3f,  0.34f },
  { I8Kernel::TILE_128x128, "tile 128x128",  16, 128, 128, 512, 128,  3.2f,  0.44f },
  { I8Kernel::TILE_256x128, "tile 256x128",  16, 256, 128, 512, 128,  5.1f,  0.72f },
  { I8Kernel::TILE_256x256, "tile 256x256",  16, 256, 256, 512, 128,  8.4f,  1.09f },
  { I8Kernel::FEW_4,        "few 4",         1,  4,   4,   512, 1024, 0.50f, 0.25f, 0.0f,   1.0f,  0.11f },
  { I8Kernel::FEW_8_PARTS,  "few 8 parts",   1,  8,   4,   512, 1024, 0.50f, 0.50f, 0.0f,   1.0f,  0.14f },
  { I8Kernel::FEW_16_PARTS, "few 16 parts",  1,  16,  4,   512, 1024, 0.60f, 0.86f, 0.0f,   1.0f,  0.16f },
  { I8Kernel::FEW_16,       "few 16",        1,  16,  16,  512, 1024, 0.0f,  0.75f, 0.035f, 5.0f,  0.19f },
  { I8Kernel::FEW_32,       "few 32",        1,  32,  16,  512, 1024, 0.0f,  0.75f, 0.035f, 5.0f,  0.19f },
  { I8Kernel::SHIFT_32x32,  "shift 32x32",   1,  32,  32,  256, 512,  2.5f,  0.54f },
  { I8Kernel::SHIFT_64x64,  "shift 64x64",   1,  64,  64,  256, 128,  1.5f,  0.40f },
  { I8Kernel::SHIFT_128x128, "shift 128x128", 1, 128, 128, 512, 128,  3.7f,  0.69f },
  { I8Kernel::SHIFT_256x128, "shift 256x128", 1, 256, 128, 512, 128,  4.7f,  1.05f }
};

int64_t ceil_div( int64_t x, int64_t y ) { return ( x + y - 1 ) / y; }

// The kernel that should take the least time on 256 compute units: tiles in
// rounds of one workgroup each, at least 1.15 times the tensors' bytes at 5.3
// TB/s.  The first of equals is the one with the smaller tiles.
Candidate const * choose_candidate( I8Args const & a, int64_t C, int32_t alignment ) {
  Candidate const * l_best = nullptr;
  double l_least = 0.0;
  int32_t const l_k = a.K();
  double const l_bytes = double( C ) * ( ( double( a.M ) + a.N ) * l_k + double( a.has( I8Args::OUT_BF16 ) ? 2 : 4 ) * a.M * a.N );
  for( Candidate const & l_c : kCandidates ) {
    // tiles: rows at multiples of 16 bytes or not; few-sided: of 4 or not
    bool const l_few = l_c.kernel <= I8Kernel::FEW_32;
    if( l_few ? ( l_c.alignment == 1 ) != ( alignment == 1 ) : ( l_c.alignment == 16 ) != ( alignment == 16 ) ) continue;
    double l_groups, l_us;
    if( l_few ) {
      if( std::min( a.M, a.N ) > l_c.rows ) continue;
      l_groups = double( ceil_div( std::max( a.M, a.N ), l_c.cols ) ) * C;
    }
    else {
      // a tile's rows are addressed by 31 bits from its first one
      if( std::max( int64_t( l_c.rows ) * a.a_row, int64_t( l_c.cols ) * a.b_col ) + l_k >= ( int64_t( 1 ) << 31 ) ) continue;
      l_groups = double( ceil_div( a.M, l_c.rows ) ) * ceil_div( a.N, l_c.cols ) * C;
      double const l_steps = double( ceil_div( l_k, l_c.step_k ) );
      l_us = std::max( double( ceil_div( int64_t( l_groups ), 256 ) ) * ( l_c.fixed_us + l_steps * l_c.step_us ),
                       1.15 * l_bytes / 5.3e6 );
    }
    if( l_few ) {
      int32_t const l_rows = std::min( a.M, a.N );
      l_us = std::max( l_c.fixed_us + double( l_k ) / l_c.step_k * ( l_c.step_us + l_c.step_few_us * l_rows ),
                       l_groups * ( l_k * 1e-6 * ( l_c.row_us + l_c.few_us * l_rows ) + 0.4e-3 ) );
    }
    // a grid's threads are counted in 32 bits
    if( l_groups * l_c.threads >= 4294967296.0 ) continue;
    if( l_best == nullptr || l_us < l_least ) {
      l_best = &l_c;
      l_least = l_us;
    }
  }
  return l_best;
}

// The kernel for a product whose loops are in plan.args; its name.
char const * choose_kernel( I8Plan & plan ) {
  I8GeneralArgs const & a = plan.args;
  bool const l_unit_k = a.k.n == 0 || ( a.k.n == 1 && a.k.stride[0][I8_A] == 1 && a.k.stride[0][I8_B] == 1 );
  if( a.c.n > 1 || a.m.n > 1 || a.n.n > 1 || !l_unit_k || a.K < 16 || a.C == 0 || a.M == 0 || a.N == 0 ) return "general";
  // strides of 32 bits
  for( I8Loops const * l_l : { &a.c, &a.m, &a.n } ) {
    for( int64_t l_s : l_l->stride[0] ) if( l_s > std::numeric_limits< int32_t >::max() ) return "general";
  }
  I8Args & f = plan.affine;
  f.M = int32_t( a.M );
  f.N = int32_t( a.N );
  f.k_flags = uint32_t( a.K ) | ( a.out_bf16 ? I8Args::OUT_BF16 : 0u ) | ( a.relu ? I8Args::RELU : 0u )
            | ( a.bias_rows ? I8Args::BIAS_ROWS : 0u );
  // without a loop every stride is 0
  f.a_row = int32_t( a.m.stride[0][I8_A] );
  f.o_row = int32_t( a.m.stride[0][I8_OUT] );
  f.sa_row = int32_t( a.m.stride[0][I8_SA] );
  f.b_col = int32_t( a.n.stride[0][I8_B] );
  f.o_col = a.n.n == 0 ? 1 : int32_t( a.n.stride[0][I8_OUT] );
  f.sb_col = int32_t( a.n.stride[0][I8_SB] );
  f.bias_step = int32_t( ( a.bias_rows ? a.m : a.n ).stride[0][I8_BIAS] );
  std::copy_n( a.c.stride[0], int( I8_TENSORS ), f.c );
  plan.alignment = i8_alignment( f );
  Candidate const * l_c = choose_candidate( f, a.C, plan.alignment );
  if( l_c == nullptr ) return "general";
  plan.kernel = l_c->kernel;
  return l_c->name;
}

int launch_affine( I8Kernel kernel, I8Args const & a, int64_t C, hipStream_t stream ) {
  if( kernel <= I8Kernel::FEW_32 ) return launch_i8_few( a, C, kernel, stream );
  return launch_i8_tile( a, C, kernel, stream );
}

}  // namespace

int plan_i8( int64_t         num_loops,
             int32_t const * dim_types,
             int64_t const * sizes,
             int64_t const * strides_left,
             int64_t const * strides_right,
             int64_t const * strides_scale_left,
             int64_t const * strides_scale_right,
             int64_t const * strides_bias,
             int64_t const * strides_out,
             int32_t         dtype_out,
             int32_t         ktype_last_touch,
             I8Plan        & plan ) {
  if( num_loops < 0 || ( num_loops > 0 && ( dim_types == nullptr || sizes == nullptr || strides_left == nullptr
                                            || strides_right == nullptr || strides_out == nullptr ) ) ) {
    return fail( ETIR_COMPILATION_FAILED, "contraction_i8: invalid loop arrays" );
  }
  if( dtype_out != ETIR_FP32 && dtype_out != ETIR_BF16 ) {
    return fail( ETIR_INVALID_DTYPE, "contraction_i8: the output is FP32 or BF16" );
  }
  if( ktype_last_touch != ETIR_KTYPE_UNDEFINED && ktype_last_touch != ETIR_KTYPE_RELU ) {
    return fail( ETIR_INVALID_KTYPE, "contraction_i8: the last touch is RELU or UNDEFINED" );
  }

  std::vector< Loop > l_loops[4];              // by ETIR_DIM_C/M/N/K
  int64_t l_total[4] = { 1, 1, 1, 1 };
  int64_t const l_limit[4] = { std::numeric_limits< int32_t >::max(), std::numeric_limits< int32_t >::max(),
                               std::numeric_limits< int32_t >::max(), kI8MaxK };
  for( int64_t l_i = 0; l_i < num_loops; l_i++ ) {
    int32_t const l_ty = dim_types[l_i];
    if( l_ty == ETIR_DIM_I || l_ty == ETIR_DIM_J ) continue;
    if( l_ty < ETIR_DIM_C || l_ty > ETIR_DIM_K ) {
      return fail( ETIR_COMPILATION_FAILED, "contraction_i8: unsupported dimension type" );
    }
    int64_t const l_sz = sizes[l_i];
    if( l_sz < 0 ) return fail( ETIR_COMPILATION_FAILED, "contraction_i8: negative loop size" );
    if( l_sz != 0 && l_total[l_ty] > l_limit[l_ty] / l_sz ) {
      return fail( ETIR_COMPILATION_FAILED, l_ty == ETIR_DIM_K
                   ? "contraction_i8: K over 131071 could exceed a 32-bit sum"
                   : "contraction_i8: more than 2^31 - 1 indices of one type" );
    }
    l_total[l_ty] *= l_sz;
    if( l_sz < 2 ) continue;
    Loop l_l{};
    l_l.size = l_sz;
    l_l.s[I8_A] = strides_left[l_i];
    l_l.s[I8_B] = strides_right[l_i];
    l_l.s[I8_OUT] = strides_out[l_i];
    if( strides_scale_left != nullptr ) l_l.s[I8_SA] = strides_scale_left[l_i];
    if( strides_scale_right != nullptr ) l_l.s[I8_SB] = strides_scale_right[l_i];
    if( strides_bias != nullptr ) l_l.s[I8_BIAS] = strides_bias[l_i];
    for( int64_t l_s : l_l.s ) {
      if( l_s < 0 ) return fail( ETIR_COMPILATION_FAILED, "contraction_i8: negative stride" );
    }
    bool const l_left = l_ty == ETIR_DIM_C || l_ty == ETIR_DIM_M;
    bool const l_right = l_ty == ETIR_DIM_C || l_ty == ETIR_DIM_N;
    if( ( !l_left && l_l.s[I8_SA] != 0 ) || ( !l_right && ( l_l.s[I8_SB] != 0 || l_l.s[I8_BIAS] != 0 ) ) ) {
      return fail( ETIR_COMPILATION_FAILED,
                   "contraction_i8: scale_left runs over C and M loops, scale_right and bias over C and N loops" );
    }
    // strides of a tensor along a loop that it does not have are not read
    if( l_ty == ETIR_DIM_M ) l_l.s[I8_B] = 0;
    if( l_ty == ETIR_DIM_N ) l_l.s[I8_A] = 0;
    if( l_ty == ETIR_DIM_K ) l_l.s[I8_OUT] = 0;
    else if( l_l.s[I8_OUT] == 0 ) {
      return fail( ETIR_COMPILATION_FAILED, "contraction_i8: output elements have to lie apart" );
    }
    l_loops[l_ty].push_back( l_l );
  }

  // the columns are the side with the output's smaller stride
  plan.swapped = smallest( l_loops[ETIR_DIM_M], I8_OUT ) < smallest( l_loops[ETIR_DIM_N], I8_OUT );
  if( plan.swapped ) {
    std::swap( l_loops[ETIR_DIM_M], l_loops[ETIR_DIM_N] );
    std::swap( l_total[ETIR_DIM_M], l_total[ETIR_DIM_N] );
    for( auto & l_ty : l_loops ) for( Loop & l_l : l_ty ) {
      std::swap( l_l.s[I8_A], l_l.s[I8_B] );
      std::swap( l_l.s[I8_SA], l_l.s[I8_SB] );
    }
  }
  plan.has_sa = strides_scale_left != nullptr;
  plan.has_sb = strides_scale_right != nullptr;
  if( plan.swapped ) std::swap( plan.has_sa, plan.has_sb );
  plan.has_bias = strides_bias != nullptr;

  I8GeneralArgs & a = plan.args;
  I8Loops * const l_to[4] = { &a.c, &a.m, &a.n, &a.k };
  for( int l_ty = 0; l_ty < 4; l_ty++ ) {
    order_and_fuse( l_loops[l_ty], l_ty == ETIR_DIM_K ? int( I8_A ) : int( I8_OUT ) );
    int const l_err = to_loops( l_loops[l_ty], *l_to[l_ty] );
    if( l_err != ETIR_SUCCESS ) return l_err;
  }
  a.C = l_total[ETIR_DIM_C];
  a.M = l_total[ETIR_DIM_M];
  a.N = l_total[ETIR_DIM_N];
  a.K = l_total[ETIR_DIM_K];
  a.out_bf16 = dtype_out == ETIR_BF16;
  a.relu = ktype_last_touch == ETIR_KTYPE_RELU;
  a.bias_rows = plan.swapped;
  a.tiles_m = int32_t( ( a.M + 63 ) / 64 );
  a.tiles_n = int32_t( ( a.N + 63 ) / 64 );
  // a grid's threads are counted in 32 bits
  double const l_grid = double( a.tiles_m ) * a.tiles_n * double( a.C );
  if( l_grid >= 4294967296.0 / 256 ) {
    return fail( ETIR_COMPILATION_FAILED, "contraction_i8: grid too large" );
  }
  plan.flops = 2 * a.C * a.M * a.N * a.K;
  int64_t const l_rows = plan.swapped ? a.N : a.M, l_cols = plan.swapped ? a.M : a.N;
  plan.bytes = a.C * ( a.M + a.N ) * a.K + ( dtype_out == ETIR_BF16 ? 2 : 4 ) * a.C * a.M * a.N
             + ( strides_scale_left != nullptr ? 4 * a.C * l_rows : 0 )
             + ( ( strides_scale_right != nullptr ? 4 : 0 ) + ( strides_bias != nullptr ? 4 : 0 ) ) * a.C * l_cols;
  plan.desc = std::string( "contraction_i8 " ) + choose_kernel( plan ) + " C=" + sizes_of( a.c ) + " rows=" + sizes_of( a.m ) + " cols=" + sizes_of( a.n )
            + " K=" + sizes_of( a.k ) + ( plan.swapped ? " swapped" : "" )
            + ( a.out_bf16 ? " out=bf16" : " out=fp32" );
  return ETIR_SUCCESS;
}

int launch_i8( I8Plan const & plan,
               void const   * left,
               void const   * right,
               void const   * scale_left,
               void const   * scale_right,
               void const   * bias,
               void         * out,
               hipStream_t    stream ) {
  I8GeneralArgs a = plan.args;
  if( a.C == 0 || a.M == 0 || a.N == 0 ) return ETIR_SUCCESS;
  a.a  = static_cast< int8_t const * >( plan.swapped ? right : left );
  a.b  = static_cast< int8_t const * >( plan.swapped ? left : right );
  a.sa = plan.has_sa ? static_cast< float const * >( plan.swapped ? scale_right : scale_left ) : nullptr;
  a.sb = plan.has_sb ? static_cast< float const * >( plan.swapped ? scale_left : scale_right ) : nullptr;
  a.bias = plan.has_bias ? static_cast< float const * >( bias ) : nullptr;
  a.out = out;
  if( out == nullptr || ( a.K > 0 && ( a.a == nullptr || a.b == nullptr ) ) ) {
    return fail( ETIR_NO_DATA_PTR_PROVIDED, "contraction_i8: null tensor pointer" );
  }
  if( ( plan.has_sa && a.sa == nullptr ) || ( plan.has_sb && a.sb == nullptr )
      || ( plan.has_bias && a.bias == nullptr ) ) {
    return fail( ETIR_NO_DATA_PTR_PROVIDED, "contraction_i8: null scale or bias, but its strides were given" );
  }
  if( plan.kernel == I8Kernel::GENERAL ) return launch_i8_general( a, stream );
  I8Args f = plan.affine;
  f.a = a.a;
  f.b = a.b;
  f.sa = a.sa;
  f.sb = a.sb;
  f.bias = a.bias;
  f.out = a.out;
  // pointers may be less aligned than the strides
  int32_t const l_alignment = i8_alignment( f );
  if( l_alignment >= plan.alignment ) return launch_affine( plan.kernel, f, a.C, stream );
  Candidate const * l_c = choose_candidate( f, a.C, l_alignment );
  return l_c == nullptr ? launch_i8_general( a, stream ) : launch_affine( l_c->kernel, f, a.C, stream );
}

namespace {

// arguments that both row operators share
int check_rows( char const * what, int64_t rows, int64_t cols, int64_t ld_q, int64_t ld_values, int32_t dtype ) {
  std::string const l_w( what );
  if( dtype != ETIR_BF16 && dtype != ETIR_FP32 ) {
    return fail( ETIR_INVALID_DTYPE, l_w + ": the rows are BF16 or FP32" );
  }
  int64_t const l_max = std::numeric_limits< int32_t >::max();
  if( rows < 0 || cols < 0 || rows > l_max || cols > l_max / 2 ) {
    return fail( ETIR_COMPILATION_FAILED, l_w + ": rows are 0 to 2^31 - 1, cols 0 to 2^30 - 1" );
  }
  if( rows > 1 && ( ld_q < cols || ld_values < cols ) ) {
    return fail( ETIR_COMPILATION_FAILED, l_w + ": rows of an output overlap" );
  }
  return ETIR_SUCCESS;
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

}  // namespace

}  // namespace etir

using etir::fail;

extern "C" {

int etir_hip_contraction_i8_create( int64_t         num_loops,
                                    int32_t const * dim_types,
                                    int64_t const * sizes,
                                    int64_t const * strides_left,
                                    int64_t const * strides_right,
                                    int64_t const * strides_scale_left,
                                    int64_t const * strides_scale_right,
                                    int64_t const * strides_bias,
                                    int64_t const * strides_out,
                                    int32_t         dtype_out,
                                    int32_t         ktype_last_touch,
                                    etir_plan_t   * plan ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr ) return fail( ETIR_UNDEFINED_ERROR, "plan output pointer is null" );
    *plan = nullptr;
    auto l_i8 = std::make_shared< etir::I8Plan >();
    int l_err = etir::plan_i8( num_loops, dim_types, sizes, strides_left, strides_right, strides_scale_left,
                               strides_scale_right, strides_bias, strides_out, dtype_out, ktype_last_touch, *l_i8 );
    if( l_err == ETIR_SUCCESS ) l_err = etir::new_plan( 3, plan );
    if( l_err == ETIR_SUCCESS ) ( *plan )->i8 = l_i8;
    return l_err;
  } );
}

int etir_hip_contraction_i8_execute( etir_plan_t  plan,
                                     void const * left,
                                     void const * right,
                                     void const * scale_left,
                                     void const * scale_right,
                                     void const * bias,
                                     void       * out,
                                     void       * stream ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr || plan->kind != 3 ) {
      return fail( ETIR_CALLED_BEFORE_COMPILATION, "not a plan of an 8-bit contraction" );
    }
    return etir::launch_i8( *plan->i8, left, right, scale_left, scale_right, bias, out,
                            reinterpret_cast< hipStream_t >( stream ) );
  } );
}

int etir_hip_norm_quant_create( int64_t       rows,
                                int64_t       cols,
                                int64_t       ld_in,
                                int64_t       ld_residual,
                                int64_t       ld_total,
                                int64_t       ld_q,
                                int64_t       ld_values,
                                int32_t       dtype,
                                int32_t       dtype_weight,
                                float         eps,
                                etir_plan_t * plan ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr ) return fail( ETIR_UNDEFINED_ERROR, "plan output pointer is null" );
    *plan = nullptr;
    int l_err = etir::check_rows( "norm_quant", rows, cols, ld_q, ld_values, dtype );
    if( l_err != ETIR_SUCCESS ) return l_err;
    if( dtype_weight != ETIR_BF16 && dtype_weight != ETIR_FP32 ) {
      return fail( ETIR_INVALID_DTYPE, "norm_quant: the weight is BF16 or FP32" );
    }
    if( ld_in < 0 || ld_residual < 0 || ( rows > 1 && ld_total < cols ) ) {
      return fail( ETIR_COMPILATION_FAILED, "norm_quant: negative row stride, or rows of total overlap" );
    }
    if( !( eps >= 0.0f ) || eps > std::numeric_limits< float >::max() ) {
      return fail( ETIR_COMPILATION_FAILED, "norm_quant: eps is finite and at least 0" );
    }
    auto l_q = std::make_shared< etir::QuantPlan >();
    l_q->norm = true;
    l_q->rows = rows;
    l_q->cols = cols;
    l_q->dtype = dtype;
    l_q->dtype_weight = dtype_weight;
    l_q->eps = eps;
    l_q->ld_in = ld_in;
    l_q->ld_second = ld_residual;
    l_q->ld_total = ld_total;
    l_q->ld_q = ld_q;
    l_q->ld_values = ld_values;
    etir::describe_quant( *l_q );
    l_err = etir::new_plan( 4, plan );
    if( l_err == ETIR_SUCCESS ) ( *plan )->quant = l_q;
    return l_err;
  } );
}

int etir_hip_norm_quant_execute( etir_plan_t  plan,
                                 void const * in,
                                 void const * residual,
                                 void const * weight,
                                 void       * total,
                                 void       * q,
                                 void       * scale,
                                 void       * values,
                                 void       * stream ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr || plan->kind != 4 ) {
      return fail( ETIR_CALLED_BEFORE_COMPILATION, "not a norm_quant plan" );
    }
    etir::QuantPlan const & p = *plan->quant;
    etir::QuantArgs a{};
    a.in = in;
    a.second = residual;
    a.weight = weight;
    a.total = total;
    a.q = static_cast< int8_t * >( q );
    a.scale = static_cast< float * >( scale );
    a.values = values;
    return etir::launch_quant( p, a, reinterpret_cast< hipStream_t >( stream ) );
  } );
}

int etir_hip_act_quant_create( int64_t       rows,
                               int64_t       cols,
                               int64_t       ld_in,
                               int64_t       ld_gate,
                               int64_t       ld_q,
                               int64_t       ld_values,
                               int32_t       dtype,
                               int32_t       ktype,
                               etir_plan_t * plan ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr ) return fail( ETIR_UNDEFINED_ERROR, "plan output pointer is null" );
    *plan = nullptr;
    int l_err = etir::check_rows( "act_quant", rows, cols, ld_q, ld_values, dtype );
    if( l_err != ETIR_SUCCESS ) return l_err;
    if( ld_in < 0 || ld_gate < 0 ) return fail( ETIR_COMPILATION_FAILED, "act_quant: negative row stride" );
    if( ktype != ETIR_KTYPE_UNDEFINED && ktype != ETIR_KTYPE_RELU && ktype != ETIR_KTYPE_SILU ) {
      return fail( ETIR_INVALID_KTYPE, "act_quant: the activation is RELU, SILU or UNDEFINED" );
    }
    auto l_q = std::make_shared< etir::QuantPlan >();
    l_q->rows = rows;
    l_q->cols = cols;
    l_q->dtype = dtype;
    l_q->ktype = ktype;
    l_q->ld_in = ld_in;
    l_q->ld_second = ld_gate;
    l_q->ld_q = ld_q;
    l_q->ld_values = ld_values;
    etir::describe_quant( *l_q );
    l_err = etir::new_plan( 5, plan );
    if( l_err == ETIR_SUCCESS ) ( *plan )->quant = l_q;
    return l_err;
  } );
}

int etir_hip_act_quant_execute( etir_plan_t  plan,
                                void const * in,
                                void const * gate,
                                void       * q,
                                void       * scale,
                                void       * values,
                                void       * stream ) {
  return etir::guarded( [&]() -> int {
    if( plan == nullptr || plan->kind != 5 ) {
      return fail( ETIR_CALLED_BEFORE_COMPILATION, "not an act_quant plan" );
    }
    etir::QuantPlan const & p = *plan->quant;
    etir::QuantArgs a{};
    a.in = in;
    a.second = gate;
    a.q = static_cast< int8_t * >( q );
    a.scale = static_cast< float * >( scale );
    a.values = values;
    return etir::launch_quant( p, a, reinterpret_cast< hipStream_t >( stream ) );
  } );
}

}  // extern "C"
