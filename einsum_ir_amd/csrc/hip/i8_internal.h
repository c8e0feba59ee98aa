// Declarations of the 8-bit layer operators: the product of 8-bit integers
// with scales (i8_plan.cpp, contract_i8*.hip) and the operators that round
// rows to 8 bits (quant_rows.hip).
#ifndef ETIR_I8_INTERNAL_H
#define ETIR_I8_INTERNAL_H

#include "etir_internal.h"

namespace etir {

// ---------------------------------------------------------------------------
// product of 8-bit integers
//   out[c,m,n] = last( sa[c,m] sb[c,n] sum_k A[c,m,k] B[c,n,k] + bias )
// m: the rows, n: the columns of the kernels; the output's unit-stride loop is
// a column loop where it is not a batch loop (A and B change places for that)
// ---------------------------------------------------------------------------
constexpr int kI8MaxLoops = 6;       // fused loops of one type

// The tensors of a product.  All offsets are elements; 8-bit elements are bytes.
enum I8Tensor : int32_t { I8_A = 0, I8_B = 1, I8_OUT = 2, I8_SA = 3, I8_SB = 4, I8_BIAS = 5, I8_TENSORS = 6 };

// The fused loops of one type, outermost first.
struct I8Loops {
  int32_t n = 0;
  int32_t size[kI8MaxLoops] = {};
  int64_t stride[kI8MaxLoops][I8_TENSORS] = {};
};

// Any loops: the general kernel decodes its indices.
struct I8GeneralArgs {
  int8_t const * a;
  int8_t const * b;
  float const  * sa;       // null: 1
  float const  * sb;       // null: 1
  float const  * bias;     // null: 0
  void         * out;
  I8Loops c, m, n, k;
  int64_t C, M, N, K;
  int32_t tiles_m, tiles_n;
  int32_t out_bf16;
  int32_t relu;
  int32_t bias_rows;       // the bias runs over rows (A and B have changed places)
};

// One loop of each type at most, both operands unit-stride along K, K >= 16.
// All strides fit 32 bits.  112 bytes: a launch with up to so many in kernel
// arguments takes 2.7 to 2.9 us of the host, one with 120 to 1024 bytes 3.3 to
// 3.5 us.
struct I8Args {
  int8_t const * a;
  int8_t const * b;
  float const  * sa;       // null: 1
  float const  * sb;       // null: 1
  float const  * bias;     // null: 0
  void         * out;
  int32_t M, N;
  uint32_t k_flags;        // K (17 bits) and flags
  // strides from row (of A), column (row of B) and batch index to the next
  int32_t a_row, b_col;
  int32_t o_row, o_col;
  int32_t sa_row, sb_col;
  int32_t bias_step;       // along rows (BIAS_ROWS) or columns
  int32_t c[I8_TENSORS];

  enum : uint32_t { K_MASK = ( 1u << 20 ) - 1, OUT_BF16 = 1u << 20, RELU = 1u << 21, BIAS_ROWS = 1u << 22,
                    VEC_OUT = 1u << 23 };   // VEC_OUT: the output's columns are adjacent (tiles)
  __host__ __device__ int32_t K() const { return int32_t( k_flags & K_MASK ); }
  __host__ __device__ bool has( uint32_t flag ) const { return ( k_flags & flag ) != 0; }
};
static_assert( sizeof( I8Args ) == 112, "kernel arguments" );

// The kernels.  TILE_*: through LDS (contract_i8_tile.hip), rows (and K) at
// multiples of 16 bytes.
enum class I8Kernel : int32_t {
  GENERAL,            // any strides, 64 x 64 tiles (contract_i8.hip)
  FEW_4,              // a side of up to 4, K over the waves and in 4 parts (contract_i8_few.hip)
  FEW_8_PARTS,        // the same, a side of up to 8
  FEW_16_PARTS,       // a side of up to 16
  FEW_16,             // a side of up to 16, K over the waves
  FEW_32,             // a side of up to 32
  TILE_32x32,
  TILE_64x32,
  TILE_64x64,
  TILE_128x64,
  TILE_128x128,
  TILE_256x128,
  TILE_256x256,
  SHIFT_32x32,        // the same, rows anywhere
  SHIFT_64x64,
  SHIFT_128x128,
  SHIFT_256x128
};

// rows of both operands, and K, at multiples of n bytes
inline bool i8_aligned( I8Args const & a, int64_t n ) {
  return a.K() % n == 0 && uintptr_t( a.a ) % n == 0 && uintptr_t( a.b ) % n == 0 && a.a_row % n == 0
      && a.b_col % n == 0 && a.c[I8_A] % n == 0 && a.c[I8_B] % n == 0;
}
// 16, 4 or 1
inline int32_t i8_alignment( I8Args const & a ) {
  return i8_aligned( a, 16 ) ? 16 : i8_aligned( a, 4 ) ? 4 : 1;
}

// 16 k of a row where K ends inside them: the row's last 16 are loaded in
// their place, and those that belong to an earlier piece count as zeros on one
// operand's side.
struct I8Piece {
  int32_t at;      // first k to load, at least 0 (K >= 16)
  int32_t skip;    // leading bytes that count as zeros, 16: all
};
__device__ inline I8Piece i8_piece( int32_t k, int32_t K ) {
  return { min( k, K - 16 ), k < K ? max( k - ( K - 16 ), 0 ) : 16 };
}
// 16 bytes of a row on their way.  BYTES: at any address, read as the five
// aligned dwords that hold them (of which only those with a byte of the 16 are
// read) and shifted into place: 16-byte loads off a 4-byte boundary run at a
// third of the rate of aligned ones (2.3 TB/s of 7.5 from the cache, 5.4 so).
// Else: at a multiple of 4.
template< bool BYTES >
struct I8Vec {
  typedef int32_t v4 __attribute__( ( ext_vector_type( 4 ) ) );
  typedef v4 v4_dword __attribute__( ( aligned( 4 ) ) );
  v4      m_v;
  int32_t m_w;
  int32_t m_shift;
  __device__ __attribute__( ( always_inline ) ) inline void load( int8_t const * p ) {
    if constexpr( BYTES ) {
      uintptr_t const l_p = reinterpret_cast< uintptr_t >( p );
      m_v = *reinterpret_cast< v4_dword const * >( l_p & ~uintptr_t( 3 ) );
      m_w = *reinterpret_cast< int32_t const * >( ( l_p + 15 ) & ~uintptr_t( 3 ) );
      m_shift = int32_t( l_p & 3 );
    }
    else m_v = *reinterpret_cast< v4_dword const * >( p );
  }
  __device__ __attribute__( ( always_inline ) ) inline v4 value() const {
    if constexpr( !BYTES ) return m_v;
    else return v4{ int32_t( __builtin_amdgcn_alignbyte( m_v[1], m_v[0], m_shift ) ),
                    int32_t( __builtin_amdgcn_alignbyte( m_v[2], m_v[1], m_shift ) ),
                    int32_t( __builtin_amdgcn_alignbyte( m_v[3], m_v[2], m_shift ) ),
                    int32_t( __builtin_amdgcn_alignbyte( m_w, m_v[3], m_shift ) ) };
  }
};

// the bytes of dword d (0 to 3) of a piece that count
__device__ inline uint32_t i8_mask( int32_t skip, int32_t d ) {
  int32_t const l_z = skip - 4 * d;
  return l_z <= 0 ? 0xffffffffu : l_z >= 4 ? 0u : 0xffffffffu << ( 8 * l_z );
}

// scale, bias and last touch of one sum
__device__ inline float i8_finish( int32_t sum, float sa, float sb, float bias, int32_t relu ) {
  float const l_v = float( sum ) * sa * sb + bias;
  return relu && l_v < 0.0f ? 0.0f : l_v;       // a NaN stays
}

struct I8Plan {
  I8Kernel kernel = I8Kernel::GENERAL;
  int32_t  alignment = 0;              // of the operands' rows that the kernel was chosen for
  bool     swapped = false;            // A = right tensor, B = left tensor
  bool     has_sa = false, has_sb = false, has_bias = false;
  I8GeneralArgs args{};                // pointers set at execution
  I8Args   affine{};                   // kernels other than GENERAL; pointers set at execution
  int64_t  flops = 0;
  int64_t  bytes = 0;
  std::string desc;
};

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
             I8Plan        & plan );
int launch_i8( I8Plan const & plan,
               void const   * left,
               void const   * right,
               void const   * scale_left,
               void const   * scale_right,
               void const   * bias,
               void         * out,
               hipStream_t    stream );

int launch_i8_general( I8GeneralArgs const & a, hipStream_t stream );
int launch_i8_few( I8Args const & a, int64_t C, I8Kernel kernel, hipStream_t stream );
int launch_i8_tile( I8Args const & a, int64_t C, I8Kernel kernel, hipStream_t stream );

// ---------------------------------------------------------------------------
// rows rounded to 8-bit integers with one scale a row
// ---------------------------------------------------------------------------
struct QuantPlan {
  bool    norm = false;                // RMS norm (else: activation)
  int64_t rows = 0;
  int64_t cols = 0;
  int32_t dtype = ETIR_BF16;
  int32_t dtype_weight = ETIR_BF16;
  int32_t ktype = ETIR_KTYPE_UNDEFINED;
  float   eps = 0.0f;
  int64_t ld_in = 0, ld_second = 0, ld_total = 0, ld_q = 0, ld_values = 0;
  int64_t bytes = 0;                   // with every optional tensor
  std::string desc;
};
void describe_quant( QuantPlan & plan );

// One row: y = norm or activation of the inputs, q = rint( y * 127 / max|y| ).
// (112 bytes, as above.)
struct QuantArgs {
  void const * in;
  void const * second;      // residual (norm) or gate (activation); null: none
  void const * weight;      // norm: null: 1
  void       * total;       // norm: in + residual; null: not wanted
  int8_t     * q;
  float      * scale;
  void       * values;      // q * scale; null: not wanted
  int64_t ld_in, ld_second, ld_total, ld_q, ld_values;
  int32_t rows, cols;
  float   eps;
  int32_t mode;             // norm: 1 where the weight is fp32; activation: the kernel type
};
static_assert( sizeof( QuantArgs ) == 112, "kernel arguments" );

int launch_quant( QuantPlan const & plan, QuantArgs const & a, hipStream_t stream );

}  // namespace etir

#endif
