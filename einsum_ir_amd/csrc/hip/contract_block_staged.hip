// The tiles of contract_block_tile.h for operands at any address: bf16, 8-bit
// products on the matrix cores with scales of either type, and 8-bit numbers
// multiplied as bf16.  What is not at multiples of 16 bytes cannot go to LDS
// directly; a step waits in registers while the last one is multiplied, and a
// deeper store of steps costs more waves than it hides.  4096^3 one byte off: 130 us,
// with 4097 k 150, at multiples of 16 bytes 64.  Operands whose groups start and end
// inside a piece of 16 bytes come here too: groups of k with an operand along k,
// groups of rows with A along them.
#include "contract_block_tile.h"

namespace etir {

namespace {

template< int KIND, bool A_E5M2 >
int launch_type( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream ) {
  using namespace block;
  // without scales there is one, 1, for 128 rows, too
  bool const l_rows = KIND != BF16 && a.sb != nullptr && !a.has( BlockArgs::SB_BLOCKS );
  switch( layout ) {
    case BlockLayout::K_K:
      return l_rows ? launch_staged< KIND, false, false, A_E5M2, KIND != BF16 >( a, kernel, stream )
                    : launch_staged< KIND, false, false, A_E5M2, false >( a, kernel, stream );
    case BlockLayout::K_ROWS:
      return l_rows ? launch_staged< KIND, false, true, A_E5M2, KIND != BF16 >( a, kernel, stream )
                    : launch_staged< KIND, false, true, A_E5M2, false >( a, kernel, stream );
    case BlockLayout::ROWS_ROWS: return launch_staged< KIND, true, true, A_E5M2, KIND != BF16 >( a, kernel, stream );
    default: return fail( ETIR_COMPILATION_FAILED, "contraction: unknown layout" );
  }
}

}  // namespace

int launch_block_staged( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream ) {
  if( !a.has( BlockArgs::F8 ) ) return launch_type< block::BF16, false >( a, kernel, layout, stream );
  if( a.has( BlockArgs::OUT_BF16 ) ) {
    return a.has( BlockArgs::A_E5M2 ) ? launch_type< block::F8, true >( a, kernel, layout, stream )
                                      : launch_type< block::F8, false >( a, kernel, layout, stream );
  }
  return a.has( BlockArgs::A_E5M2 ) ? launch_type< block::EXACT, true >( a, kernel, layout, stream )
                                    : launch_type< block::EXACT, false >( a, kernel, layout, stream );
}

}  // namespace etir
