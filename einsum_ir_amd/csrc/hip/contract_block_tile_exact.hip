// The tiles of contract_block_tile.h: 8-bit numbers multiplied as bf16.
#include "contract_block_tile.h"

namespace etir {

namespace {

template< bool A_E5M2 >
int launch_type( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream ) {
  using namespace block;
  bool const l_rows = !a.has( BlockArgs::SB_BLOCKS );
  switch( layout ) {
    case BlockLayout::K_K:
      return l_rows ? launch_tiles< EXACT, false, false, A_E5M2, true >( a, kernel, stream )
                    : launch_tiles< EXACT, false, false, A_E5M2, false >( a, kernel, stream );
    case BlockLayout::K_ROWS:
      return l_rows ? launch_tiles< EXACT, false, true, A_E5M2, true >( a, kernel, stream )
                    : launch_tiles< EXACT, false, true, A_E5M2, false >( a, kernel, stream );
    case BlockLayout::ROWS_ROWS: return launch_tiles< EXACT, true, true, A_E5M2, true >( a, kernel, stream );
    default: return fail( ETIR_COMPILATION_FAILED, "contraction: unknown layout" );
  }
}

}  // namespace

int launch_block_tile_exact( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream ) {
  return a.has( BlockArgs::A_E5M2 ) ? launch_type< true >( a, kernel, layout, stream ) : launch_type< false >( a, kernel, layout, stream );
}

}  // namespace etir
