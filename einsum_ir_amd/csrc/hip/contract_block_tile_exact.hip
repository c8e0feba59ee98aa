// The tiles of contract_block_tile.h: 8-bit numbers multiplied as bf16, with scales
// of either type.
#include "contract_block_tile.h"

namespace etir {

namespace {

template< int KIND, bool A_E5M2 >
int launch_type( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream ) {
  using namespace block;
  bool const l_rows = !a.has( BlockArgs::SB_BLOCKS );
  switch( layout ) {
    case BlockLayout::K_K:
      return l_rows ? launch_tiles< KIND, false, false, A_E5M2, true >( a, kernel, stream )
                    : launch_tiles< KIND, false, false, A_E5M2, false >( a, kernel, stream );
    case BlockLayout::K_ROWS:
      return l_rows ? launch_tiles< KIND, false, true, A_E5M2, true >( a, kernel, stream )
                    : launch_tiles< KIND, false, true, A_E5M2, false >( a, kernel, stream );
    case BlockLayout::ROWS_ROWS: return launch_tiles< KIND, true, true, A_E5M2, true >( a, kernel, stream );
    default: return fail( ETIR_COMPILATION_FAILED, "contraction: unknown layout" );
  }
}

}  // namespace

int launch_block_tile_exact( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream ) {
  if( a.has( BlockArgs::E8M0 ) ) {
    return a.has( BlockArgs::A_E5M2 ) ? launch_type< block::EXACT_E8M0, true >( a, kernel, layout, stream )
                                      : launch_type< block::EXACT_E8M0, false >( a, kernel, layout, stream );
  }
  return a.has( BlockArgs::A_E5M2 ) ? launch_type< block::EXACT, true >( a, kernel, layout, stream )
                                    : launch_type< block::EXACT, false >( a, kernel, layout, stream );
}

}  // namespace etir
