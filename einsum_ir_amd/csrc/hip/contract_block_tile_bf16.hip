// The tiles of contract_block_tile.h: bf16.
#include "contract_block_tile.h"

namespace etir {

int launch_block_tile_bf16( BlockArgs const & a, BlockKernel kernel, BlockLayout layout, hipStream_t stream ) {
  using namespace block;
  switch( layout ) {
    case BlockLayout::K_K:       return launch_tiles< BF16, false, false, false, false >( a, kernel, stream );
    case BlockLayout::K_ROWS:    return launch_tiles< BF16, false, true, false, false >( a, kernel, stream );
    case BlockLayout::ROWS_ROWS: return launch_tiles< BF16, true, true, false, false >( a, kernel, stream );
    default: return fail( ETIR_COMPILATION_FAILED, "contraction: unknown layout" );
  }
}

}  // namespace etir
