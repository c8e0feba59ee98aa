// Plans of block and grouped products without a GPU: reads one plan a line from
// standard input and prints what it is described as, or the code of its refusal.
// Planning asks the device's number and nothing else, which is answered here.
//   f8      <loops> <left> <right> <scale_left> <scale_right> <bias> <out> <block_left> <block_right> <types>... <last touch>
//   grouped <loops> <left> <right> <scale_left> <scale_right> <out> <ragged> <block_left> <block_right> <types>...
// <loops>: dimension types, then sizes; lists are "a,b,c" and an absent one is "-".
#include "einsum_ir_hip.h"
#include <cstdio>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

extern "C" int hipGetDevice( int * device ) {
  *device = 0;
  return 0;
}

namespace {

template< class T >
struct List {
  std::vector< T > values;
  bool there = false;
  explicit List( std::istream & in ) {
    std::string l_text, l_value;
    in >> l_text;
    there = l_text != "-";
    std::istringstream l_in( l_text );
    while( there && std::getline( l_in, l_value, ',' ) ) values.push_back( T( std::stoll( l_value ) ) );
  }
  T const * get() const { return there ? values.data() : nullptr; }
};

}  // namespace

int main() {
  std::string l_line;
  while( std::getline( std::cin, l_line ) ) {
    std::istringstream l_in( l_line );
    std::string l_kind;
    l_in >> l_kind;
    List< int32_t > const l_types( l_in );
    List< int64_t > const l_sizes( l_in ), l_left( l_in ), l_right( l_in ), l_sa( l_in ), l_sb( l_in );
    int64_t const l_n = int64_t( l_types.values.size() );
    etir_plan_t l_plan = nullptr;
    int l_err = 0;
    if( l_kind == "f8" ) {
      List< int64_t > const l_bias( l_in ), l_out( l_in );
      int32_t l_v[7];
      for( int32_t & l_x : l_v ) l_in >> l_x;
      l_err = etir_hip_contraction_f8_create( l_n, l_types.get(), l_sizes.get(), l_left.get(), l_right.get(), l_sa.get(), l_sb.get(),
                                              l_bias.get(), l_out.get(), l_v[0], l_v[1], l_v[2], l_v[3], l_v[4], l_v[5], l_v[6], &l_plan );
    }
    else {
      List< int64_t > const l_out( l_in );
      int64_t l_ragged = 0;
      int32_t l_v[6];
      l_in >> l_ragged;
      for( int32_t & l_x : l_v ) l_in >> l_x;
      l_err = etir_hip_contraction_grouped_create( l_n, l_types.get(), l_sizes.get(), l_left.get(), l_right.get(), l_sa.get(), l_sb.get(),
                                                   l_out.get(), l_ragged, l_v[0], l_v[1], l_v[2], l_v[3], l_v[4], l_v[5], &l_plan );
    }
    char l_text[512] = "";
    if( l_err == ETIR_SUCCESS ) {
      etir_hip_plan_describe( l_plan, l_text, sizeof( l_text ) );
      etir_hip_plan_destroy( l_plan );
    }
    else std::snprintf( l_text, sizeof( l_text ), "%d %s", l_err, etir_hip_last_error() );
    std::cout << l_text << std::endl;
  }
  return 0;
}
