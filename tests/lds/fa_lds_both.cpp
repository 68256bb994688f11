// Host build of the offsets of lds::TileBoth, for tests/test_lds_both.py.
#include "fa_lds_layout.h"

template <int D>
static int offset(int what, int lane, int i) {
  using T = fa::lds::TileBoth<D>;
  return what == 0 ? T::swz(i) : what == 1 ? T::row_offset(lane) ^ T::row_step(i) : T::turned_offset(lane) ^ T::turned_block(i);
}

extern "C" int fa_lds_both(int d, int what, int lane, int i) {
  return d == 128 ? offset<128>(what, lane, i) : offset<64>(what, lane, i);
}
