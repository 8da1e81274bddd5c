// The paged cache's address arithmetic, compiled for the host from the kernels' own header.
#include "../../tacotron_amd/csrc/taco_place.h"

extern "C" uint32_t place_divide(uint32_t n, uint32_t d) { return taco_divide(n, taco_make_divisor(d)); }
extern "C" void place_find(const int32_t* row, int32_t width, int32_t n_pages, int64_t at, uint32_t per_page, int32_t* out) {
  const taco_place p = taco_find(row, width, n_pages, at, taco_make_divisor(per_page));
  out[0] = p.page;
  out[1] = (int32_t)p.unit;
  out[2] = (int32_t)p.flag;
}
