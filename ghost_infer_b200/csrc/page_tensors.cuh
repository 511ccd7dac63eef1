// Storage tensors of cache pages, [layers][pages][heads][64][numbers], as kernels that move whole rows take them.
#pragma once

#include "common.cuh"

namespace gi {

struct PageTensors {
  static constexpr int MOST = 8;
  void* base[MOST];
  int layers[MOST], pages[MOST], heads[MOST], row_units[MOST];       // a row's size in units of 16, 4 or 2 bytes

  // From five words a tensor: address, layers, pages, heads, bytes of a row.  `unit`: the widest of 16, 4 and 2 bytes that all rows
  // and addresses are multiples of.
  int read(const long* words, int n, int* unit, const char* what) {
    if (n < 0 || n > MOST) return fail(GI_ERR_UNSUPPORTED, "%s: %d tensors of pages, at most %d in one launch", what, n, MOST);
    *this = {};
    *unit = 16;
    for (int i = 0; i < n; ++i) {
      const long* w = words + 5 * i;
      for (int k = 1; k < 5; ++k)
        if (w[k] < 1 || w[k] > 0x3fffffffL) return fail(GI_ERR_ARG, "%s: tensor %d has %ld layers, %ld pages, %ld heads, rows of %ld bytes", what, i, w[1], w[2], w[3], w[4]);
      if (w[4] % 2 != 0 || (w[0] & 1)) return fail(GI_ERR_ARG, "%s: rows of %ld bytes do not come in units of 2", what, w[4]);
      while (*unit > 2 && (w[4] % *unit != 0 || w[0] % *unit != 0)) *unit = *unit == 16 ? 4 : 2;
    }
    for (int i = 0; i < n; ++i) {
      const long* w = words + 5 * i;
      base[i] = (void*)w[0], layers[i] = (int)w[1], pages[i] = (int)w[2], heads[i] = (int)w[3], row_units[i] = (int)(w[4] / *unit);
    }
    return GI_OK;
  }
};

}  // namespace gi
