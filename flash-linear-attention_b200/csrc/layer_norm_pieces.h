// The elements of a row that layer_norm.cu moves at a time.  No CUDA in here: a host compiler can check the rule.
#pragma once
#include <stdint.h>

#include <initializer_list>

#include "../../include/b200gdn.h"

namespace gdn {

// 16 bytes of the rows' elements, of 16-bit ones else two, else one: what divides the width and what every tensor that is read or
// written so lies on a boundary of.  N parameters are read N x their own size at once (16 bytes at most), which may be more than the
// rows' N elements take.
inline int layer_norm_piece(const b200gdn_layer_norm_args& a) {
  const int size = a.dtype == 2 ? 4 : 2;
  auto addresses = [](std::initializer_list<const void*> all) {
    uintptr_t bits = 0;
    for (const void* p : all) bits |= reinterpret_cast<uintptr_t>(p);
    return bits;
  };
  const uintptr_t rows = addresses({a.x, a.residual, a.z, a.y, a.dy, a.dz, a.dx}), params = addresses({a.weight, a.bias});
  const int param_size = a.param_dtype == B200GDN_F32 ? 4 : 2;
  for (int n = 16 / size; n >= 2; n = n > 2 && size == 2 ? 2 : 1)
    if (a.D % n == 0 && rows % (n * size) == 0 && params % (n * param_size < 16 ? n * param_size : 16) == 0) return n;
  return 1;
}

}  // namespace gdn
