// What the kernels of a paged key/value cache share (PagedAttn: kernels.h).
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace nxd {

NXD_DEVICE int paged_new_tokens(const PagedAttn& p, int b) {
  const long n = p.lens ? p.lens[b] : p.W;
  return p.positions[b] < 0 ? 0 : (int)(n < 0 ? 0 : n > p.W ? p.W : n);
}
// One past the last key that a sequence's newest token sees; what lies behind the page table's end nobody sees
NXD_DEVICE int paged_keys(const PagedAttn& p, int b) {
  const int m = paged_new_tokens(p, b);
  if (m == 0) return 0;
  const long n = p.positions[b] + m, cap = (long)p.cols * p.ps;
  return (int)(n < cap ? n : cap);
}

}  // namespace nxd
