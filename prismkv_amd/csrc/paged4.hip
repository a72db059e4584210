// Attention of one new query token of every sequence over pages in 4 bits: the
// kernels of paged_attend.h, which read 17/64 of the bytes of 16-bit pages.
#include "paged_attend.h"

namespace prismkv {

int attend_in_four(const PagedAttend& a, int dtype, int head_dim, int64_t units, hipStream_t stream) {
  return dtype == (kFour | kBf16) ? launch_attend_dim<kFour | kBf16>(a, head_dim, units, stream)
                                  : launch_attend_dim<kFour | kFp16>(a, head_dim, units, stream);
}

}  // namespace prismkv
