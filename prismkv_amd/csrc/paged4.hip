// Attention of one new query token of every sequence over pages in 4 bits: the
// kernels of paged_attend.h, which read 17/64 of the bytes of 16-bit pages.  Measured: 65792
// tokens of 8 x 4 heads in bf16 23.2 us = 3.1 TB/s (from 16-bit pages 46.8); 32 sequences of
// 6.4K tokens in fp16 51.4 us = 4.3 TB/s.  About 10 us of either are the launch, the chain
// lengths -> page -> rows and the join; what is added to a length goes at 5.2 TB/s.
#include "paged_attend.h"

namespace prismkv {

int attend_in_four(const PagedAttend& a, int dtype, int head_dim, int64_t units, hipStream_t stream) {
  return dtype == (kFour | kBf16) ? launch_attend_dim<kFour | kBf16>(a, head_dim, units, stream)
                                  : launch_attend_dim<kFour | kFp16>(a, head_dim, units, stream);
}

}  // namespace prismkv
