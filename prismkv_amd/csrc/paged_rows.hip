// Rows into and out of the paged cache's pages where they are not copied as they
// are: turned by their positions, held in 4 bits, or read back.
#include <cfloat>

#include "paged_host.h"

namespace prismkv {
namespace {

// ------------------------------------------------------------------ append, with a turn or into 4 bits
//
// x' = x cos - y sin, y' = y cos + x sin for each pair of dims and the angle that
// belongs to it and to the row's position.  Bound by reading and writing the rows, once
// each: the angles' sines are computed once for a row (in LDS) and used by all of its
// heads.  The angle is an integer, 2^-64 of a turn: position times turns[j] modulo 2^64
// is exact for any position, where a product in fp32 is off by 0.06 radians at 10^6.
// Measured: 20011 rows of 32 + 8 + 8 heads of 64 in fp16, 47.4 us = 5.2 TB/s of what is
// read and written; one row for each of 128 sequences, 32 + 8 + 8 heads of 128, 5.6 us, most
// of it the launch and the chain lengths -> page -> store.
//
// In 4 bits 32 dims share a scale: a thread has 8 dims, so the largest of four
// neighbouring lanes' is the block's, and the conversion instruction divides, rounds
// (ties to even) and saturates.  Measured: 20011 rows of 8 heads of 128, k and v, 29.2 us =
// 3.6 TB/s; bound by the latency of a row's reads.  Four items' loads in flight for a thread
// were slower (with a read of all after it 54 us against 51; turned 58 against 47).

constexpr int kRowsEach = 8;   // packed rows of a workgroup
constexpr int64_t kLaunchRows = 1 << 26;  // (a launch has fewer than 2^32 threads: 2^27 rows)

struct PagedRows {
  const char *k, *v, *q;
  char *kp, *vp, *q_out;
  uint8_t *ks, *vs;
  const int32_t *table, *offsets, *lengths, *seen;
  const uint64_t* turns;
  int32_t *lengths_out, *seen_out, *positions, *positions_out;
  float *scores, *scores_out;
  unsigned* err;
  int64_t first_row, rows;                              // this launch's first, all
  int64_t k_row, k_head, v_row, v_head, q_row, q_head;  // bytes
  int64_t page_bytes, head_bytes, slot_bytes, scale_page, scale_head, scale_slot;
  PageDiv div;
  float amplitude;
  int sequences, kv_heads, heads, page_size, max_pages, pages, slots, rotary, interleaved;  // heads of q
};

struct RowPlace {
  size_t at, scales;  // bytes from the pages' base
  int64_t position;
  int b, slot, length;  // slot -1: a row that is dropped; length: of its sequence before
};

// The last b with offsets[b] <= row.
__device__ __forceinline__ int sequence_of(const int32_t* offsets, int sequences, int64_t row) {
  int lo = 0, hi = sequences;
  while (lo + 1 < hi) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ RowPlace row_place(const PagedRows& a, int64_t row) {
  RowPlace p{0, 0, 0, 0, -1, 0};
  int64_t step = 0;
  if (!a.offsets) {
    p.b = (int)row;
  } else {
    p.b = sequence_of(a.offsets, a.sequences, row);
    step = row - a.offsets[p.b];
    if (step < 0 || row >= a.offsets[p.b + 1]) return p;  // a row of no sequence
  }
  p.length = min(max(a.lengths[p.b], 0), a.slots);
  p.position = a.positions ? (int)((unsigned)a.seen[p.b] + (unsigned)step) : p.length + step;
  const int64_t slot = p.length + step;
  const int page = slot < a.slots ? a.table[(size_t)p.b * a.max_pages + a.div.of((int)slot)] : -1;
  if ((unsigned)page >= (unsigned)a.pages) {  // no page: the row is dropped
    report_error(a.err, error_host_slot(a.err), kErrPages);
    return p;
  }
  p.slot = (int)slot;
  const int in = p.slot - a.div.of(p.slot) * a.page_size;
  p.at = (size_t)page * a.page_bytes + (size_t)in * a.slot_bytes;
  p.scales = (size_t)page * a.scale_page + (size_t)in * a.scale_slot;
  return p;
}

// Lengths and tokens seen of sequence b with its packed rows; offsets that do not
// cover the rows, ascending from 0, are reported.
__device__ __forceinline__ void advance_rows(const PagedRows& a, int b) {
  const int from = a.offsets[b], to = a.offsets[b + 1], more = max(to - from, 0);
  if (from > to || (b == 0 && from) || (b == a.sequences - 1 && to != a.rows))
    report_error(a.err, error_host_slot(a.err), kErrRows);
  a.lengths_out[b] = (int)min((int64_t)max(a.lengths[b], 0) + more, (int64_t)a.slots);
  if (a.positions) a.seen_out[b] = a.seen[b] + more;
}

// Eight dims as loaded, in 32 bits, and back.
template <int DT>
struct Eight {
  uint4 x[kElem<DT> / 2];
  __device__ __forceinline__ void load(const char* p) {
#pragma unroll
    for (int i = 0; i < kElem<DT> / 2; ++i) x[i] = load_nt16(p + 16 * i);
  }
  __device__ __forceinline__ void widen(float (&f)[8]) const {
    if constexpr (kType<DT> == kFp32) {
      const float4 lo = *reinterpret_cast<const float4*>(&x[0]), hi = *reinterpret_cast<const float4*>(&x[1]);
      f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w;
      f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
    } else if constexpr (kType<DT> == kBf16) {
      unpack8(x[0], f);
    } else {
      const f16x8 h = __builtin_bit_cast(f16x8, x[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
    }
  }
  __device__ __forceinline__ void narrow(const float (&f)[8]) {
    if constexpr (kType<DT> == kFp32) {
      x[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      x[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    } else if constexpr (kType<DT> == kBf16) {
      bf16x8 h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (__bf16)f[i];
      x[0] = __builtin_bit_cast(uint4, h);
    } else {
      f16x8 h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (_Float16)f[i];
      x[0] = __builtin_bit_cast(uint4, h);
    }
  }
  __device__ __forceinline__ void store(char* p) const {
#pragma unroll
    for (int i = 0; i < kElem<DT> / 2; ++i) *reinterpret_cast<uint4*>(p + 16 * i) = x[i];
  }
};

// The scale byte of 32 values by the bits of the largest magnitude: a NaN's or an
// infinity's are the largest.  Above 1.75 of its power of two a value takes the next.
template <int DT>
__device__ __forceinline__ unsigned scale_byte(unsigned amax) {
  return amax >= 0x7f800000u
             ? 255u
             : (unsigned)min(max((int)((amax + 0x1fffffu) >> 23) - 2, kLeastScale<DT>), kMostScale<DT>);
}

// Eight codes of eight of the 32 values, the others being with the neighbouring lanes.
template <int DT>
__device__ __forceinline__ unsigned codes8(const float (&f)[8], unsigned& byte) {
  unsigned amax = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(f[i]) & 0x7fffffffu);
  amax = max(amax, __float_as_uint(xor1(__uint_as_float(amax))));
  amax = max(amax, __float_as_uint(xor2(__uint_as_float(amax))));
  byte = scale_byte<DT>(amax);
  const float scale = __uint_as_float(byte == 255u ? 0x3f800000u : byte << 23);
  unsigned c = 0u;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], scale, 3);
}

// Dims [c, c + 8) of a row turned: x as they are, y their partners' chunk (half layout).
__device__ __forceinline__ void turn8(const PagedRows& a, float (&x)[8], const float (&y)[8], const float2* row, int c) {
  const int half = a.rotary >> 1;
  if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 cs = row[(c + i) >> 1];
      const float u = x[i], w = x[i + 1];
      x[i] = u * cs.x - w * cs.y;
      x[i + 1] = w * cs.x + u * cs.y;
    }
  } else {
    const float sign = c < half ? -1.f : 1.f;
    const int j = c < half ? c : c - half;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 cs = row[j + i];
      x[i] = x[i] * cs.x + sign * y[i] * cs.y;
    }
  }
}

template <int DT, int D, bool kTurn>
__global__ __launch_bounds__(kPT) void paged_rows_kernel(PagedRows a) {
  constexpr int kC = D / 8;  // chunks of a head
  __shared__ RowPlace places[kRowsEach];
  extern __shared__ float2 angles[];  // [rows][rotary / 2] {cos, sin}
  const int tid = threadIdx.x, each = a.offsets ? kRowsEach : 1;
  const int64_t row0 = a.first_row + (int64_t)blockIdx.x * each;
  const int rows = (int)min((int64_t)each, a.rows - row0);
  if (tid < rows) places[tid] = row_place(a, row0 + tid);
  __syncthreads();
  const int half = a.rotary >> 1;
  if constexpr (kTurn) {
    for (int i = tid; i < rows * half; i += kPT) {
      const int r = i / half;
      const uint64_t phase = (uint64_t)places[r].position * a.turns[i - r * half];
      // (the upper 32 bits as a signed fraction of a turn; 2^-31 of a half turn each)
      float s, c;
      sincospif((float)(int)(phase >> 32) * 0x1p-31f, &s, &c);
      angles[i] = make_float2(c * a.amplitude, s * a.amplitude);
    }
    __syncthreads();
  }
  const int per_row = (a.heads + 2 * a.kv_heads) * kC, items = rows * per_row;
  for (int i = tid; i < items; i += kPT) {  // (a multiple of 4: the lanes of a block of 32 dims go together)
    const int r = i / per_row, head = (i - r * per_row) / kC, c = (i & (kC - 1)) * 8;
    const RowPlace& p = places[r];
    const int kind = head < a.heads ? 0 : head < a.heads + a.kv_heads ? 1 : 2;  // q, k, v
    const int h = head - (kind == 0 ? 0 : kind == 1 ? a.heads : a.heads + a.kv_heads);
    const char* from = kind == 0 ? a.q + (row0 + r) * a.q_row + h * a.q_head
                     : kind == 1 ? a.k + (row0 + r) * a.k_row + h * a.k_head
                                 : a.v + (row0 + r) * a.v_row + h * a.v_head;
    Eight<DT> x;
    x.load(from + c * kElem<DT>);
    float f[8];
    if (kTurn || kInFour<DT>) x.widen(f);
    if constexpr (kTurn) {
      const bool turned = kind < 2 && c < a.rotary;
      float y[8];
      if (!a.interleaved) {
        Eight<DT> partner = x;
        if (turned) partner.load(from + (c < half ? c + half : c - half) * kElem<DT>);
        partner.widen(y);
      }
      if (turned) {
        turn8(a, f, y, angles + r * half, c);
        x.narrow(f);
        if constexpr (kInFour<DT>) x.widen(f);
      }
    }
    if (kind == 0) {
      x.store(a.q_out + (((row0 + r) * a.heads + h) * D + c) * kElem<DT>);
      if constexpr (!kInFour<DT>) continue;
    }
    if constexpr (kInFour<DT>) {
      unsigned byte;
      const unsigned codes = codes8<DT>(f, byte);
      if (kind == 0 || p.slot < 0) continue;
      *reinterpret_cast<unsigned*>((kind == 1 ? a.kp : a.vp) + p.at + (size_t)h * a.head_bytes + c / 2) = codes;
      if ((c & 31) == 0) (kind == 1 ? a.ks : a.vs)[p.scales + (size_t)h * a.scale_head + c / 32] = (uint8_t)byte;
    } else if (p.slot >= 0) {
      x.store((kind == 1 ? a.kp : a.vp) + p.at + (size_t)h * a.head_bytes + c * kElem<DT>);
    }
  }
  if (a.positions)
    for (int i = tid; i < rows * a.kv_heads; i += kPT) {
      const RowPlace& p = places[i / a.kv_heads];
      if (p.slot < 0) continue;
      const size_t at = ((size_t)p.b * a.kv_heads + i % a.kv_heads) * a.slots + p.slot;
      a.scores[at] = a.scores_out[at] = 0.f;
      a.positions[at] = a.positions_out[at] = (int)p.position;
    }
  if (!a.offsets) {  // (the row's workgroup alone reads its sequence's length)
    if (tid == 0) {
      a.lengths_out[blockIdx.x] = min(places[0].length + 1, a.slots);
      if (a.positions) a.seen_out[blockIdx.x] = (int)places[0].position + 1;
    }
  } else if (a.lengths_out != a.lengths) {
    for (int64_t b = (int64_t)blockIdx.x * kPT + tid; b < a.sequences; b += (int64_t)gridDim.x * kPT)
      advance_rows(a, (int)b);
  }
}

// Packed rows onto lengths that are advanced in place: after every workgroup has read them.
__global__ __launch_bounds__(kPT) void paged_rows_advance_kernel(PagedRows a) {
  const int b = blockIdx.x * kPT + threadIdx.x;
  if (b < a.sequences) advance_rows(a, b);
}

// ------------------------------------------------------------------ read

// The rows of the sequences' last slots, widened from 4 bits (exactly) or copied: bound
// by reading and writing them; a thread has 8 dims of a row's key and value.  Measured: 20011
// rows of 8 heads of 128 out of 4 bits 19.4 us = 5.3 TB/s.
struct PagedRead {
  const char *kp, *vp;
  const uint8_t *ks, *vs;
  char *k, *v;
  const int32_t *table, *offsets, *lengths;
  unsigned* err;
  int64_t first_row, rows;
  int64_t page_bytes, head_bytes, slot_bytes, scale_page, scale_head, scale_slot;
  PageDiv div;
  int sequences, kv_heads, page_size, max_pages, pages, slots;
};

// The place of a row (slot -1: none); reports a slot or a page that there is not.
__device__ __forceinline__ RowPlace read_place(const PagedRead& a, int64_t row) {
  RowPlace p{0, 0, 0, 0, -1, 0};
  int64_t back = 1;  // from the sequence's end
  if (!a.offsets) {
    p.b = (int)row;
  } else {
    p.b = sequence_of(a.offsets, a.sequences, row);
    const int from = a.offsets[p.b], to = a.offsets[p.b + 1];
    if (row < from || row >= to) return p;  // a row of no sequence
    back = to - row;
  }
  const int64_t slot = min(max(a.lengths[p.b], 0), a.slots) - back;
  if (slot < 0) {
    report_error(a.err, error_host_slot(a.err), kErrHeld);
    return p;
  }
  const int page = a.table[(size_t)p.b * a.max_pages + a.div.of((int)slot)];
  if ((unsigned)page >= (unsigned)a.pages) {
    report_error(a.err, error_host_slot(a.err), kErrPages);
    return p;
  }
  p.slot = (int)slot;
  const int in = p.slot - a.div.of(p.slot) * a.page_size;
  p.at = (size_t)page * a.page_bytes + (size_t)in * a.slot_bytes;
  p.scales = (size_t)page * a.scale_page + (size_t)in * a.scale_slot;
  return p;
}

template <int DT>
__device__ __forceinline__ void widen_codes(unsigned codes, unsigned byte, float (&f)[8]) {
  const float scale = __uint_as_float(byte << 23);  // (255: an infinity, which makes NaN of any code)
#define PRISMKV_PAIR(i)                                                              \
  {                                                                                  \
    const auto x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, i);        \
    f[2 * i] = x[0];                                                                 \
    f[2 * i + 1] = x[1];                                                             \
  }
  PRISMKV_PAIR(0) PRISMKV_PAIR(1) PRISMKV_PAIR(2) PRISMKV_PAIR(3)
#undef PRISMKV_PAIR
}

template <int DT, int D>
__global__ __launch_bounds__(kPT) void paged_read_kernel(PagedRead a) {
  constexpr int kC = D / 8;
  __shared__ RowPlace places[kRowsEach];
  const int tid = threadIdx.x;
  const int64_t row0 = a.first_row + (int64_t)blockIdx.x * kRowsEach;
  const int rows = (int)min((int64_t)kRowsEach, a.rows - row0);
  if (tid < rows) places[tid] = read_place(a, row0 + tid);
  if (row0 == 0 && a.offsets)
    for (int b = tid; b < a.sequences; b += kPT) {
      const int from = a.offsets[b], to = a.offsets[b + 1];
      if (from > to || (b == 0 && from) || (b == a.sequences - 1 && to != a.rows))
        report_error(a.err, error_host_slot(a.err), kErrOffsets);
    }
  __syncthreads();
  const int per_row = a.kv_heads * kC, items = rows * per_row;
  for (int i = tid; i < items; i += kPT) {
    const int r = i / per_row, h = (i - r * per_row) / kC, c = (i & (kC - 1)) * 8;
    const RowPlace& p = places[r];
    Eight<DT> k{}, v{};
    if (p.slot >= 0) {
      if constexpr (kInFour<DT>) {
        const size_t at = p.at + (size_t)h * a.head_bytes + c / 2, s = p.scales + (size_t)h * a.scale_head + c / 32;
        float f[8];
        const unsigned kc = *reinterpret_cast<const unsigned*>(a.kp + at), vc = *reinterpret_cast<const unsigned*>(a.vp + at);
        const unsigned kb = a.ks[s], vb = a.vs[s];
        widen_codes<DT>(kc, kb, f);
        k.narrow(f);
        widen_codes<DT>(vc, vb, f);
        v.narrow(f);
      } else {
        const size_t at = p.at + (size_t)h * a.head_bytes + c * kElem<DT>;
        k.load(a.kp + at);
        v.load(a.vp + at);
      }
    }
    const size_t to = (((row0 + r) * a.kv_heads + h) * D + c) * kElem<DT>;
    k.store(a.k + to);
    v.store(a.v + to);
  }
}

template <int DT, int D>
int launch_rows(PagedRows a, hipStream_t stream) {
  const bool turn = a.turns != nullptr;
  const auto kernel = turn ? paged_rows_kernel<DT, D, true> : paged_rows_kernel<DT, D, false>;
  const int lds = turn ? (a.offsets ? kRowsEach : 1) * (a.rotary / 2) * (int)sizeof(float2) : 0;
  if (!a.offsets) {
    hipLaunchKernelGGL(kernel, dim3(a.sequences), dim3(kPT), lds, stream, a);
    return (int)hipGetLastError();
  }
  for (; a.first_row < a.rows; a.first_row += kLaunchRows) {
    const int64_t more = a.rows - a.first_row < kLaunchRows ? a.rows - a.first_row : kLaunchRows;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((more + kRowsEach - 1) / kRowsEach)), dim3(kPT), lds, stream, a);
    if (const int rc = (int)hipGetLastError()) return rc;
  }
  if (a.rows && a.lengths_out != a.lengths) return 0;  // (advanced by the rows' launches)
  hipLaunchKernelGGL(paged_rows_advance_kernel, dim3((a.sequences + kPT - 1) / kPT), dim3(kPT), 0, stream, a);
  return (int)hipGetLastError();
}

template <int DT, int D>
int launch_read(PagedRead a, hipStream_t stream) {
  do {  // (once for no rows, whose offsets are looked at too)
    const int64_t more = a.rows - a.first_row < kLaunchRows ? a.rows - a.first_row : kLaunchRows;
    const unsigned groups = (unsigned)((more + kRowsEach - 1) / kRowsEach);
    hipLaunchKernelGGL((paged_read_kernel<DT, D>), dim3(groups ? groups : 1), dim3(kPT), 0, stream, a);
    if (const int rc = (int)hipGetLastError()) return rc;
    a.first_row += kLaunchRows;
  } while (a.first_row < a.rows);
  return 0;
}

// f.template of<DT, D>() for the cache's type and head dimension.
template <typename F>
int by_type(int dtype, int head_dim, F f) {
#define PRISMKV_DIMS(DT) \
  return head_dim == 64 ? f.template of<DT, 64>() : head_dim == 128 ? f.template of<DT, 128>() : f.template of<DT, 256>()
  switch (dtype) {
    case kBf16: PRISMKV_DIMS(kBf16);
    case kFp16: PRISMKV_DIMS(kFp16);
    case kFp32: PRISMKV_DIMS(kFp32);
    case kFour | kBf16: PRISMKV_DIMS(kFour | kBf16);
    default: PRISMKV_DIMS(kFour | kFp16);
  }
#undef PRISMKV_DIMS
}

struct RowsLaunch {
  const PagedRows& a;
  hipStream_t stream;
  template <int DT, int D>
  int of() const { return launch_rows<DT, D>(a, stream); }
};

struct ReadLaunch {
  const PagedRead& a;
  hipStream_t stream;
  template <int DT, int D>
  int of() const { return launch_read<DT, D>(a, stream); }
};

}  // namespace
}  // namespace prismkv

using namespace prismkv;

extern "C" {

int prismkv_paged_append_rows(const prismkv_paged_cache* cache, const prismkv_paged_cache* into, uint64_t k, uint64_t v,
                              uint64_t q, uint64_t q_out, uint64_t offsets, uint64_t turns, int64_t rows,
                              int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                              int64_t q_row_stride, int64_t q_head_stride, int heads, int rotary_dim, int interleaved,
                              double amplitude, uint64_t stream) {
  if (const int rc = check_cache(cache, into, false)) return rc;
  const prismkv_paged_cache& c = *cache;
  if (rows < 0 || rows > INT32_MAX || (!offsets && rows != c.sequences)) return kBadSize;
  if (rows && (!k || !v)) return kBadSize;
  if ((heads != 0) != (q != 0) || (q != 0) != (q_out != 0) || heads < 0 || heads > 1024 * 65535) {
    if (!(heads > 0 && !rows)) return kBadSize;  // (no rows have no address)
  }
  if (!turns && (q || rotary_dim || interleaved)) return kBadSize;
  if (turns && (rotary_dim < 16 || rotary_dim > c.head_dim || rotary_dim % 16 || interleaved < 0 || interleaved > 1 ||
                !(amplitude >= -FLT_MAX && amplitude <= FLT_MAX)))
    return kBadSize;
  const int64_t es = element_bytes(c.dtype), limit = 1ll << 40;
  for (const int64_t stride : {k_row_stride, k_head_stride, v_row_stride, v_head_stride, q_row_stride, q_head_stride})
    if (stride < -limit || stride > limit || stride * es & 15) return kBadSize;
  if ((k | v | q | q_out) & 15 || offsets & 3 || turns & 7) return kBadSize;
  const int64_t per_row = ((int64_t)heads + 2 * c.kv_heads) * (c.head_dim / 8);  // items of a workgroup fit 32 bits
  if (per_row * kRowsEach > INT32_MAX) return kBadSize;
  PagedRows a{};
  a.k = reinterpret_cast<const char*>(k);
  a.v = reinterpret_cast<const char*>(v);
  a.q = reinterpret_cast<const char*>(q);
  a.q_out = reinterpret_cast<char*>(q_out);
  a.kp = reinterpret_cast<char*>(c.k);
  a.vp = reinterpret_cast<char*>(c.v);
  a.table = reinterpret_cast<const int32_t*>(c.table);
  a.offsets = reinterpret_cast<const int32_t*>(offsets);
  a.turns = reinterpret_cast<const uint64_t*>(turns);
  a.lengths = reinterpret_cast<const int32_t*>(c.lengths);
  a.lengths_out = reinterpret_cast<int32_t*>(into->lengths);
  a.seen = reinterpret_cast<const int32_t*>(c.seen);
  a.seen_out = reinterpret_cast<int32_t*>(into->seen);
  a.positions = reinterpret_cast<int32_t*>(c.positions);
  a.positions_out = reinterpret_cast<int32_t*>(into->positions);
  a.scores = reinterpret_cast<float*>(c.scores);
  a.scores_out = reinterpret_cast<float*>(into->scores);
  a.err = reinterpret_cast<unsigned*>(c.err);
  a.rows = rows;
  a.k_row = k_row_stride * es;
  a.k_head = k_head_stride * es;
  a.v_row = v_row_stride * es;
  a.v_head = v_head_stride * es;
  a.q_row = q_row_stride * es;
  a.q_head = q_head_stride * es;
  const int64_t pes = page_element_bytes(c.dtype);
  a.page_bytes = c.page_stride * pes;
  a.head_bytes = c.head_stride * pes;
  a.slot_bytes = c.slot_stride * pes;
  if (c.dtype >= kFour) {
    a.ks = reinterpret_cast<uint8_t*>(c.k_scales);
    a.vs = reinterpret_cast<uint8_t*>(c.v_scales);
    a.scale_page = c.scale_page_stride;
    a.scale_head = c.scale_head_stride;
    a.scale_slot = c.scale_slot_stride;
  }
  a.div = page_div(c.page_size);
  a.amplitude = (float)amplitude;
  a.sequences = c.sequences;
  a.kv_heads = c.kv_heads;
  a.heads = heads;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.pages = (int)c.pages;
  a.slots = c.page_size * c.max_pages;
  a.rotary = rotary_dim;
  a.interleaved = interleaved;
  return by_type(c.dtype, c.head_dim, RowsLaunch{a, (hipStream_t)stream});
}

int prismkv_paged_read(const prismkv_paged_cache* cache, uint64_t offsets, uint64_t k_out, uint64_t v_out, int64_t rows,
                       uint64_t stream) {
  if (const int rc = check_cache(cache, cache, false)) return rc;
  const prismkv_paged_cache& c = *cache;
  if (rows < 0 || rows > INT32_MAX || (!offsets && rows != c.sequences)) return kBadSize;
  if ((rows && (!k_out || !v_out)) || (k_out | v_out) & 15 || offsets & 3) return kBadSize;
  if ((int64_t)c.kv_heads * (c.head_dim / 8) * kRowsEach > INT32_MAX) return kBadSize;
  PagedRead a{};
  a.kp = reinterpret_cast<const char*>(c.k);
  a.vp = reinterpret_cast<const char*>(c.v);
  a.k = reinterpret_cast<char*>(k_out);
  a.v = reinterpret_cast<char*>(v_out);
  a.table = reinterpret_cast<const int32_t*>(c.table);
  a.offsets = reinterpret_cast<const int32_t*>(offsets);
  a.lengths = reinterpret_cast<const int32_t*>(c.lengths);
  a.err = reinterpret_cast<unsigned*>(c.err);
  a.rows = rows;
  const int64_t pes = page_element_bytes(c.dtype);
  a.page_bytes = c.page_stride * pes;
  a.head_bytes = c.head_stride * pes;
  a.slot_bytes = c.slot_stride * pes;
  if (c.dtype >= kFour) {
    a.ks = reinterpret_cast<const uint8_t*>(c.k_scales);
    a.vs = reinterpret_cast<const uint8_t*>(c.v_scales);
    a.scale_page = c.scale_page_stride;
    a.scale_head = c.scale_head_stride;
    a.scale_slot = c.scale_slot_stride;
  }
  a.div = page_div(c.page_size);
  a.sequences = c.sequences;
  a.kv_heads = c.kv_heads;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.pages = (int)c.pages;
  a.slots = c.page_size * c.max_pages;
  return by_type(c.dtype, c.head_dim, ReadLaunch{a, (hipStream_t)stream});
}

}  // extern "C"
