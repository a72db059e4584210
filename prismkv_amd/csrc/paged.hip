// The paged key-value cache: writing rows into pages, attention of one new
// query token of every sequence over its pages, and eviction by accumulated
// attention weight.
//
// K and V pages are [pages][kv_heads][page_size][head_dim] with any strides of
// 16-byte multiples (the same for both); slot t of sequence b lies in page
// table[b][t / page_size].  A table entry outside [0, pages) within a
// sequence's length is reported through the cache's error word and never read
// through.
#include "paged.h"

#include <cfloat>

#include "prismkv_hip.h"

namespace prismkv {
namespace {

// ------------------------------------------------------------------ attention
//
// s_t = scale q.k_t, p_t = e^(s_t - m) / z, o = sum p_t v_t for the `group`
// query heads of one KV head: every K and V row is read once for all of them
// (2 bytes x 2 head_dim per 4 group head_dim flops), so the kernel is bound by
// the reads.  One pass with the running maximum and sum (flash form).
//
// Split: the tokens of all pairs of a sequence and a KV head (with more than 16
// query heads a tile of them) are dealt evenly to the workgroups, on the device,
// where the lengths are; a workgroup's share may end one pair and begin others.
// Each of its waves takes every 8th 32-token tile (fp32: 16 tokens) by itself: no
// barrier and no LDS until the waves' states meet at a pair's end.  A pair of
// several workgroups is joined from their states in the order of its tokens, by
// the last to arrive or by a second launch, so the result does not depend on the
// order of arrival.
//
// Measured (MI355X, launches after one another in a graph): 65792 tokens, 8 x 4
// heads, bf16, 47.3 us = 5.7 TB/s; 32 sequences of 6.4K tokens 136 us = 6.2 TB/s
// (a plain read of as much memory reaches 6.9); 16 x 8192 of head_dim 256 in fp32, 2
// x 4 heads, 92 us = 5.9; of head_dim 64, 8 x 4 heads, 48 us = 5.6; 75 tokens 6.4 us.
// About 6 us of a call are the launch and the chain lengths -> page -> rows, 3.7 more
// the join (65792 tokens 43.7 us without it).

// 16-bit types: P is a sum of terms of the type, each with a product of its own into
// one accumulator: bf16 takes three, which hold all 24 bits of an fp32 p (with two,
// outputs that cancel are off by 2^-17 of their terms; 65792 tokens, 8 x 4 heads take
// as long with either), fp16 two, 22 bits.  Every term is positive wherever p is, so
// that an infinite V is not multiplied by a term of 0: at least the type's least
// number, which for fp16, with its bias, is 2^-39 of the maximum's weight.
// The tile of one step as loaded.  16-bit (32 tokens, two 16-token blocks):
// lane (j, q) holds row j of each block at dims 32c + 8q .. +8 (K, the A operand
// of the 16x16x32 product) and of rows 4q + t (V) 16 bytes out of every 256 (8 of
// head_dim 64's 128), so that the 16 lanes of a load cover whole rows.  Column
// block n of the output takes element n of a lane, dim(n, j); the rows' pairs are
// joined per dim with one byte permutation.
// fp32 (16 tokens): K dims 16c + 4q .. +4 (four 16x16x4 products per load), V
// the same with float columns.
template <int DT, int D>
struct Tile {
  static constexpr int kBlocks = DT == kFp32 ? 1 : 2;
  static constexpr int kTokens = 16 * kBlocks;
  static constexpr int kKLoads = D * kElem<DT> / 64;        // 16-byte loads of a K row per lane
  static constexpr int kVWords = D * kElem<DT> / 64;        // 32-bit words of a V row per lane
  static constexpr int kVStep = kVWords < 4 ? 4 * kVWords : 16;  // bytes of a piece
  static constexpr int kRun = kVStep / kElem<DT>;           // elements of a piece
  static __device__ __forceinline__ int dim(int n, int j) { return n / kRun * (16 * kRun) + j * kRun + n % kRun; }
  uint4 k[kBlocks][kKLoads];
  unsigned v[kBlocks][4][kVWords];
};

template <int W>
__device__ __forceinline__ void load_words(unsigned (&dst)[W], const char* p) {
  if constexpr (W == 2) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    dst[0] = x.x;
    dst[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const uint4 x = load_nt16(p + 64 * i);
      dst[i] = x.x;
      dst[i + 1] = x.y;
      dst[i + 2] = x.z;
      dst[i + 3] = x.w;
    }
  }
}

template <int W>
__device__ __forceinline__ void load_words_buf(unsigned (&dst)[W], __amdgpu_buffer_rsrc_t r, unsigned byte_offset) {
  if constexpr (W == 2) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(r, byte_offset, 0, 2);
    dst[0] = x[0];
    dst[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const uint4 x = load_nt16_buf(r, byte_offset + 64 * i);
      dst[i] = x.x;
      dst[i + 1] = x.y;
      dst[i + 2] = x.z;
      dst[i + 3] = x.w;
    }
  }
}

// Element N of two rows' words as a pair (low half from a).
template <int N, int W>
__device__ __forceinline__ unsigned pair16(const unsigned (&a)[W], const unsigned (&b)[W]) {
  return __builtin_amdgcn_perm(b[N >> 1], a[N >> 1], (N & 1) ? 0x07060302u : 0x05040100u);
}

template <int DT>
__device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// p >= 0 as terms of the 16-bit type, each in the upper half of a word.  A NaN may be
// lost here: the sum of the weights has it.
template <int DT>
constexpr int kTerms = DT == kBf16 ? 3 : 2;
template <int DT>
__device__ __forceinline__ void split16(float p, unsigned (&term)[kTerms<DT>]) {
  if constexpr (DT == kBf16) {
    // 8 bits each from the top, which is exact (as signed integers: a remainder
    // below 0 is left behind a term that was raised)
    const int least = p > 0.f ? 0x10000 : 0;
    const int hi = max(__float_as_int(p) & (int)0xffff0000, least);
    const float rest = p - __int_as_float(hi);
    const int mid = max(__float_as_int(rest) & (int)0xffff0000, least);
    term[0] = (unsigned)hi;
    term[1] = (unsigned)mid;
    term[2] = (unsigned)max(__float_as_int(rest - __int_as_float(mid)), least);
  } else {
    // the head rounded down, so that the remainder is positive
    const float least = p > 0.f ? 0x1p-24f : 0.f, head = fmaxf(p, least);
    const auto h = __builtin_amdgcn_cvt_pkrtz(0.f, head);  // {0, head}
    const _Float16 l = (_Float16)fmaxf(head - (float)h[1], least);
    term[0] = __builtin_bit_cast(unsigned, h);
    term[1] = (unsigned)__builtin_bit_cast(unsigned short, l) << 16;
  }
}

// The upper halves of two words (low half from a).
__device__ __forceinline__ unsigned upper16(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

template <int N, int DT, int D>
__device__ __forceinline__ void pv_columns(f32x4 (&acc)[D / 16], const Tile<DT, D>& t,
                                           const u32x4 (&p)[kTerms<DT>]) {
  if constexpr (N < D / 16) {
    const u32x4 vb = {pair16<N>(t.v[0][0], t.v[0][1]), pair16<N>(t.v[0][2], t.v[0][3]),
                      pair16<N>(t.v[1][0], t.v[1][1]), pair16<N>(t.v[1][2], t.v[1][3])};
#pragma unroll
    for (int i = 0; i < kTerms<DT>; ++i) acc[N] = mfma32<DT>(p[i], vb, acc[N]);
    pv_columns<N + 1, DT, D>(acc, t, p);
  }
}

// 2^(scale s - m): one rounding of the difference.  m is a rounded product itself;
// from 2^22 on, where its rounding is 1/8 and more (and at 2^32 takes all of the
// exponent's range), the other products are rounded as it was, so that the largest
// score's weight is 1.  m is finite or +infinity (no_less): where no score is above
// -infinity, 0 serves.
__device__ __forceinline__ float weight(float s, float scale, float m) {
#pragma clang fp contract(off)
  const float product = s * scale;
  const float rounded = product - m;
  return __builtin_amdgcn_exp2f(fabsf(m) < 0x1p22f ? fmaf(s, scale, -m) : rounded);
}
__device__ __forceinline__ float no_less(float m) { return m == -INFINITY ? 0.f : m; }

// Factor of a state with maximum m under the joint maximum M >= m (no state: 0).
__device__ __forceinline__ float rescale(float m, float M) {
  return m == -INFINITY ? 0.f : m == M ? 1.f : exp2f(m - M);
}

// The joint maximum and sum of a pair's head g over its states, and the states'
// factors in wt[c * stride] (LDS); by one wave.
__device__ __forceinline__ float2 join_sums(const float* base, const PagedParts& parts, unsigned state_stride, int g,
                                            float* wt, int stride) {
  const int lane = threadIdx.x & 63;
  float M = -INFINITY, den = 0.f;
  for (int c0 = 0; c0 < parts.chunks; c0 += 64) {
    const int c = c0 + lane;
    const bool in = c < parts.chunks;
    const float2 mz = ld_dev2(base + (in && c ? 2 * c : parts.odd) * state_stride + 2 * g);
    const float m = in ? mz.x : -INFINITY;
    const float nM = fmaxf(M, wave_max(m));
    den = den * rescale(M, nM) + wave_sum(in ? rescale(m, nM) * mz.y : 0.f);
    M = nM;
    if (in && wt) wt[c * stride] = m;
  }
  if (wt)
    for (int c = lane; c < parts.chunks; c += 64) wt[c * stride] = rescale(wt[c * stride], M);
  return make_float2(M, den);
}

// Joins columns [col0, col0 + columns) (4 floats each of the [rows][D] output) of a
// pair's states, by a workgroup of kThreads: the maxima and sums a wave per head,
// while the first states' loads are in flight, then a thread per column and share
// of the states, the shares added in LDS.
template <int DT, int D, int kThreads>
__device__ __forceinline__ void join_states(const PagedAttend& a, size_t head0, int rows, const PagedParts& parts, int col0,
                                            int columns, float* lds) {
  const int tid = threadIdx.x, w = tid >> 6;
  float4* part = reinterpret_cast<float4*>(lds);  // [threads]
  float* top = lds + 4 * kThreads;                // [16] joint maxima, [16] sums
  float* wt = top + 32;                           // [chunks][rows] factors
  const float* base = a.state + (size_t)2 * parts.unit * a.state_stride;
  const __amdgpu_buffer_rsrc_t r = raw_buffer(base, 2 * parts.chunks * (int)a.state_stride * 4);
  const int chunks = parts.chunks;
  const int shares = max(kThreads / columns, 1), share = tid / columns;  // (columns > threads: in turns)
  constexpr int kU = 8;
  float4 x[kU];
  auto load = [&](int c0, int col) {
#pragma unroll
    for (int e = 0; e < kU; ++e) {
      const int c = min(c0 + e * shares, chunks - 1);
      x[e] = ld_dev4(r, ((unsigned)(c ? 2 * c : parts.odd) * a.state_stride + 2 * rows + 4 * col) * 4);
    }
  };
  int col = col0 + tid - share * columns;
  load(share, col);
  const int head = 4 * col0 / D, heads = (4 * (col0 + columns) - 1) / D + 1;  // of these columns
  for (int i = head + w; i < heads; i += kThreads / 64) {
    const float2 mz = join_sums(base, parts, a.state_stride, i, wt + i, rows);
    if ((tid & 63) == 0) {
      top[i] = mz.x;
      top[16 + i] = mz.y;
    }
  }
  __syncthreads();
  while (true) {
    const int g = 4 * col / D;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = share; share < shares && c0 < chunks;) {
#pragma unroll
      for (int e = 0; e < kU; ++e) {
        const int c = c0 + e * shares;
        if (c < chunks) {
          const float f = wt[c * rows + g];
          sum.x = fmaf(f, x[e].x, sum.x);
          sum.y = fmaf(f, x[e].y, sum.y);
          sum.z = fmaf(f, x[e].z, sum.z);
          sum.w = fmaf(f, x[e].w, sum.w);
        }
      }
      c0 += kU * shares;
      if (c0 < chunks) load(c0, col);
    }
    if (shares > 1) {  // (then all columns are in this turn)
      part[tid] = sum;
      __syncthreads();
      for (int k = 1; share == 0 && k < shares; ++k) {
        const float4 y = part[tid + k * columns];
        sum.x += y.x;
        sum.y += y.y;
        sum.z += y.z;
        sum.w += y.w;
      }
    }
    if (share == 0) {
      finish<DT, D>(a, head0, 4 * col, top[g], top[16 + g], sum.x);
      finish<DT, D>(a, head0, 4 * col + 1, top[g], top[16 + g], sum.y);
      finish<DT, D>(a, head0, 4 * col + 2, top[g], top[16 + g], sum.z);
      finish<DT, D>(a, head0, 4 * col + 3, top[g], top[16 + g], sum.w);
    }
    col += kThreads;
    if (shares > 1 || col >= col0 + columns) return;
    load(share, col);
  }
}

// Where a wave's tiles lie.  `ask` looks up the pages of the tile at t0, `move`
// makes it the tile that is loaded.
template <int DT, int D, bool kAligned>
struct Rows;

// Pages of whole 16-token blocks: a block's page is the same for all lanes, so it
// is looked up through the scalar cache, beside the vector loads' order, and read
// through a buffer resource of its own that ends with the last token: rows past
// the end come back as zeros, a block past the end is not read at all, and a lane
// has one fixed offset per row.
template <int DT, int D>
struct Rows<DT, D, true> {
  typedef Tile<DT, D> T;
  const PagedAttend& a;
  const char *k, *v;
  const int32_t* tab;
  unsigned k_lane, v_lane[4];
  int end;
  int token[T::kBlocks], page[T::kBlocks];
  __amdgpu_buffer_rsrc_t kr[T::kBlocks], vr[T::kBlocks];
  bool bad = false;
  __device__ __forceinline__ Rows(const PagedAttend& a, int b, int h, int end) : a(a), end(end) {
    const unsigned lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4, slot = a.slot_units << 4;
    k = reinterpret_cast<const char*>(a.k) + (size_t)h * a.head_bytes;
    v = reinterpret_cast<const char*>(a.v) + (size_t)h * a.head_bytes;
    tab = a.table + (size_t)b * a.max_pages;
    k_lane = j * slot + 16 * q;
#pragma unroll
    for (int r = 0; r < 4; ++r) v_lane[r] = (4 * q + r) * slot + j * T::kVStep;
  }
  __device__ __forceinline__ void ask(int t0) {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      token[i] = t0 + 16 * i;
      typedef const __attribute__((address_space(4))) int32_t* Uniform;
      page[i] = *(Uniform)(uint64_t)(tab + __builtin_amdgcn_readfirstlane(a.div.of(min(token[i], end - 1))));
    }
  }
  __device__ __forceinline__ void move() {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      const int rows = min(end - token[i], 16);
      bad |= rows > 0 && (unsigned)page[i] >= (unsigned)a.pages;
      const unsigned from = (unsigned)page[i] < (unsigned)a.pages ? (unsigned)page[i] : 0u;
      const size_t at = ((size_t)from * a.page_units +
                         (unsigned)(token[i] - a.div.of(token[i]) * a.page_size) * a.slot_units) << 4;
      const int bytes = rows > 0 ? (int)((rows - 1) * (a.slot_units << 4)) + D * kElem<DT> : 0;
      kr[i] = raw_buffer(k + at, bytes);
      vr[i] = raw_buffer(v + at, bytes);
    }
  }
  __device__ __forceinline__ void load_k(T& t) const {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int c = 0; c < T::kKLoads; ++c) t.k[i][c] = load_nt16_buf(kr[i], k_lane + 64 * c);
  }
  __device__ __forceinline__ void load_v(T& t) const {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) load_words_buf(t.v[i][r], vr[i], v_lane[r]);
  }
};

// Any page size: each lane looks up the rows that it loads keys of, and takes the
// values' rows from the lanes that have them.  Tokens past the end repeat the last.
template <int DT, int D>
struct Rows<DT, D, false> {
  typedef Tile<DT, D> T;
  const PagedAttend& a;
  const char *k, *v;
  const int32_t* tab;
  int end, token[T::kBlocks], page[T::kBlocks];
  unsigned row[T::kBlocks];  // 16-byte units
  bool bad = false;
  __device__ __forceinline__ Rows(const PagedAttend& a, int b, int h, int end) : a(a), end(end) {
    const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
    k = reinterpret_cast<const char*>(a.k) + (size_t)h * a.head_bytes + 16 * q;
    v = reinterpret_cast<const char*>(a.v) + (size_t)h * a.head_bytes + j * T::kVStep;
    tab = a.table + (size_t)b * a.max_pages;
  }
  __device__ __forceinline__ void ask(int t0) {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      token[i] = min(t0 + 16 * i + (int)(threadIdx.x & 15), end - 1);
      page[i] = tab[a.div.of(token[i])];
    }
  }
  __device__ __forceinline__ void move() {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      if ((unsigned)page[i] >= (unsigned)a.pages) {
        bad = true;
        page[i] = 0;
      }
      row[i] = (unsigned)page[i] * a.page_units +
               (unsigned)(token[i] - a.div.of(token[i]) * a.page_size) * a.slot_units;
    }
  }
  __device__ __forceinline__ void load_k(T& t) const {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int c = 0; c < T::kKLoads; ++c) t.k[i][c] = load_nt16(k + ((size_t)row[i] << 4) + 64 * c);
  }
  __device__ __forceinline__ void load_v(T& t) const {
    const int q = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) load_words(t.v[i][r], v + ((size_t)(unsigned)__shfl((int)row[i], 4 * q + r) << 4));
  }
};

// `count` quanta of one pair from its quantum u.first on: this workgroup's state
// of them, and the pair's output if it is the only or the last to come.
template <int DT, int D, bool kAligned, bool kMany>
__device__ __forceinline__ void attend_segment(const PagedAttend& a, const PagedSpan<kLeast<DT, D>>& u, int quanta, int count, float* lds) {
  typedef Tile<DT, D> T;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, q = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = u.hh / a.tiles, g0 = 16 * (u.hh - h * a.tiles);
  const int rows = min(a.group - g0, 16);  // query heads of this tile
  const int start = min(u.first * kQuantum, u.n), end = min(start + count * kQuantum, u.n);
  // (a pair alone: all tiles are this wave's)
  const bool alone = kMany && u.alone;
  const int step = alone ? T::kTokens : kAWaves<D> * T::kTokens;

  // Q^T: column j is head j (zero past the tile's heads)
  u32x4 qop[T::kKLoads];
  {
    const char* qp = reinterpret_cast<const char*>(a.q) +
                     (((size_t)u.b * a.kv_heads + h) * a.group + g0 + min(j, rows - 1)) * (D * kElem<DT>) + 16 * q;
#pragma unroll
    for (int c = 0; c < T::kKLoads; ++c) {
      const uint4 x = *reinterpret_cast<const uint4*>(qp + 64 * c);
      qop[c] = j < rows ? u32x4{x.x, x.y, x.z, x.w} : u32x4{0u, 0u, 0u, 0u};
    }
  }
  f32x4 acc[D / 16];
#pragma unroll
  for (int n = 0; n < D / 16; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, z = 0.f;  // head j's running maximum (exp2 domain), this lane's share of its sum

  float* logits = a.logits ? a.logits + (((size_t)u.b * a.kv_heads + h) * a.group + g0 + j) * a.logit_stride : nullptr;
  Rows<DT, D, kAligned> rows_of(a, u.b, h, end);

  // Loads run ahead without registers of their own: the next tile's keys are
  // requested as soon as this one's are used up by the scores, its values after
  // the products with this one's, and the pages of the tile after that in
  // between (memory answers in order: whatever is waited for was asked first).
  int t0 = start + (alone ? 0 : T::kTokens * w);
  T t;
  if (t0 < end) {
    rows_of.ask(t0);
    rows_of.move();
    rows_of.load_k(t);
    rows_of.ask(t0 + step);
    rows_of.load_v(t);
  }
  // (the loads of the tile behind the last are issued too: on every path as many
  // are in flight, so that the compiler's wait counts are exact)
  for (; t0 < end; t0 += step) {
    // scores: lane (j, q) gets tokens 16i + 4q + r of head j
    float s[T::kBlocks][4];
    float bm = -INFINITY;
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
      f32x4 d = {0.f, 0.f, 0.f, 0.f}, d2 = d;  // (fp32: two shorter chains, whose rounding errors are smaller)
#pragma unroll
      for (int c = 0; c < T::kKLoads; ++c) {
        const u32x4 kw = {t.k[i][c].x, t.k[i][c].y, t.k[i][c].z, t.k[i][c].w};
        const u32x4 qw = qop[c];
        if constexpr (DT == kFp32) {
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            d = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[e]), __uint_as_float(qw[e]), d, 0, 0, 0);
            d2 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[e + 1]), __uint_as_float(qw[e + 1]), d2, 0, 0,
                                                      0);
          }
        } else {
          d = mfma32<DT>(kw, qw, d);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[i][r] = DT == kFp32 ? d[r] + d2[r] : d[r];
        bm = fmaxf(bm, t0 + 16 * i + 4 * q + r < end ? s[i][r] * a.scale : -INFINITY);
      }
    }
    rows_of.move();
    rows_of.load_k(t);
    rows_of.ask(t0 + 2 * step);
    bm = fmaxf(bm, xor16(bm));
    bm = fmaxf(bm, xor32(bm));
    if (__ballot(bm > m)) {
      const float nm = fmaxf(m, bm);
      const float alpha = m == nm ? 1.f : exp2_or_zero(m - nm);
      m = nm;
      z *= alpha;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float ah = __shfl(alpha, 4 * q + r);
#pragma unroll
        for (int n = 0; n < D / 16; ++n) acc[n][r] *= ah;
      }
    }
    const float top = no_less(m);
    float p[T::kBlocks][4];
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[i][r] = weight(s[i][r], a.scale, top);
        if (t0 + 16 * i + 4 * q + r >= end) p[i][r] = 0.f;
        if constexpr (kBias<DT> != 0) p[i][r] = ldexpf(p[i][r], kBias<DT>);
        z += p[i][r];
      }
    if (!kAligned && t0 + T::kTokens > end) {  // rows past the end repeat the last one: 0 times its infinity must not be added
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t0 + 16 * i + 4 * q + r >= end) {
#pragma unroll
            for (int n = 0; n < T::kVWords; ++n) t.v[i][r][n] = 0u;
          }
    }
    if constexpr (DT == kFp32) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[0][r], __uint_as_float(t.v[0][r][n]), acc[n], 0, 0, 0);
    } else {
      unsigned term[8][kTerms<DT>];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) split16<DT>(p[i][r], term[4 * i + r]);
      u32x4 pw[kTerms<DT>];
#pragma unroll
      for (int k = 0; k < kTerms<DT>; ++k)
        pw[k] = u32x4{upper16(term[0][k], term[1][k]), upper16(term[2][k], term[3][k]), upper16(term[4][k], term[5][k]),
                      upper16(term[6][k], term[7][k])};
      pv_columns<0, DT, D>(acc, t, pw);
    }
    rows_of.load_v(t);
    // behind the loads: memory answers stores in the same order, and what the next
    // step waits for must not be behind them (16 sequences of 4099: 47.5 us before)
    if (logits && j < rows) {
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i)
        *reinterpret_cast<float4*>(logits + t0 + 16 * i + 4 * q) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    }
  }
  if (__ballot(rows_of.bad) && lane == 0) report_error(a.err, error_host_slot(a.err), kErrPages);

  z += xor16(z);
  z += xor32(z);
  const size_t head0 = ((size_t)u.b * a.kv_heads + h) * a.group + g0;  // this tile's first query head
  if (alone) {  // lane (j, q) has dims dim(n, j) of heads 4q + r
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float M = __shfl(m, 4 * q + r), den = __shfl(z, 4 * q + r);
      if (4 * q + r < rows) {
#pragma unroll
        for (int n = 0; n < D / 16; ++n) finish<DT, D>(a, head0, (4 * q + r) * D + T::dim(n, j), M, den, acc[n][r]);
      }
    }
    return;
  }
  // the waves' states meet in LDS
  float* sm = lds;  // [waves][16] maxima
  float* sz = sm + 16 * kAWaves<D>;   // [waves][16] sums
  float* sacc = sz + 16 * kAWaves<D>; // [waves][rows][D]
  if (lane < 16) {
    sm[16 * w + j] = m;
    sz[16 * w + j] = z;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (4 * q + r < rows) {
      float* dst = sacc + ((size_t)w * rows + 4 * q + r) * D;
#pragma unroll
      for (int n = 0; n < D / 16; n += 4)  // (a piece is 4 or 8 elements)
        *reinterpret_cast<float4*>(dst + T::dim(n, j)) = make_float4(acc[n][r], acc[n + 1][r], acc[n + 2][r], acc[n + 3][r]);
    }
  __syncthreads();
  const int pair0 = u.at - u.first, unit = (int)blockIdx.x;
  const bool whole = count == quanta;
  float* state = a.state + (size_t)(2 * unit + (u.at != u.deal.begin(unit))) * a.state_stride;  // {max, sum}[rows], [rows][D]
  for (int i = 2 * tid; i < rows * D; i += 128 * kAWaves<D>) {
    const int g = i / D;
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < kAWaves<D>; ++k) M = fmaxf(M, sm[16 * k + g]);
    float den = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int k = 0; k < kAWaves<D>; ++k) {
      const float wt = rescale(sm[16 * k + g], M);
      const float2 v = *reinterpret_cast<const float2*>(sacc + (size_t)k * rows * D + i);
      den = fmaf(wt, sz[16 * k + g], den);
      x = fmaf(wt, v.x, x);
      y = fmaf(wt, v.y, y);
    }
    if (whole) {
      finish<DT, D>(a, head0, i, M, den, x);
      finish<DT, D>(a, head0, i + 1, M, den, y);
    } else {
      if (i % D == 0) st_dev2(state + 2 * g, M, den);
      st_dev2(state + 2 * rows + i, x, y);
    }
  }
  if (whole || !a.counters) return;

  // the last workgroup of the pair joins the states
  const PagedParts parts(u.deal, pair0, quanta);
  int* last = reinterpret_cast<int*>(lds);
  drain();
  __syncthreads();
  unsigned* counter = a.counters + (size_t)u.b * a.kv_heads * a.tiles + u.hh;
  if (tid == 0) *last = inc_dev(counter) == (unsigned)(parts.chunks - 1);
  __syncthreads();
  const int is_last = *last;
  __syncthreads();
  if (!is_last) return;
  if (tid == 0) st_dev(counter, 0u);
  join_states<DT, D, 64 * kAWaves<D>>(a, head0, rows, parts, 0, rows * D / 4, lds);
}

template <int DT, int D, bool kAligned, bool kMany>
__global__ __launch_bounds__(64 * kAWaves<D>, kAWaves<D> / 4) void paged_attend_kernel(PagedAttend a) {
  extern __shared__ float lds[];
  constexpr int kL = kLeast<DT, D>;
  PagedSpan<kL> u = find_span<kL, kMany>(a, blockIdx.x);
  if constexpr (kMany) {
    if (u.alone) {
      const int heads = a.kv_heads * a.tiles;
      u.first = 0;
      for (int pair = blockIdx.x + gridDim.x * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); pair < a.sequences * heads;
           pair += gridDim.x * kAWaves<D>) {
        u.b = pair / heads;
        u.hh = pair - u.b * heads;
        u.n = __builtin_amdgcn_readfirstlane(clamp_length(a, a.lengths[u.b]));
        const int quanta = quanta_of<kL>(u.n);
        attend_segment<DT, D, kAligned, kMany>(a, u, quanta, quanta, lds);
      }
      return;
    }
  }
  while (u.at < u.end) {  // the pairs that this workgroup's share lies in
    const int quanta = quanta_of<kL>(u.n);
    const int count = min(quanta - u.first, u.end - u.at);
    attend_segment<DT, D, kAligned, kMany>(a, u, quanta, count, lds);
    u.at += count;
    u.first = 0;
    if (++u.hh == a.kv_heads * a.tiles) {
      u.hh = 0;
      u.n = ++u.b < a.sequences ? clamp_length(a, a.lengths[u.b]) : 0;
    }
    __syncthreads();  // the next pair's states go where these were
  }
}

// Joins in a launch of their own: the states of a pair that are many and wide, over
// several workgroups, kJoinColumns columns each.
constexpr int kJoinColumns = 16;

template <int DT, int D>
__global__ __launch_bounds__(kPT) void paged_join_kernel(PagedAttend a) {
  extern __shared__ float lds[];
  const int b = blockIdx.z;
  const int h = blockIdx.y / a.tiles, tile = blockIdx.y - h * a.tiles;
  const int rows = min(a.group - 16 * tile, 16), col0 = blockIdx.x * kJoinColumns;
  if (col0 >= rows * D / 4) return;
  constexpr int kL = kLeast<DT, D>;
  int longest = 0;
  const PagedDeal<kL> deal{quanta_before<kL>(a, a.sequences, longest) * a.kv_heads * a.tiles};
  if (pairs_alone(a, longest)) return;
  const int from = quanta_before<kL>(a, b, longest), n = __builtin_amdgcn_readfirstlane(clamp_length(a, a.lengths[b]));
  const int quanta = quanta_of<kL>(n);
  const PagedParts parts(deal, from * a.kv_heads * a.tiles + (int)blockIdx.y * quanta, quanta);
  if (parts.chunks == 1) return;  // its workgroup has finished it
  join_states<DT, D, kPT>(a, ((size_t)b * a.kv_heads + h) * a.group + 16 * tile, rows, parts, col0, kJoinColumns, lds);
}

// scores_out[t] = scores[t] + sum over the group's heads of its weight, from their
// maxima and sums as the attention had them (a log-sum's rounding, 2^-24 of it, would
// be the weights' error: 4e-4 at scores of 2e4): a thread per slot; bound by the scores that it reads (4 bytes per query head and
// slot) and the two score arrays.
__global__ __launch_bounds__(kPT) void paged_weigh_kernel(PagedAttend a) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int n = clamp_length(a, a.lengths[b]);
  const float2* sums = a.sums_work + ((size_t)b * a.kv_heads + h) * a.group;
  const float* logits = a.logits + ((size_t)b * a.kv_heads + h) * a.group * a.logit_stride;
  const size_t at = ((size_t)b * a.kv_heads + h) * a.slots;
  for (int t = blockIdx.x * kPT + threadIdx.x; t < n; t += gridDim.x * kPT) {
    const float before = a.scores[at + t];
    float sum = 0.f;
    for (int g0 = 0; g0 < a.group; g0 += 4) {  // (four heads' loads together)
      float s[4];
      float2 z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int g = min(g0 + e, a.group - 1);
        s[e] = logits[(size_t)g * a.logit_stride + t];
        z[e] = sums[g];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (g0 + e < a.group) sum = fmaf(weight(s[e], a.scale, z[e].x), z[e].y, sum);
    }
    a.scores_out[at + t] = before + sum;
  }
}

// ------------------------------------------------------------------ append
//
// A copy of rows: bound by reading and writing them.  A workgroup finds the places
// of its rows (one of a sequence each, or kAppendRows packed ones) with a thread
// per row, then copies them with 16 bytes per thread, kU loads each of K and V in
// flight.  20011 rows of 8 heads and 128 dims in bf16 (164 MB read and written):
// 31.7 us = 5.2 TB/s (a copy as large: 32.2); 128 single rows 3.5 us.

constexpr int kAppendRows = 8;
constexpr int64_t kLaunchRows = 1 << 26;  // (a launch has fewer than 2^32 threads: 2^27 rows)

struct AppendPlace {
  size_t at;  // bytes from the pages' base
  int b, slot, position, length;  // slot -1: a row that is dropped; length: of its sequence before
};

__device__ __forceinline__ AppendPlace append_place(const PagedAppend& a, int64_t row) {
  AppendPlace p{0, 0, -1, 0, 0};
  int64_t step = 0;
  if (!a.offsets) {
    p.b = (int)row;
  } else {  // the last b with offsets[b] <= row
    int lo = 0, hi = a.sequences;
    while (lo + 1 < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.offsets[mid] <= row) lo = mid;
      else hi = mid;
    }
    p.b = lo;
    step = row - a.offsets[lo];
    if (step < 0 || row >= a.offsets[lo + 1]) return p;  // a row of no sequence
  }
  p.length = min(max(a.lengths[p.b], 0), a.slots);
  if (a.positions) p.position = a.seen[p.b] + (int)step;
  const int64_t slot = p.length + step;
  const int page = slot < a.slots ? a.table[(size_t)p.b * a.max_pages + a.div.of((int)slot)] : -1;
  if ((unsigned)page >= (unsigned)a.pages) {  // no page: the row is dropped
    report_error(a.err, error_host_slot(a.err), kErrPages);
    return p;
  }
  p.slot = (int)slot;
  p.at = (size_t)page * a.page_bytes + (size_t)(p.slot - a.div.of(p.slot) * a.page_size) * a.slot_bytes;
  return p;
}

// lengths and tokens seen of sequence b with its packed rows; offsets that do not
// cover the rows, ascending from 0, are reported
__device__ __forceinline__ void advance(const PagedAppend& a, int b) {
  const int from = a.offsets[b], to = a.offsets[b + 1], more = max(to - from, 0);
  if (from > to || (b == 0 && from) || (b == a.sequences - 1 && to != a.rows))
    report_error(a.err, error_host_slot(a.err), kErrRows);
  a.lengths_out[b] = (int)min((int64_t)max(a.lengths[b], 0) + more, (int64_t)a.slots);
  if (a.positions) a.seen_out[b] = a.seen[b] + more;
}

__global__ __launch_bounds__(kPT) void paged_append_kernel(PagedAppend a) {
  __shared__ AppendPlace places[kAppendRows];
  const int tid = threadIdx.x, each = a.offsets ? kAppendRows : 1;
  const int64_t row0 = a.first_row + (int64_t)blockIdx.x * each;
  const int rows = (int)min((int64_t)each, a.rows - row0);
  const int log = a.log_pieces, per_row = a.kv_heads << log, items = rows * per_row;  // pieces of 16 bytes
  constexpr int kU = 4;
  uint4 kv[kU], vv[kU];
  // piece i: its row, and its bytes from the row's first
  auto piece = [&](int i, int& r, int& h, int& c) {
    r = i / per_row;
    h = (i - r * per_row) >> log;
    c = (i & ((1 << log) - 1)) << 4;
  };
  auto load = [&](int i0) {
#pragma unroll
    for (int e = 0; e < kU; ++e) {
      if (i0 - tid + e * kPT >= items) break;
      int r, h, c;
      piece(min(i0 + e * kPT, items - 1), r, h, c);
      kv[e] = load_nt16(a.k + (row0 + r) * a.k_row + (int64_t)h * a.k_head + c);
      vv[e] = load_nt16(a.v + (row0 + r) * a.v_row + (int64_t)h * a.v_head + c);
    }
    asm volatile("" ::: "memory");  // (all of them are asked for before anything is stored)
  };
  load(tid);
  if (tid < rows) places[tid] = append_place(a, row0 + tid);
  __syncthreads();
  for (int i0 = tid; i0 < items;) {
#pragma unroll
    for (int e = 0; e < kU; ++e) {
      if (i0 + e * kPT >= items) break;
      int r, h, c;
      piece(i0 + e * kPT, r, h, c);
      const AppendPlace& p = places[r];
      if (p.slot >= 0) {
        const size_t at = p.at + (size_t)h * a.head_bytes + c;
        *reinterpret_cast<uint4*>(a.kp + at) = kv[e];
        *reinterpret_cast<uint4*>(a.vp + at) = vv[e];
      }
    }
    i0 += kU * kPT;
    if (i0 < items) load(i0);
  }
  if (a.positions)
    for (int i = tid; i < rows * a.kv_heads; i += kPT) {
      const AppendPlace& p = places[i / a.kv_heads];
      if (p.slot < 0) continue;
      const size_t at = ((size_t)p.b * a.kv_heads + i % a.kv_heads) * a.slots + p.slot;
      a.scores[at] = a.scores_out[at] = 0.f;
      a.positions[at] = a.positions_out[at] = p.position;
    }
  if (!a.offsets) {  // (the row's workgroup alone reads its sequence's length)
    if (tid == 0) {
      a.lengths_out[blockIdx.x] = min(places[0].length + 1, a.slots);
      if (a.positions) a.seen_out[blockIdx.x] = places[0].position + 1;
    }
  } else if (a.lengths_out != a.lengths) {
    for (int64_t b = (int64_t)blockIdx.x * kPT + tid; b < a.sequences; b += (int64_t)gridDim.x * kPT)
      advance(a, (int)b);
  }
}

// Packed rows onto lengths that are advanced in place: after every workgroup has read them.
__global__ __launch_bounds__(kPT) void paged_advance_kernel(PagedAppend a) {
  const int b = blockIdx.x * kPT + threadIdx.x;
  if (b < a.sequences) advance(a, b);
}

// ------------------------------------------------------------------ eviction

// The order of the scores as an unsigned key: NaN above the numbers, -0 as 0; above
// them all 0xffffffff, a protected slot's.
__device__ __forceinline__ unsigned evict_key(float score) {
  const unsigned u = __float_as_uint(score + 0.f);
  const unsigned key = u ^ (unsigned)((int)u >> 31 | (int)0x80000000);
  return score != score ? 0xfffffffeu : key;
}

__device__ __forceinline__ int evict_keep(const PagedEvict& a, int b) {
  const int keep = a.keeps ? a.keeps[b] : a.keep;
  return max(keep, 0);
}

constexpr int kET = 1024, kEWaves = kET / 64;  // threads and waves of the selection
constexpr int kFew = 256;                      // moves that the selection makes by itself

struct EvictRow {
  int n, m, edge;  // length, slots that stay, first position that is among the newest
  size_t row;
  const float* scores;
  const int32_t* positions;
  bool copy;  // the fork gets what stays where it is (the moves overwrite the holes)
  // sizes: {n, m} where the sequence's length may be written meanwhile
  __device__ __forceinline__ EvictRow(const PagedEvict& a, int b, int h, const unsigned* sizes = nullptr) {
    n = __builtin_amdgcn_readfirstlane(sizes ? (int)sizes[0] : min(max(a.lengths[b], 0), a.slots));
    m = __builtin_amdgcn_readfirstlane(sizes ? (int)sizes[1] : min(n, evict_keep(a, b)));
    edge = max(a.seen[b] - a.recent, a.sinks);
    row = (size_t)b * a.kv_heads + h;
    scores = a.scores + row * a.slots;
    positions = a.positions + row * a.slots;
    copy = a.scores_out != a.scores;
  }
};

// Scores and positions of kU x 64 slots from t0 on, asked for together; then their
// keys, 0 at and behind `last`.
template <int kU>
struct EvictSlots {
  float score[kU];
  int position[kU];
  __device__ __forceinline__ void load(const EvictRow& r, int t0) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int t = min(t0 + 64 * u + lane, r.n - 1);
      score[u] = r.scores[t];
      position[u] = r.positions[t];
    }
    asm volatile("" ::: "memory");
  }
  __device__ __forceinline__ void keys(const PagedEvict& a, const EvictRow& r, int t0, int last, bool copy,
                                       unsigned (&key)[kU]) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int t = t0 + 64 * u + lane;
      // (position < sinks or >= edge as one comparison, edge >= sinks)
      const bool held = (unsigned)(position[u] - a.sinks) >= (unsigned)(r.edge - a.sinks);
      key[u] = t >= last ? 0u : held ? 0xffffffffu : evict_key(score[u]);
      if (copy && t < min(last, r.m)) {
        a.scores_out[r.row * a.slots + t] = score[u];
        a.positions_out[r.row * a.slots + t] = position[u];
      }
    }
  }
};

// The digits of a key from the top.  (No key has the first digit 0, where slots
// that are none are counted.)
template <int kPass>
__device__ __forceinline__ unsigned digit(unsigned key) {
  return kPass == 0 ? key >> 21 : kPass == 1 ? (key >> 10) & 2047u : key & 1023u;
}
// Whether the digits before this pass's are those found, `prefix`.
template <int kPass>
__device__ __forceinline__ bool matches(unsigned key, unsigned prefix) {
  return kPass == 0 || (kPass == 1 ? key >> 21 : key >> 10) == prefix;
}

// The digit of the need-th largest key, given the counts of digits 2047 - 2i (x) and
// 2046 - 2i (y) in thread i: appended to `prefix`, and `need` among its keys.
template <int kPass>
__device__ __forceinline__ void find_digit(unsigned x, unsigned y, unsigned* wsum, unsigned* found, unsigned& prefix,
                                           unsigned& need) {
  const int tid = threadIdx.x;
  const unsigned before = block_incl_scan<kET>(x + y, wsum) - x - y;
  if (before < need && need <= before + x + y) {
    const bool upper = need <= before + x;
    found[0] = 2047 - 2 * tid - !upper;
    found[1] = need - before - (upper ? 0u : x);
  }
  __syncthreads();
  prefix = prefix << (kPass < 2 ? 11 : 10) | __builtin_amdgcn_readfirstlane(found[0]);
  need = __builtin_amdgcn_readfirstlane(found[1]);
}

// Lanes of 64 slots from t0 that lie before slot m.
__device__ __forceinline__ unsigned long long lanes_before(int m, int t0) {
  const int n = m - t0;
  return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull;
}

// Counts of a share of the slots: evicted before the budget and kept behind it if no
// key equal to the bound stays, and such keys before and behind it.
struct EvictCounts {
  int hole, source, front, back;
  // the holes and sources where `room` of the keys equal to the bound stay, the lowest
  __device__ __forceinline__ int holes(int room) const { return hole - min(max(room, 0), front); }
  __device__ __forceinline__ int sources(int room) const { return source + min(max(room - front, 0), back); }
};

// The counts of the wave's share given by each_key (f(t0, key): 64 slots from t0,
// ascending).
template <typename E>
__device__ __forceinline__ EvictCounts count_moves(E each_key, unsigned bound, int m, int last) {
  EvictCounts c{0, 0, 0, 0};
  each_key([&](int t0, unsigned key) {
    const unsigned long long above = __ballot(key > bound), eq = __ballot(key == bound), front = lanes_before(m, t0);
    c.hole += __popcll(~above & front & lanes_before(last, t0));
    c.source += __popcll(above & ~front);
    c.front += __popcll(eq & front);
    c.back += __popcll(eq & ~front);
  });
  return c;
}

// Appends the slots t0 + (lanes of mask), ascending.
__device__ __forceinline__ void put_slots(int32_t*& to, int t0, unsigned long long mask) {
  if (!mask) return;
  const int lane = threadIdx.x & 63;
  if (mask >> lane & 1)
    to[__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u))] = t0 + lane;
  to += __popcll(mask);
}

// Sum over the workgroup, in every thread.
__device__ __forceinline__ int block_sum(int v, int* lds) {
  v = wave_sum_i(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int k = 0; k < kEWaves; ++k) total += lds[k];
  return __builtin_amdgcn_readfirstlane(total);
}

// Writes the wave's holes and sources (each_key as above, its counts `mine`) behind
// those of the waves before it, to dst and src, which begin with the workgroup's;
// `room` of the workgroup's keys equal to the bound stay.  Returns the workgroup's
// number of holes; where it is `few` at most they go to few_dst and few_src.
template <typename E>
__device__ __forceinline__ int write_moves(E each_key, const EvictCounts& mine, unsigned bound, int room, int m, int last,
                                           int32_t* dst, int32_t* src, EvictCounts* counts, int few, int32_t* few_dst,
                                           int32_t* few_src) {
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((threadIdx.x & 63) == 0) counts[w] = mine;
  __syncthreads();
  int hole = 0, source = 0, total = 0, own = 0, left = room;  // room left for the wave's own
#pragma unroll
  for (int k = 0; k < kEWaves; ++k) {
    const EvictCounts c = counts[k];
    if (k == w) own = left;
    const int holes = c.holes(left);
    hole += k < w ? holes : 0;
    source += k < w ? c.sources(left) : 0;
    total += holes;
    left -= c.front + c.back;
  }
  total = __builtin_amdgcn_readfirstlane(total);
  own = __builtin_amdgcn_readfirstlane(own);
  dst = (total <= few ? few_dst : dst) + __builtin_amdgcn_readfirstlane(hole);
  src = (total <= few ? few_src : src) + __builtin_amdgcn_readfirstlane(source);
  each_key([&](int t0, unsigned key) {
    unsigned long long kept = __ballot(key > bound);
    const unsigned long long eq = __ballot(key == bound), front = lanes_before(m, t0);
    if (eq) {
      const int at = (int)__builtin_amdgcn_mbcnt_hi((unsigned)(eq >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)eq, 0u));
      kept |= eq & __ballot(at < own);
      own -= __popcll(eq);
    }
    put_slots(dst, t0, ~kept & front & lanes_before(last, t0));
    put_slots(src, t0, kept & ~front);
  });
  return total;
}

// A move's rows of K and V, kRows of them in flight per thread; a row takes as many
// lanes as it has 16-byte pieces.  Slots in srcs and dsts (`count` of them), this
// workgroup's from its index on, every groups-th kRows * rows-at-a-time of them.
template <int kThreads, int kRows>
__device__ __forceinline__ void move_rows(const PagedEvict& a, int b, int h, size_t row, const int32_t* srcs,
                                          const int32_t* dsts, int count, int group, int groups) {
  const int c = (threadIdx.x & ((1 << a.log_pieces) - 1)) << 4, step = kThreads >> a.log_pieces;
  const int32_t* tab = a.table + (size_t)b * a.max_pages;
  for (int k1 = group * step * kRows; k1 < count; k1 += groups * step * kRows) {
    const int k0 = k1 + (threadIdx.x >> a.log_pieces);
    int src[kRows], dst[kRows];
    size_t to[kRows];
    bool in[kRows];
    uint4 kv[kRows], vv[kRows];
#pragma unroll
    for (int e = 0; e < kRows; ++e) {
      if (k1 + e * step >= count) break;
      const int k = min(k0 + e * step, count - 1);
      src[e] = srcs[k];
      dst[e] = dsts[k];
      in[e] = k0 + e * step < count;
    }
#pragma unroll
    for (int e = 0; e < kRows; ++e) {
      if (k1 + e * step >= count) break;
      const int ps = a.div.of(src[e]), pd = a.div.of(dst[e]);
      int from = tab[ps], into = tab[pd];
      if ((unsigned)from >= (unsigned)a.pages || (unsigned)into >= (unsigned)a.pages) {
        if (in[e]) report_error(a.err, error_host_slot(a.err), kErrPages);
        in[e] = false;
        from = into = 0;
      }
      const size_t f = (size_t)from * a.page_bytes + (size_t)(src[e] - ps * a.page_size) * a.slot_bytes +
                       (size_t)h * a.head_bytes + c;
      to[e] = (size_t)into * a.page_bytes + (size_t)(dst[e] - pd * a.page_size) * a.slot_bytes +
              (size_t)h * a.head_bytes + c;
      kv[e] = load_nt16(a.kp + f);
      vv[e] = load_nt16(a.vp + f);
    }
    asm volatile("" ::: "memory");  // (all of them are asked for before anything is stored)
#pragma unroll
    for (int e = 0; e < kRows; ++e)
      if (k1 + e * step < count && in[e]) {
        *reinterpret_cast<uint4*>(a.kp + to[e]) = kv[e];
        *reinterpret_cast<uint4*>(a.vp + to[e]) = vv[e];
        if (c == 0) {
          a.scores_out[row * a.slots + dst[e]] = a.scores[row * a.slots + src[e]];
          a.positions_out[row * a.slots + dst[e]] = a.positions[row * a.slots + src[e]];
        }
      }
  }
}

// The sequence's new length and tokens seen, by the last of its workgroups to come;
// called behind a barrier, when all threads have read the old ones, and late, by
// the last wave, which others need not wait for.
__device__ __forceinline__ void evict_lengths(const PagedEvict& a, const EvictRow& r, int b, int workgroups) {
  if (threadIdx.x != kET - 1) return;
  if (inc_dev(&a.counters[b]) != (unsigned)(workgroups - 1)) return;
  st_dev(&a.counters[b], 0u);
  a.lengths_out[b] = r.m;
  if (a.seen_out != a.seen) a.seen_out[b] = a.seen[b];
}

// One workgroup per (sequence, KV head), rows of up to kLongRow slots: the keys in
// LDS, the budget-th largest by three histogram passes (11, 11 and 10 bits), then
// the slots that move, found by each wave in its own share, and, if they are few,
// their rows.  Bound by the latency of its steps and, its 16 waves on one CU, the
// instructions of each 64 slots: 2112 slots to 2048, 8 x 8 rows, 11.5 us, of which by
// clock reads the reads and the first counts 1.4, the passes 2.4, counts and lists of
// the moves 3.0, the moves 1.8; up to 9001 slots, 16 x 4 rows, 15 traced.
// Up to this many slots; twice as many where the rows fill the CUs by themselves (31
// steps of 64 slots a wave: one row of 32000 slots 45 us, 43 in parts; 64 rows 59,
// 75 in parts).
constexpr int kLongRow = 16384, kManyRows = 64;

__global__ __launch_bounds__(kET) void paged_select_kernel(PagedEvict a) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  __shared__ unsigned hist[3][2048], wsum[kEWaves], found[3][2];
  __shared__ EvictCounts counts[kEWaves];
  __shared__ int32_t few[2][kFew];
  extern __shared__ unsigned keys[];  // of whole 64-slot steps
  for (int i = tid; i < 3 * 2048; i += kET) (&hist[0][0])[i] = 0u;
  const EvictRow r(a, b, h);
  asm volatile("" ::"s"(r.n), "s"(r.m));  // (read, not only asked for, before others may write the length)
  __syncthreads();
  const bool cut = r.n > r.m && r.m > 0;
  const int steps = (r.n + 64 * kEWaves - 1) / (64 * kEWaves);  // of 64 slots per wave
  const int first = min(64 * steps * w, r.n), last = min(first + 64 * steps, r.n);
  constexpr int kU = 4;
  for (int t0 = first; t0 < last; t0 += kU * 64) {
    EvictSlots<kU> slots;
    unsigned k[kU];
    slots.load(r, t0);
    slots.keys(a, r, t0, last, r.copy, k);
    if (!cut) continue;
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (t0 + 64 * u < last) {
        keys[t0 + 64 * u + lane] = k[u];
        atomicAdd(&hist[0][digit<0>(k[u])], 1u);
      }
  }
  if (!cut) {
    if (tid == 0) a.count[r.row] = 0;
    evict_lengths(a, r, b, a.kv_heads);
    return;
  }
  auto each_key = [&](auto f) {  // (a wave reads what it wrote itself)
#pragma unroll 1
    for (int t0 = first; t0 < last; t0 += 64) f(t0, keys[t0 + lane]);
  };
  __syncthreads();
  unsigned bound = 0, need = r.m;
  find_digit<0>(hist[0][2047 - 2 * tid], hist[0][2046 - 2 * tid], wsum, found[0], bound, need);
  each_key([&](int, unsigned key) {
    if (matches<1>(key, bound)) atomicAdd(&hist[1][digit<1>(key)], 1u);
  });
  __syncthreads();
  find_digit<1>(hist[1][2047 - 2 * tid], hist[1][2046 - 2 * tid], wsum, found[1], bound, need);
  each_key([&](int, unsigned key) {
    if (matches<2>(key, bound)) atomicAdd(&hist[2][digit<2>(key)], 1u);
  });
  __syncthreads();
  find_digit<2>(hist[2][2047 - 2 * tid], hist[2][2046 - 2 * tid], wsum, found[2], bound, need);
  const EvictCounts mine = count_moves(each_key, bound, r.m, last);
  const int total = write_moves(each_key, mine, bound, (int)need, r.m, last, a.dst + r.row * a.moves,
                                a.src + r.row * a.moves, counts, kFew, few[1], few[0]);
  if (tid == 0) a.count[r.row] = total <= kFew ? 0 : total;
  if (total <= kFew) __syncthreads();  // (the fork's copies of what stays come before the moves')
  evict_lengths(a, r, b, a.kv_heads);
  if (total <= kFew) move_rows<kET, 4>(a, b, h, r.row, few[0], few[1], total, 0, 1);
}

// Longer rows take one launch per pass, a part of a row per workgroup: a.part slots,
// kPart or, so that no row has more than kMostParts and a few, a multiple of it.
// The slots before the budget and those behind it have parts of their own.  Each
// workgroup leaves its counts of the digits, from which all of the next launch find
// theirs.  65536 slots, 8 rows: 6 + 7 + 7 + 15 us; one workgroup for each row 60.
constexpr int kPart = 8192, kPartKeys = kPart / kET, kMostParts = 128;

struct EvictPart {
  int part, first, last, front, parts;  // slots; parts before the budget, parts
  __device__ __forceinline__ EvictPart(const PagedEvict& a, const EvictRow& r, int x) : part(a.part) {
    front = (r.m + part - 1) / part;
    parts = front + (r.n - r.m + part - 1) / part;
    first = x < front ? x * part : r.m + (x - front) * part;
    last = min(first + part, x < front ? r.m : r.n);
  }
  // slots of part y (before the budget)
  __device__ __forceinline__ int size(const EvictRow& r, int y) const { return min(part, r.m - y * part); }
};

// The keys of a wave's share of a part: kept in LDS where the part is kPart slots,
// read again by every pass over them where it is longer.
struct EvictKeys {
  const PagedEvict& a;
  const EvictRow& r;
  int first, last;
  bool copy;
  EvictSlots<kPartKeys> slots;
  unsigned* lds;  // [kPart]
  __device__ __forceinline__ EvictKeys(const PagedEvict& a, const EvictRow& r, const EvictPart& p, bool copy, unsigned* lds)
      : a(a), r(r), copy(copy) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), share = p.part / kEWaves;
    first = p.first + share * w;
    last = min(p.last, first + share);
    this->lds = lds + 64 * kPartKeys * w + (threadIdx.x & 63);
    slots.load(r, first);
  }
  __device__ __forceinline__ void put(int t0, bool copy) {
    unsigned key[kPartKeys];
    slots.keys(a, r, t0, last, copy, key);
#pragma unroll
    for (int k = 0; k < kPartKeys; ++k) lds[64 * k] = key[k];
  }
  __device__ __forceinline__ void ready() {  // once, behind the caller's own loads
    put(first, copy);
    if (!copy) return;
    for (int t0 = first + 64 * kPartKeys; t0 < last; t0 += 64 * kPartKeys) {
      slots.load(r, t0);
      put(t0, true);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    for (int t0 = first; t0 < last; t0 += 64 * kPartKeys) {
      if (a.part != kPart) {
        slots.load(r, t0);
        put(t0, false);
      }
#pragma unroll 1
      for (int k = 0; k < kPartKeys && t0 + 64 * k < last; ++k) f(t0 + 64 * k, lds[64 * k]);
    }
  }
};

// Workspace of a row: each pass's prefix and need, then per part the number of its
// keys above the digits found so far, and its counts of the pass's digits.
struct EvictTables {
  unsigned *state, *above, *hist;
  __device__ __forceinline__ EvictTables(const PagedEvict& a, size_t row) {
    state = a.tables + row * a.table_words;
    above = state + 8;
    hist = above + ((a.most_parts + 7) & ~7);
  }
  __device__ __forceinline__ unsigned* digits(int part, int pass) const { return hist + ((size_t)part * 3 + pass) * 2048; }
};

// What pass kPass (0..3; 3: the bound itself) starts from: the digits found by the
// passes before it.
template <int kPass>
__device__ __forceinline__ void start_pass(const EvictRow& r, const EvictPart& p, const EvictTables& t, int x,
                                           unsigned* wsum, unsigned* found, unsigned& prefix, unsigned& need) {
  prefix = 0;
  need = r.m;
  if constexpr (kPass > 0) {
    const int tid = threadIdx.x;
    if (kPass > 1) {
      prefix = t.state[2 * kPass - 4];
      need = t.state[2 * kPass - 3];
    }
    uint2 sum = make_uint2(0u, 0u);
    for (int y0 = 0; y0 < p.parts; y0 += 8) {
      uint2 c[8];
#pragma unroll
      for (int y = 0; y < 8; ++y)
        c[y] = *reinterpret_cast<const uint2*>(t.digits(min(y0 + y, p.parts - 1), kPass - 1) + 2046 - 2 * tid);
#pragma unroll
      for (int y = 0; y < 8; ++y)
        if (y0 + y < p.parts) {
          sum.x += c[y].x;
          sum.y += c[y].y;
        }
    }
    find_digit<kPass - 1>(sum.y, sum.x, wsum, found, prefix, need);
    if (x == 0 && tid == 0) {
      t.state[2 * kPass - 2] = prefix;
      t.state[2 * kPass - 1] = need;
    }
  }
}

template <int kPass>
__global__ __launch_bounds__(kET) void paged_rank_kernel(PagedEvict a) {
  const int x = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  __shared__ unsigned hist[2048], wsum[kEWaves], found[2], part_keys[kPart];
  __shared__ int sums[kEWaves];
  const EvictRow r(a, b, h);
  const EvictPart p(a, r, x);
  if (kPass == 0 && x == 0 && tid == 0) {  // (paged_pick_kernel writes the new lengths)
    unsigned* sizes = EvictTables(a, r.row).state + 6;
    sizes[0] = (unsigned)r.n;
    sizes[1] = (unsigned)r.m;
  }
  if (x >= p.parts) return;
  EvictKeys keys(a, r, p, kPass == 0 && r.copy, part_keys);
  if (r.n <= r.m || r.m == 0) {
    if (kPass == 0) keys.ready();  // (the fork gets its copies)
    return;
  }
  for (int i = tid; i < 2048; i += kET) hist[i] = 0u;
  const EvictTables t(a, r.row);
  unsigned prefix, need;
  start_pass<kPass>(r, p, t, x, wsum, found, prefix, need);
  keys.ready();
  __syncthreads();
  if constexpr (kPass > 0) {  // this part's keys above the digit found
    const uint2 c = *reinterpret_cast<const uint2*>(t.digits(x, kPass - 1) + 2046 - 2 * tid);
    const int d = (int)(prefix & 2047u);
    const int above = block_sum((2047 - 2 * tid > d ? (int)c.y : 0) + (2046 - 2 * tid > d ? (int)c.x : 0), sums);
    if (tid == 0) t.above[x] = (kPass > 1 ? t.above[x] : 0u) + (unsigned)above;
  }
  keys.each([&](int, unsigned key) {
    if (matches<kPass>(key, prefix)) atomicAdd(&hist[digit<kPass>(key)], 1u);
  });
  __syncthreads();
  uint2* out = reinterpret_cast<uint2*>(t.digits(x, kPass));
  out[tid] = *reinterpret_cast<const uint2*>(&hist[2 * tid]);
}

__global__ __launch_bounds__(kET) void paged_pick_kernel(PagedEvict a) {
  const int x = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  __shared__ unsigned wsum[kEWaves], found[2], part_keys[kPart];
  __shared__ int above_s[kEWaves], equal_s[kEWaves];
  __shared__ EvictCounts counts[kEWaves];
  const EvictTables t(a, (size_t)b * a.kv_heads + h);
  const EvictRow r(a, b, h, t.state + 6);
  const EvictPart p(a, r, x);
  if (x == 0 && h == 0 && tid == 0) {
    a.lengths_out[b] = r.m;
    if (a.seen_out != a.seen) a.seen_out[b] = a.seen[b];
  }
  const bool cut = r.n > r.m && r.m > 0;
  if (!cut && x == 0 && tid == 0) a.count[r.row] = 0;
  if (!cut || x >= p.parts) return;
  EvictKeys keys(a, r, p, false, part_keys);
  unsigned bound, need;
  start_pass<3>(r, p, t, x, wsum, found, bound, need);
  keys.ready();
  // the parts in order, a wave each: what lies before this one
  const int d = (int)(bound & 1023u);
  int tie = 0, hole = 0, source = 0, tie_x = 0, hole_x = 0, source_x = 0;
  for (int y0 = 0; y0 < p.parts; y0 += kEWaves) {
    const int y = min(y0 + w, p.parts - 1);
    const unsigned* c = t.digits(y, 2);
    int more = 0;
    for (int i = 0; i < 1024; i += 256) {
      const uint4 v = reinterpret_cast<const uint4*>(c + i)[lane];
      const int at = i + 4 * lane;
      more += (at > d ? (int)v.x : 0) + (at + 1 > d ? (int)v.y : 0) + (at + 2 > d ? (int)v.z : 0) + (at + 3 > d ? (int)v.w : 0);
    }
    more = wave_sum_i(more);
    if (lane == 0) {
      above_s[w] = (int)t.above[y] + more;
      equal_s[w] = (int)c[d];
    }
    __syncthreads();
    for (int k = 0; k < min(kEWaves, p.parts - y0); ++k) {
      if (y0 + k == x) {
        tie_x = tie;
        hole_x = hole;
        source_x = source;
      }
      const int kept = above_s[k] + min(max((int)need - tie, 0), equal_s[k]);
      tie += equal_s[k];
      if (y0 + k < p.front) hole += p.size(r, y0 + k) - kept;
      else source += kept;
    }
    __syncthreads();
  }
  if (x == 0 && tid == 0) a.count[r.row] = hole;
  auto each_key = [&](auto f) { keys.each(f); };
  const EvictCounts mine = count_moves(each_key, bound, r.m, keys.last);
  write_moves(each_key, mine, bound, (int)need - tie_x, r.m, keys.last, a.dst + r.row * a.moves + hole_x,
              a.src + r.row * a.moves + source_x, counts, -1, nullptr, nullptr);
}

// Moves the kept rows into the holes where the selection has not: a copy, bound by
// the rows it reads and writes.  No source is another move's destination.  100 MB
// of 256-byte rows read and written: 23.2 us = 4.4 TB/s (4 or 8 rows in flight per
// thread: fewer workgroups, and 1 to 4 us more).
constexpr int kMoveRows = 2;

__global__ __launch_bounds__(kPT) void paged_move_kernel(PagedEvict a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const size_t row = (size_t)b * a.kv_heads + h;
  move_rows<kPT, kMoveRows>(a, b, h, row, a.src + row * a.moves, a.dst + row * a.moves, a.count[row], blockIdx.x, gridDim.x);
}

}  // namespace
}  // namespace prismkv

using namespace prismkv;

namespace {

PageDiv page_div(int page_size) {
  int log = 0;
  while ((1ll << log) < page_size) ++log;
  const int shift = 31 + log;
  return PageDiv{(unsigned)(((1ull << shift) + page_size - 1) / page_size), shift};
}

int element_bytes(int dtype) { return dtype == kFp32 ? 4 : 2; }

// The second cache's lengths, tokens seen, scores and positions are all the first's or
// lie apart from all of them: a launch reads the first's while it writes the second's.
bool results_fit(const prismkv_paged_cache& c, const prismkv_paged_cache& to) {
  if (to.lengths == c.lengths && to.seen == c.seen && to.scores == c.scores && to.positions == c.positions) return true;
  const uint64_t few = 4ull * c.sequences, many = few * c.kv_heads * c.page_size * c.max_pages;
  const uint64_t from[4] = {c.lengths, c.seen, c.scores, c.positions}, into[4] = {to.lengths, to.seen, to.scores, to.positions};
  const uint64_t size[4] = {few, few, many, many};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (from[i] && into[j] && from[i] < into[j] + size[j] && into[j] < from[i] + size[i]) return false;
  return true;
}

// The cache and where its results go, checked alike by every entry point: rows,
// heads and pages lie at 16-byte multiples, and a page's last row within 2^32
// 16-byte units.  0, or the code to return.
int check_cache(const prismkv_paged_cache* cache, const prismkv_paged_cache* into, bool scored) {
  if (!cache || !into) return kBadSize;
  const prismkv_paged_cache& c = *cache;
  const prismkv_paged_cache& to = *into;
  if (c.dtype < kBf16 || c.dtype > kFp32) return kBadMode;
  if (c.sequences < 1 || c.sequences > 65535 || c.kv_heads < 1 || c.kv_heads > 65535 || c.page_size < 1 ||
      c.max_pages < 1 || c.pages < 1 || c.pages > INT32_MAX)
    return kBadSize;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return kBadSize;
  const int64_t slots = (int64_t)c.page_size * c.max_pages;
  if (slots > (1 << 30) || slots * c.sequences > INT32_MAX) return kBadSize;
  const int64_t es = element_bytes(c.dtype), limit = 1ll << 36;  // bytes
  if (c.page_stride < 0 || c.head_stride < 0 || c.slot_stride < c.head_dim) return kBadSize;
  if (c.page_stride > limit || c.head_stride > limit || c.slot_stride > limit) return kBadSize;
  if ((c.page_stride * es | c.head_stride * es | c.slot_stride * es) & 15) return kBadSize;
  if (c.page_stride * es > limit / c.pages || c.slot_stride * es > limit / c.page_size) return kBadSize;
  if ((c.pages - 1) * c.page_stride * es + (c.page_size - 1) * c.slot_stride * es >= limit) return kBadSize;
  if (to.k != c.k || to.v != c.v || to.table != c.table || to.pages != c.pages || to.page_stride != c.page_stride ||
      to.head_stride != c.head_stride || to.slot_stride != c.slot_stride || to.sequences != c.sequences ||
      to.kv_heads != c.kv_heads || to.head_dim != c.head_dim || to.page_size != c.page_size ||
      to.max_pages != c.max_pages || to.dtype != c.dtype)
    return kBadSize;
  if (!c.k || !c.v || !c.table || !c.lengths || !to.lengths || !c.err) return kBadSize;
  if ((c.k | c.v) & 15 || c.err & 7 ||
      (c.table | c.lengths | c.seen | c.scores | c.positions | to.lengths | to.seen | to.scores | to.positions) & 3)
    return kBadSize;
  const bool some = c.seen || c.scores || c.positions || to.seen || to.scores || to.positions;
  const bool all = c.seen && c.scores && c.positions && to.seen && to.scores && to.positions;
  return some != all || (scored && !all) || !results_fit(c, to) ? kBadSize : 0;
}

struct WorkLayout {
  size_t sums, state, logits, bytes;  // counters first
  unsigned state_stride;
  int64_t logit_stride, quanta, units;
};

WorkLayout attend_layout(int sequences, int kv_heads, int group, int head_dim, int64_t slots, bool weigh, int dtype) {
  WorkLayout w;
  const int64_t tiles = (group + 15) / 16, heads = (int64_t)kv_heads * tiles;
  const int least = (dtype == kFp32 ? 1 : 2) * (head_dim == 256 ? kAWaves<256> : kAWaves<128>) / 2;
  const int64_t workgroups = sequences * heads * ((slots + least * kQuantum - 1) / (least * kQuantum));  // of full tables
  w.quanta = workgroups * least;
  w.units = workgroups < kUnits ? workgroups : kUnits;
  w.state_stride = (unsigned)((group < 16 ? group : 16) * (head_dim + 2));
  w.logit_stride = (slots + 31) & ~31ll;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  w.sums = up((size_t)sequences * heads * sizeof(unsigned));
  w.state = w.sums + up((size_t)sequences * kv_heads * group * sizeof(float2));
  w.logits = w.state + up((size_t)2 * w.units * w.state_stride * sizeof(float));
  w.bytes = w.logits + (weigh ? (size_t)sequences * kv_heads * group * w.logit_stride * sizeof(float) : 0);
  return w;
}

struct EvictLayout {
  size_t count, src, dst, tables, bytes;  // counters (a word per sequence) first
  int64_t moves, part, parts, table_words;
};

EvictLayout evict_layout(int sequences, int kv_heads, int64_t slots) {
  EvictLayout w;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t rows = (size_t)sequences * kv_heads;
  w.moves = slots / 2 + 1;
  w.part = kPart * ((slots + (int64_t)kPart * kMostParts - 1) / ((int64_t)kPart * kMostParts));
  w.parts = slots > ((int64_t)rows < kManyRows ? kLongRow : 2 * kLongRow) ? slots / w.part + 2 : 0;
  w.table_words = w.parts ? 8 + ((w.parts + 7) & ~7ll) + w.parts * 3 * 2048 : 0;
  w.count = up((size_t)sequences * sizeof(unsigned));
  w.src = w.count + up(rows * sizeof(int32_t));
  w.dst = w.src + up(rows * w.moves * sizeof(int32_t));
  w.tables = w.dst + up(rows * w.moves * sizeof(int32_t));
  w.bytes = w.tables + rows * w.table_words * sizeof(unsigned);
  return w;
}

template <int DT, int D, bool kAligned, bool kMany>
int launch_attend_rows(const PagedAttend& a, int64_t units, int lds, hipStream_t stream) {
  const auto kernel = paged_attend_kernel<DT, D, kAligned, kMany>;
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)units), dim3(64 * kAWaves<D>), lds, stream, a);
  return (int)hipGetLastError();
}

template <int DT, int D>
int launch_attend(PagedAttend a, int64_t units, hipStream_t stream) {
  const int rows = a.group < 16 ? a.group : 16;
  const int64_t longest = a.slots / (kLeast<DT, D> * kQuantum) + 2;
  const int64_t most = kUnits / (a.kv_heads * a.tiles) + 2;  // (a sequence's pairs are alike)
  const int chunks = (int)(longest < most ? longest : most);  // of one pair at most
  // Where a pair's states may be many and wide a second launch joins them: 65536
  // tokens of one KV head and 16 query heads (264K floats) 20.3 us, 44.9 by the last
  // workgroup; of 8 KV heads and 4 (17K) 48.5 against 47.3.
  const bool apart = (int64_t)chunks * rows * D > 49152;
  const int merge = 32 * kAWaves<D> + kAWaves<D> * rows * D, sums = 32 + chunks * rows;
  const int join = apart ? 0 : 256 * kAWaves<D> + sums;
  const int lds = (merge > join ? merge : join) * (int)sizeof(float);
  if (apart) a.counters = nullptr;
  // a lane's offset within a block is 32 bits
  const bool aligned = a.page_size % 16 == 0 && a.slot_units < (1u << 23);
  a.many = (int64_t)a.sequences * a.kv_heads * a.tiles >= kSoloPairs;
  const auto launch = aligned ? a.many ? launch_attend_rows<DT, D, true, true> : launch_attend_rows<DT, D, true, false>
                              : a.many ? launch_attend_rows<DT, D, false, true> : launch_attend_rows<DT, D, false, false>;
  const int rc = launch(a, units, lds, stream);
  if (rc || !apart) return rc;
  hipLaunchKernelGGL((paged_join_kernel<DT, D>), dim3((rows * D / 4 + kJoinColumns - 1) / kJoinColumns,
                     a.kv_heads * a.tiles, a.sequences), dim3(kPT), (4 * kPT + sums) * (int)sizeof(float), stream, a);
  return (int)hipGetLastError();
}

template <int DT>
int launch_attend_dim(const PagedAttend& a, int head_dim, int64_t units, hipStream_t stream) {
  if (head_dim == 64) return launch_attend<DT, 64>(a, units, stream);
  if (head_dim == 128) return launch_attend<DT, 128>(a, units, stream);
  return launch_attend<DT, 256>(a, units, stream);
}

}  // namespace

extern "C" {

size_t prismkv_paged_attend_work_bytes(int sequences, int kv_heads, int group, int head_dim, int64_t slots, int weigh,
                                       int dtype) {
  if (dtype < kBf16 || dtype > kFp32 || sequences < 1 || kv_heads < 1 || group < 1 || head_dim < 1 || slots < 1) return 0;
  const WorkLayout w = attend_layout(sequences, kv_heads, group, head_dim, slots, weigh != 0, dtype);
  return w.quanta > INT32_MAX ? 0 : w.bytes;  // (refused: quanta are counted in 32 bits)
}

int prismkv_paged_attend(const prismkv_paged_cache* cache, const prismkv_paged_cache* into, uint64_t q, uint64_t lse,
                         uint64_t paged_work, uint64_t out, int group, int flags, double scale, size_t work_bytes,
                         uint64_t stream) {
  const bool weigh = flags & 1;
  if (const int rc = check_cache(cache, into, weigh)) return rc;
  if (flags & ~3) return kBadMode;
  const prismkv_paged_cache& c = *cache;
  const double scale2 = scale * 1.4426950408889634;  // the exponents are powers of 2, in fp32
  if (group < 1 || group > 1024 || !(scale2 >= -FLT_MAX && scale2 <= FLT_MAX)) return kBadSize;
  if (!q || !paged_work || !out || (q | paged_work) & 15 || lse & 3 || out & 3) return kBadSize;
  const int64_t slots = (int64_t)c.page_size * c.max_pages;
  const WorkLayout w = attend_layout(c.sequences, c.kv_heads, group, c.head_dim, slots, weigh, c.dtype);
  if (work_bytes < w.bytes || w.quanta > INT32_MAX) return kBadSize;
  const int es = element_bytes(c.dtype);
  PagedAttend a{};
  a.q = reinterpret_cast<const void*>(q);
  a.k = reinterpret_cast<const void*>(c.k);
  a.v = reinterpret_cast<const void*>(c.v);
  a.table = reinterpret_cast<const int32_t*>(c.table);
  a.lengths = reinterpret_cast<const int32_t*>(flags & 2 ? into->lengths : c.lengths);
  a.lse_out = reinterpret_cast<float*>(lse);
  a.out = reinterpret_cast<void*>(out);
  char* work = reinterpret_cast<char*>(paged_work);
  a.counters = reinterpret_cast<unsigned*>(work);
  a.state = reinterpret_cast<float*>(work + w.state);
  if (weigh) {
    a.scores = reinterpret_cast<const float*>(c.scores);
    a.scores_out = reinterpret_cast<float*>(into->scores);
    a.sums_work = reinterpret_cast<float2*>(work + w.sums);
    a.logits = reinterpret_cast<float*>(work + w.logits);
  }
  a.err = reinterpret_cast<unsigned*>(c.err);
  a.head_bytes = c.head_stride * es;
  a.logit_stride = w.logit_stride;
  a.slots = slots;
  a.page_units = (unsigned)(c.page_stride * es >> 4);
  a.slot_units = (unsigned)(c.slot_stride * es >> 4);
  a.state_stride = w.state_stride;
  a.div = page_div(c.page_size);
  a.sequences = c.sequences;
  a.kv_heads = c.kv_heads;
  a.group = group;
  a.tiles = (group + 15) / 16;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.pages = (int)c.pages;
  a.scale = (float)scale2;
  const hipStream_t s = (hipStream_t)stream;
  int rc;
  if (c.dtype == kBf16) rc = launch_attend_dim<kBf16>(a, c.head_dim, w.units, s);
  else if (c.dtype == kFp16) rc = launch_attend_dim<kFp16>(a, c.head_dim, w.units, s);
  else rc = launch_attend_dim<kFp32>(a, c.head_dim, w.units, s);
  if (rc || !weigh) return rc;
  const int64_t blocks = (slots + kPT - 1) / kPT;
  hipLaunchKernelGGL(paged_weigh_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024), c.kv_heads, c.sequences),
                     dim3(kPT), 0, s, a);
  return (int)hipGetLastError();
}

int prismkv_paged_append(const prismkv_paged_cache* cache, const prismkv_paged_cache* into, uint64_t k, uint64_t v,
                         uint64_t offsets, int64_t rows, int64_t k_row_stride, int64_t k_head_stride,
                         int64_t v_row_stride, int64_t v_head_stride, uint64_t stream) {
  if (const int rc = check_cache(cache, into, false)) return rc;
  const prismkv_paged_cache& c = *cache;
  if (rows < 0 || rows > INT32_MAX || (!offsets && rows != c.sequences)) return kBadSize;
  if (rows && (!k || !v)) return kBadSize;
  const int64_t es = element_bytes(c.dtype), limit = 1ll << 40;
  for (const int64_t stride : {k_row_stride, k_head_stride, v_row_stride, v_head_stride})
    if (stride < -limit || stride > limit || stride * es & 15) return kBadSize;
  if ((k | v) & 15 || offsets & 3) return kBadSize;
  PagedAppend a{};
  a.k = reinterpret_cast<const char*>(k);
  a.v = reinterpret_cast<const char*>(v);
  a.kp = reinterpret_cast<char*>(c.k);
  a.vp = reinterpret_cast<char*>(c.v);
  a.table = reinterpret_cast<const int32_t*>(c.table);
  a.offsets = reinterpret_cast<const int32_t*>(offsets);
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
  a.page_bytes = c.page_stride * es;
  a.head_bytes = c.head_stride * es;
  a.slot_bytes = c.slot_stride * es;
  a.div = page_div(c.page_size);
  a.sequences = c.sequences;
  a.kv_heads = c.kv_heads;
  while (16 << a.log_pieces < c.head_dim * es) ++a.log_pieces;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.pages = (int)c.pages;
  a.slots = c.page_size * c.max_pages;
  const hipStream_t s = (hipStream_t)stream;
  if (!offsets) {
    hipLaunchKernelGGL(paged_append_kernel, dim3(c.sequences), dim3(kPT), 0, s, a);
    return (int)hipGetLastError();
  }
  for (; a.first_row < rows; a.first_row += kLaunchRows) {
    const int64_t more = rows - a.first_row < kLaunchRows ? rows - a.first_row : kLaunchRows;
    hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)((more + kAppendRows - 1) / kAppendRows)), dim3(kPT), 0, s, a);
    if (const int rc = (int)hipGetLastError()) return rc;
  }
  if (rows && a.lengths_out != a.lengths) return 0;  // (advanced by the rows' launches)
  hipLaunchKernelGGL(paged_advance_kernel, dim3((c.sequences + kPT - 1) / kPT), dim3(kPT), 0, s, a);
  return (int)hipGetLastError();
}

size_t prismkv_paged_evict_work_bytes(int sequences, int kv_heads, int64_t slots) {
  if (sequences < 1 || kv_heads < 1 || slots < 1 || slots > 1 << 30) return 0;
  return evict_layout(sequences, kv_heads, slots).bytes;
}

int prismkv_paged_evict(const prismkv_paged_cache* cache, const prismkv_paged_cache* into, uint64_t keeps,
                        uint64_t paged_work, int keep, int recent, int sinks, size_t work_bytes, uint64_t stream) {
  if (const int rc = check_cache(cache, into, true)) return rc;
  const prismkv_paged_cache& c = *cache;
  if (keep < 0 || recent < 0 || sinks < 0 || (keeps && keep)) return kBadSize;
  if (!paged_work || paged_work & 15 || keeps & 3) return kBadSize;
  const int64_t slots = (int64_t)c.page_size * c.max_pages;
  const EvictLayout l = evict_layout(c.sequences, c.kv_heads, slots);
  if (work_bytes < l.bytes) return kBadSize;
  const int es = element_bytes(c.dtype);
  PagedEvict a{};
  a.kp = reinterpret_cast<char*>(c.k);
  a.vp = reinterpret_cast<char*>(c.v);
  a.table = reinterpret_cast<const int32_t*>(c.table);
  a.lengths = reinterpret_cast<const int32_t*>(c.lengths);
  a.lengths_out = reinterpret_cast<int32_t*>(into->lengths);
  a.seen = reinterpret_cast<const int32_t*>(c.seen);
  a.seen_out = reinterpret_cast<int32_t*>(into->seen);
  a.scores = reinterpret_cast<const float*>(c.scores);
  a.scores_out = reinterpret_cast<float*>(into->scores);
  a.positions = reinterpret_cast<const int32_t*>(c.positions);
  a.positions_out = reinterpret_cast<int32_t*>(into->positions);
  a.keeps = reinterpret_cast<const int32_t*>(keeps);
  char* work = reinterpret_cast<char*>(paged_work);
  a.moves = l.moves;
  a.counters = reinterpret_cast<unsigned*>(work);
  a.count = reinterpret_cast<int32_t*>(work + l.count);
  a.src = reinterpret_cast<int32_t*>(work + l.src);
  a.dst = reinterpret_cast<int32_t*>(work + l.dst);
  a.tables = reinterpret_cast<unsigned*>(work + l.tables);
  a.table_words = l.table_words;
  a.part = (int)l.part;
  a.most_parts = (int)l.parts;
  a.err = reinterpret_cast<unsigned*>(c.err);
  a.page_bytes = c.page_stride * es;
  a.head_bytes = c.head_stride * es;
  a.slot_bytes = c.slot_stride * es;
  a.div = page_div(c.page_size);
  a.sequences = c.sequences;
  a.kv_heads = c.kv_heads;
  while (16 << a.log_pieces < c.head_dim * es) ++a.log_pieces;
  a.page_size = c.page_size;
  a.max_pages = c.max_pages;
  a.pages = (int)c.pages;
  a.slots = (int)slots;
  a.keep = keep;
  a.recent = recent;
  a.sinks = sinks;
  const hipStream_t s = (hipStream_t)stream;
  int64_t most = slots / 2;  // moves of a row
  if (!keeps) most = keep < slots - keep ? keep : slots > keep ? slots - keep : 0;
  if (most > slots / 2) most = slots / 2;
  int rc;
  if (!l.parts) {
    const int lds = (int)((slots + 64 * kEWaves - 1) / (64 * kEWaves)) * 64 * kEWaves * (int)sizeof(unsigned);
    if (lds > 32 * 1024) {  // (beside the static 27 KB)
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_select_kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 2 * kLongRow * (int)sizeof(unsigned));
      if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(paged_select_kernel, dim3(c.kv_heads, c.sequences), dim3(kET), lds, s, a);
    rc = (int)hipGetLastError();
    if (rc || most <= kFew) return rc;
  } else {
    const dim3 grid((unsigned)l.parts, c.kv_heads, c.sequences);
    hipLaunchKernelGGL(paged_rank_kernel<0>, grid, dim3(kET), 0, s, a);
    hipLaunchKernelGGL(paged_rank_kernel<1>, grid, dim3(kET), 0, s, a);
    hipLaunchKernelGGL(paged_rank_kernel<2>, grid, dim3(kET), 0, s, a);
    hipLaunchKernelGGL(paged_pick_kernel, grid, dim3(kET), 0, s, a);
    rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  const int64_t blocks = (most + (kPT >> a.log_pieces) * kMoveRows - 1) / ((kPT >> a.log_pieces) * kMoveRows);
  const int64_t room = 4096 / ((int64_t)c.sequences * c.kv_heads) + 1;  // workgroups of a row where there are many rows
  const int64_t grid = blocks < 1 ? 1 : blocks < room ? blocks : room;
  hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)grid, c.kv_heads, c.sequences), dim3(kPT), 0, s, a);
  return (int)hipGetLastError();
}

}  // extern "C"
