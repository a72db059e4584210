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
// heads, bf16, 47.8 us = 5.6 TB/s; 32 sequences of 6.4K tokens 136 us = 6.2 TB/s
// (a plain read of as much memory reaches 6.9); 16 x 8192 of head_dim 256 in fp32
// 93 us = 5.8; of head_dim 64 50 us = 5.3; 75 tokens 6.7 us.  About 6 us of a call
// are the launch and the chain lengths -> page -> rows, 4 more the join.

// 16-bit types: P is a head and a remainder of the type (two products into one
// accumulator: about twice the type's significant bits).  The head is taken from
// slightly below p, so that both are positive wherever p is and an infinite V
// is not multiplied by a remainder of 0.
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

// p as a head and a remainder of the 16-bit type.
template <int DT>
__device__ __forceinline__ void split16(float p, unsigned& hi, unsigned& lo) {
  if constexpr (DT == kBf16) {
    const unsigned u = __float_as_uint(p * (1.f - 0x1p-9f)) & 0xffff0000u;
    hi = u >> 16;
    lo = f32_to_bf16(p - __uint_as_float(u));
  } else {
    const _Float16 h = (_Float16)(p * (1.f - 0x1p-10f));
    const _Float16 l = (_Float16)(p - (float)h);
    hi = __builtin_bit_cast(unsigned short, h);
    lo = __builtin_bit_cast(unsigned short, l);
  }
}

template <int N, int DT, int D>
__device__ __forceinline__ void pv_columns(f32x4 (&acc)[D / 16], const Tile<DT, D>& t, u32x4 ph, u32x4 pl) {
  if constexpr (N < D / 16) {
    const u32x4 vb = {pair16<N>(t.v[0][0], t.v[0][1]), pair16<N>(t.v[0][2], t.v[0][3]),
                      pair16<N>(t.v[1][0], t.v[1][1]), pair16<N>(t.v[1][2], t.v[1][3])};
    acc[N] = mfma32<DT>(ph, vb, acc[N]);
    acc[N] = mfma32<DT>(pl, vb, acc[N]);
    pv_columns<N + 1, DT, D>(acc, t, ph, pl);
  }
}

// 2^(scale s - m): one rounding of the difference, however large the two are.  m
// is finite or +infinity (no_less): where no score is above -infinity, 0 serves.
__device__ __forceinline__ float weight(float s, float scale, float m) {
  return __builtin_amdgcn_exp2f(fmaf(s, scale, -m));
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
template <int DT, int D, bool kAligned>
__device__ __forceinline__ void attend_segment(const PagedAttend& a, const PagedSpan<kLeast<DT, D>>& u, int quanta, int count, float* lds) {
  typedef Tile<DT, D> T;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, q = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = u.hh / a.tiles, g0 = 16 * (u.hh - h * a.tiles);
  const int rows = min(a.group - g0, 16);  // query heads of this tile
  const int start = min(u.first * kQuantum, u.n), end = min(start + count * kQuantum, u.n);

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
  constexpr int kStep = kAWaves<D> * T::kTokens;
  int t0 = start + T::kTokens * w;
  T t;
  if (t0 < end) {
    rows_of.ask(t0);
    rows_of.move();
    rows_of.load_k(t);
    rows_of.ask(t0 + kStep);
    rows_of.load_v(t);
  }
  // (the loads of the tile behind the last are issued too: on every path as many
  // are in flight, so that the compiler's wait counts are exact)
  for (; t0 < end; t0 += kStep) {
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
      if (logits && j < rows)
        *reinterpret_cast<float4*>(logits + t0 + 16 * i + 4 * q) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    }
    rows_of.move();
    rows_of.load_k(t);
    rows_of.ask(t0 + 2 * kStep);
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
      unsigned hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) split16<DT>(p[i][r], hi[4 * i + r], lo[4 * i + r]);
      const u32x4 ph = {hi[0] | hi[1] << 16, hi[2] | hi[3] << 16, hi[4] | hi[5] << 16, hi[6] | hi[7] << 16};
      const u32x4 pl = {lo[0] | lo[1] << 16, lo[2] | lo[3] << 16, lo[4] | lo[5] << 16, lo[6] | lo[7] << 16};
      pv_columns<0, DT, D>(acc, t, ph, pl);
    }
    rows_of.load_v(t);
  }
  if (__ballot(rows_of.bad) && lane == 0) report_error(a.err, error_host_slot(a.err), kErrPages);

  // the waves' states meet in LDS
  float* sm = lds;  // [waves][16] maxima
  float* sz = sm + 16 * kAWaves<D>;   // [waves][16] sums
  float* sacc = sz + 16 * kAWaves<D>; // [waves][rows][D]
  z += xor16(z);
  z += xor32(z);
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
  const size_t head0 = ((size_t)u.b * a.kv_heads + h) * a.group + g0;  // this tile's first query head
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

template <int DT, int D, bool kAligned>
__global__ __launch_bounds__(64 * kAWaves<D>, kAWaves<D> / 4) void paged_attend_kernel(PagedAttend a) {
  extern __shared__ float lds[];
  PagedSpan<kLeast<DT, D>> u = find_span<kLeast<DT, D>>(a, blockIdx.x);
  while (u.at < u.end) {  // the pairs that this workgroup's share lies in
    const int quanta = quanta_of<kLeast<DT, D>>(u.n);
    const int count = min(quanta - u.first, u.end - u.at);
    attend_segment<DT, D, kAligned>(a, u, quanta, count, lds);
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
  const int b = blockIdx.z, lane = threadIdx.x & 63;
  const int h = blockIdx.y / a.tiles, tile = blockIdx.y - h * a.tiles;
  const int rows = min(a.group - 16 * tile, 16), col0 = blockIdx.x * kJoinColumns;
  if (col0 >= rows * D / 4) return;
  constexpr int kL = kLeast<DT, D>;
  PagedDeal<kL> deal{0};
  int from = 0, n = 0;  // quanta before sequence b, its length
  each_64<kL>(a, [&](int i, int len, int c) {
    deal.total += wave_sum_i(c);
    from += wave_sum_i(i + lane < b ? c : 0);
    if (i <= b && b < i + 64) n = __builtin_amdgcn_readlane(len, b - i);
    return false;
  });
  deal.total *= a.kv_heads * a.tiles;
  const int quanta = quanta_of<kL>(n);
  const PagedParts parts(deal, from * a.kv_heads * a.tiles + (int)blockIdx.y * quanta, quanta);
  if (parts.chunks == 1) return;  // its workgroup has finished it
  join_states<DT, D, kPT>(a, ((size_t)b * a.kv_heads + h) * a.group + 16 * tile, rows, parts, col0, kJoinColumns, lds);
}

// scores_out[t] = scores[t] + sum over the group's heads of e^(s_t - lse): a
// thread per slot; bound by the scores that it reads (4 bytes per query head and
// slot) and the two score arrays.
__global__ __launch_bounds__(kPT) void paged_weigh_kernel(PagedAttend a) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int n = clamp_length(a, a.lengths[b]);
  const float* lse = a.lse_work + ((size_t)b * a.kv_heads + h) * a.group;
  const float* logits = a.logits + ((size_t)b * a.kv_heads + h) * a.group * a.logit_stride;
  const size_t at = ((size_t)b * a.kv_heads + h) * a.slots;
  for (int t = blockIdx.x * kPT + threadIdx.x; t < n; t += gridDim.x * kPT) {
    float sum = 0.f;
    for (int g = 0; g < a.group; ++g) sum += weight(logits[(size_t)g * a.logit_stride + t], a.scale, no_less(lse[g]));
    a.scores_out[at + t] = a.scores[at + t] + sum;
  }
}

// ------------------------------------------------------------------ append
//
// A copy of rows: bound by reading and writing them.  One workgroup per
// sequence (one token each) or per kAppendRows packed rows, 16 bytes per thread
// and step.

constexpr int kAppendRows = 4;

__device__ __forceinline__ void append_row(const PagedAppend& a, int64_t row, int b, int slot, int position) {
  const int p = a.div.of(slot);
  const bool room = p < a.max_pages;
  const int page = room ? a.table[(size_t)b * a.max_pages + p] : -1;
  if ((unsigned)page >= (unsigned)a.pages) {  // no page: the row is dropped
    if (threadIdx.x == 0) report_error(a.err, error_host_slot(a.err), kErrPages);
    return;
  }
  const size_t at = (size_t)page * a.page_bytes + (size_t)(slot - p * a.page_size) * a.slot_bytes;
  const int pieces = a.row_bytes >> 4;
  for (int i = threadIdx.x; i < a.kv_heads * pieces; i += kPT) {
    const int h = i / pieces, c = (i - h * pieces) << 4;
    const uint4 kv = *reinterpret_cast<const uint4*>(a.k + row * a.k_row + (int64_t)h * a.k_head + c);
    const uint4 vv = *reinterpret_cast<const uint4*>(a.v + row * a.v_row + (int64_t)h * a.v_head + c);
    *reinterpret_cast<uint4*>(a.kp + at + (size_t)h * a.head_bytes + c) = kv;
    *reinterpret_cast<uint4*>(a.vp + at + (size_t)h * a.head_bytes + c) = vv;
  }
  if (a.positions)
    for (int h = threadIdx.x; h < a.kv_heads; h += kPT) {
      const size_t i = ((size_t)b * a.kv_heads + h) * a.slots + slot;
      a.scores[i] = a.scores_out[i] = 0.f;
      a.positions[i] = a.positions_out[i] = position;
    }
}

__global__ __launch_bounds__(kPT) void paged_append_kernel(PagedAppend a) {
  if (!a.offsets) {  // one token each: row b
    const int b = blockIdx.x;
    const int n = max(a.lengths[b], 0), seen = a.positions ? a.seen[b] : 0;
    __syncthreads();  // every thread has read the length before it moves
    append_row(a, b, b, n, seen);
    if (threadIdx.x == 0) {
      a.lengths_out[b] = min(n, a.slots) + (n < a.slots);
      if (a.positions) a.seen_out[b] = seen + 1;
    }
    return;
  }
  const int64_t row0 = (int64_t)blockIdx.x * kAppendRows;
  int b = 0;
  {  // the sequence of row0: the last b with offsets[b] <= row0
    int lo = 0, hi = a.sequences;
    while (lo + 1 < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.offsets[mid] <= row0) lo = mid;
      else hi = mid;
    }
    b = lo;
  }
  for (int r = 0; r < kAppendRows && row0 + r < a.rows; ++r) {
    const int64_t row = row0 + r;
    while (b + 1 < a.sequences && a.offsets[b + 1] <= row) ++b;
    const int64_t step = row - a.offsets[b];
    if (step < 0 || row >= a.offsets[b + 1]) continue;  // a row of no sequence
    const int64_t slot = max(a.lengths[b], 0) + step;
    append_row(a, row, b, (int)min(slot, (int64_t)a.slots), a.positions ? a.seen[b] + (int)step : 0);
  }
}

__global__ __launch_bounds__(kPT) void paged_advance_kernel(PagedAppend a) {
  const int b = blockIdx.x * kPT + threadIdx.x;
  if (b >= a.sequences) return;
  const int more = max(a.offsets[b + 1] - a.offsets[b], 0);
  a.lengths_out[b] = (int)min((int64_t)max(a.lengths[b], 0) + more, (int64_t)a.slots);
  if (a.positions) a.seen_out[b] = a.seen[b] + more;
}

// ------------------------------------------------------------------ eviction

constexpr int kET = 1024;  // threads of the selection
constexpr int kEWaves = kET / 64;

// The order of the slots as an unsigned key: protected above NaN above the
// numbers (-0 as 0).
__device__ __forceinline__ unsigned evict_key(const PagedEvict& a, float score, const int32_t* positions, int edge, int t) {
  if (a.guard) {
    const int p = positions[t];
    if (p >= edge || p < a.sinks) return 0xffffffffu;
  }
  if (score != score) return 0xfffffffeu;
  const unsigned u = __float_as_uint(score == 0.f ? 0.f : score);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int evict_keep(const PagedEvict& a, int b) {
  const int keep = a.keeps ? a.keeps[b] : a.keep;
  return max(keep, 0);
}

// One workgroup per (sequence, KV head): the budget-th largest key by three
// histogram passes (11, 11 and 10 bits), then the slots that move: holes
// (evicted slots before the budget) and sources (kept slots behind it), both
// ascending, found by each wave in its own share of the slots.
__global__ __launch_bounds__(kET) void paged_select_kernel(PagedEvict a) {
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  __shared__ unsigned hist[2048], wsum[kEWaves];
  __shared__ unsigned found[2];  // the digit of the threshold, what remains of the budget
  __shared__ int ties[kEWaves], holes[kEWaves], sources[kEWaves];
  const int n = min(max(a.lengths[b], 0), a.slots), m = min(n, evict_keep(a, b));
  const size_t row = (size_t)b * a.kv_heads + h;
  const float* scores = a.scores + row * a.slots;
  const int32_t* positions = a.positions + row * a.slots;
  const int edge = a.seen[b] - a.recent;
  int* count = a.count + row;
  const bool apart = a.scores_out != a.scores;
  if (apart)  // what stays where it is; the moves overwrite the holes
    for (int t = tid; t < m; t += kET) {
      a.scores_out[row * a.slots + t] = scores[t];
      a.positions_out[row * a.slots + t] = positions[t];
    }
  if (n <= m || m == 0) {
    if (tid == 0) *count = 0;
    return;
  }
  unsigned prefix = 0, need = m;  // the need-th largest of the keys whose top bits equal prefix
  int shift = 21;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    for (int i = tid; i < 2048; i += kET) hist[i] = 0u;
    __syncthreads();
    for (int t = tid; t < n; t += kET) {
      const unsigned key = evict_key(a, scores[t], positions, edge, t);
      if (pass == 0 || key >> (shift + bits) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    // thread i owns bins 2i and 2i + 1 from the top
    const unsigned hi = hist[2047 - 2 * tid], lo = hist[2046 - 2 * tid];
    const unsigned incl = block_incl_scan<kET>(hi + lo, wsum), before = incl - hi - lo;
    if (before < need && need <= incl) {
      const bool upper = need <= before + hi;
      found[0] = upper ? 2047 - 2 * tid : 2046 - 2 * tid;
      found[1] = need - before - (upper ? 0u : hi);
    }
    __syncthreads();
    prefix = pass == 2 ? (prefix << 10) | found[0] : (prefix << 11) | found[0];
    need = found[1];
    shift = pass == 0 ? 10 : 0;
    __syncthreads();
  }
  // kept: keys above `prefix`, and the first `need` slots whose key equals it
  const int share = ((n + kEWaves - 1) / kEWaves + 63) & ~63;
  const int lo = min(w * share, n), hi = min(lo + share, n);
  int mine = 0;
  for (int t = lo + lane; t < hi; t += 64) mine += evict_key(a, scores[t], positions, edge, t) == prefix;
  mine = wave_sum_i(mine);
  if (lane == 0) ties[w] = mine;
  __syncthreads();
  int tie0 = 0;
  for (int k = 0; k < w; ++k) tie0 += ties[k];
  const unsigned long long below = (1ull << lane) - 1ull;
  int hole0 = 0, source0 = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int tie = tie0, nh = 0, ns = 0;
    for (int t0 = lo; t0 < hi; t0 += 64) {
      const int t = t0 + lane;
      const bool live = t < hi;
      const unsigned key = live ? evict_key(a, scores[t], positions, edge, t) : 0u;
      const unsigned long long eq = __ballot(live && key == prefix);
      const bool kept = live && (key > prefix || (key == prefix && tie + __popcll(eq & below) < (int)need));
      tie += __popcll(eq);
      const unsigned long long hm = __ballot(live && t < m && !kept), sm = __ballot(kept && t >= m);
      if (pass == 1) {
        if (hm >> lane & 1) a.dst[row * a.moves + hole0 + nh + __popcll(hm & below)] = t;
        if (sm >> lane & 1) a.src[row * a.moves + source0 + ns + __popcll(sm & below)] = t;
      }
      nh += __popcll(hm);
      ns += __popcll(sm);
    }
    if (pass == 0) {
      if (lane == 0) {
        holes[w] = nh;
        sources[w] = ns;
      }
      __syncthreads();
      int total = 0;
      for (int k = 0; k < kEWaves; ++k) {
        if (k < w) {
          hole0 += holes[k];
          source0 += sources[k];
        }
        total += holes[k];
      }
      if (tid == 0) *count = total;
    }
  }
}

// Moves the kept rows into the holes: a copy, bound by the rows it reads and
// writes.  No source is another move's destination.
__global__ __launch_bounds__(kPT) void paged_move_kernel(PagedEvict a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const size_t row = (size_t)b * a.kv_heads + h;
  const int count = a.count[row];
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
    a.lengths_out[b] = min(min(max(a.lengths[b], 0), a.slots), evict_keep(a, b));
    if (a.seen_out != a.seen) a.seen_out[b] = a.seen[b];
  }
  const int pieces = a.row_bytes >> 4;
  const int32_t* tab = a.table + (size_t)b * a.max_pages;
  for (int i = blockIdx.x * kPT + threadIdx.x; i < count * pieces; i += gridDim.x * kPT) {
    const int k = i / pieces, c = (i - k * pieces) << 4;
    const int src = a.src[row * a.moves + k], dst = a.dst[row * a.moves + k];
    const int ps = a.div.of(src), pd = a.div.of(dst);
    const int from = tab[ps], to = tab[pd];
    if ((unsigned)from >= (unsigned)a.pages || (unsigned)to >= (unsigned)a.pages) {
      report_error(a.err, error_host_slot(a.err), kErrPages);
      continue;
    }
    const size_t f = (size_t)from * a.page_bytes + (size_t)(src - ps * a.page_size) * a.slot_bytes +
                     (size_t)h * a.head_bytes + c;
    const size_t t = (size_t)to * a.page_bytes + (size_t)(dst - pd * a.page_size) * a.slot_bytes +
                     (size_t)h * a.head_bytes + c;
    const uint4 kv = *reinterpret_cast<const uint4*>(a.kp + f);
    const uint4 vv = *reinterpret_cast<const uint4*>(a.vp + f);
    *reinterpret_cast<uint4*>(a.kp + t) = kv;
    *reinterpret_cast<uint4*>(a.vp + t) = vv;
    if (c == 0) {
      a.scores_out[row * a.slots + dst] = a.scores[row * a.slots + src];
      a.positions_out[row * a.slots + dst] = a.positions[row * a.slots + src];
    }
  }
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

// Sizes that every entry point takes, checked alike.  Strides are in elements;
// rows, heads and pages lie at 16-byte multiples, and a page's last row within
// 2^32 16-byte units.
bool bad_cache(int sequences, int kv_heads, int head_dim, int page_size, int max_pages, int64_t pages, int64_t page_stride,
               int64_t head_stride, int64_t slot_stride, int dtype) {
  if (sequences < 1 || sequences > 65535 || kv_heads < 1 || kv_heads > 65535 || page_size < 1 || max_pages < 1 ||
      pages < 1 || pages > INT32_MAX)
    return true;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return true;
  const int64_t slots = (int64_t)page_size * max_pages;
  if (slots > (1 << 30) || slots * sequences > INT32_MAX) return true;
  const int64_t es = element_bytes(dtype);
  if (page_stride < 0 || head_stride < 0 || slot_stride < head_dim) return true;
  if ((page_stride * es | head_stride * es | slot_stride * es) & 15) return true;
  const int64_t limit = 1ll << 36;  // bytes
  if (page_stride > limit || head_stride > limit || slot_stride > limit) return true;
  if (page_stride * es > limit / pages || slot_stride * es > limit / page_size) return true;
  if ((pages - 1) * page_stride * es + (page_size - 1) * slot_stride * es >= limit) return true;
  return false;
}

struct WorkLayout {
  size_t lse, state, logits, bytes;  // counters first
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
  w.lse = up((size_t)sequences * heads * sizeof(unsigned));
  w.state = w.lse + up((size_t)sequences * kv_heads * group * sizeof(float));
  w.logits = w.state + up((size_t)2 * w.units * w.state_stride * sizeof(float));
  w.bytes = w.logits + (weigh ? (size_t)sequences * kv_heads * group * w.logit_stride * sizeof(float) : 0);
  return w;
}

template <int DT, int D, bool kAligned>
int launch_attend_rows(const PagedAttend& a, int64_t units, int lds, hipStream_t stream) {
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_attend_kernel<DT, D, kAligned>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL((paged_attend_kernel<DT, D, kAligned>), dim3((unsigned)units), dim3(64 * kAWaves<D>), lds, stream, a);
  return (int)hipGetLastError();
}

template <int DT, int D>
int launch_attend(PagedAttend a, int64_t units, hipStream_t stream) {
  const int rows = a.group < 16 ? a.group : 16;
  const int64_t longest = a.slots / (kLeast<DT, D> * kQuantum) + 2;
  const int64_t most = kUnits / (a.kv_heads * a.tiles) + 2;  // (a sequence's pairs are alike)
  const int chunks = (int)(longest < most ? longest : most);  // of one pair at most
    // Where a pair's states may be many and wide a second launch joins them: 65536
  // tokens of one KV head and 16 query heads (264K floats) 20.0 us, 47.5 by the last
  // workgroup; of 8 KV heads and 4 (17K) 48.2 against 47.8.
  const bool apart = (int64_t)chunks * rows * D > 49152;
  const int merge = 32 * kAWaves<D> + kAWaves<D> * rows * D, sums = 32 + chunks * rows;
  const int join = apart ? 0 : 256 * kAWaves<D> + sums;
  const int lds = (merge > join ? merge : join) * (int)sizeof(float);
  if (apart) a.counters = nullptr;
  // a lane's offset within a block is 32 bits
  const bool aligned = a.page_size % 16 == 0 && a.slot_units < (1u << 23);
  const int rc = aligned ? launch_attend_rows<DT, D, true>(a, units, lds, stream)
                         : launch_attend_rows<DT, D, false>(a, units, lds, stream);
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
  return attend_layout(sequences, kv_heads, group, head_dim, slots, weigh != 0, dtype).bytes;
}

int prismkv_paged_attend(uint64_t q, uint64_t k, uint64_t v, uint64_t table, uint64_t lengths, uint64_t scores,
                         uint64_t scores_out, uint64_t lse, uint64_t paged_work, uint64_t err, uint64_t out, int sequences,
                         int kv_heads, int group, int head_dim, int page_size, int max_pages, int64_t pages,
                         int64_t page_stride, int64_t head_stride, int64_t slot_stride, double scale, int dtype,
                         size_t work_bytes, uint64_t stream) {
  if (dtype < kBf16 || dtype > kFp32) return kBadMode;
  if (bad_cache(sequences, kv_heads, head_dim, page_size, max_pages, pages, page_stride, head_stride, slot_stride, dtype))
    return kBadSize;
  if (group < 1 || group > 1024 || !(scale == scale)) return kBadSize;
  if (!q || !k || !v || !table || !lengths || !paged_work || !err || !out || !scores != !scores_out) return kBadSize;
  if ((q | k | v | paged_work) & 15 || (table | lengths | scores | scores_out | lse) & 3 || err & 7) return kBadSize;
  const int64_t slots = (int64_t)page_size * max_pages;
  const WorkLayout w = attend_layout(sequences, kv_heads, group, head_dim, slots, scores != 0, dtype);
  if (work_bytes < w.bytes || w.quanta > INT32_MAX) return kBadSize;  // (quanta are counted in 32 bits)
  const int es = element_bytes(dtype);
  PagedAttend a{};
  a.q = reinterpret_cast<const void*>(q);
  a.k = reinterpret_cast<const void*>(k);
  a.v = reinterpret_cast<const void*>(v);
  a.table = reinterpret_cast<const int32_t*>(table);
  a.lengths = reinterpret_cast<const int32_t*>(lengths);
  a.scores = reinterpret_cast<const float*>(scores);
  a.scores_out = reinterpret_cast<float*>(scores_out);
  a.lse_out = reinterpret_cast<float*>(lse);
  a.out = reinterpret_cast<void*>(out);
  char* work = reinterpret_cast<char*>(paged_work);
  a.counters = reinterpret_cast<unsigned*>(work);
  a.state = reinterpret_cast<float*>(work + w.state);
  if (scores) {
    a.lse_work = reinterpret_cast<float*>(work + w.lse);
    a.logits = reinterpret_cast<float*>(work + w.logits);
  }
  a.err = reinterpret_cast<unsigned*>(err);
  a.head_bytes = head_stride * es;
  a.logit_stride = w.logit_stride;
  a.slots = slots;
  a.page_units = (unsigned)(page_stride * es >> 4);
  a.slot_units = (unsigned)(slot_stride * es >> 4);
  a.state_stride = w.state_stride;
  a.div = page_div(page_size);
  a.sequences = sequences;
  a.kv_heads = kv_heads;
  a.group = group;
  a.tiles = (group + 15) / 16;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.pages = (int)pages;
  a.scale = (float)(scale * 1.4426950408889634);
  const hipStream_t s = (hipStream_t)stream;
  int rc;
  if (dtype == kBf16) rc = launch_attend_dim<kBf16>(a, head_dim, w.units, s);
  else if (dtype == kFp16) rc = launch_attend_dim<kFp16>(a, head_dim, w.units, s);
  else rc = launch_attend_dim<kFp32>(a, head_dim, w.units, s);
  if (rc || !scores) return rc;
  const int64_t blocks = (slots + kPT - 1) / kPT;
  hipLaunchKernelGGL(paged_weigh_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024), kv_heads, sequences), dim3(kPT), 0,
                     s, a);
  return (int)hipGetLastError();
}

int prismkv_paged_append(uint64_t k, uint64_t v, uint64_t k_pages, uint64_t v_pages, uint64_t table, uint64_t offsets,
                         uint64_t lengths, uint64_t lengths_out, uint64_t seen, uint64_t seen_out, uint64_t scores,
                         uint64_t scores_out, uint64_t positions, uint64_t positions_out, uint64_t err, int64_t rows,
                         int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                         int sequences, int kv_heads, int head_dim, int page_size, int max_pages, int64_t pages,
                         int64_t page_stride, int64_t head_stride, int64_t slot_stride, int dtype, uint64_t stream) {
  if (dtype < kBf16 || dtype > kFp32) return kBadMode;
  if (bad_cache(sequences, kv_heads, head_dim, page_size, max_pages, pages, page_stride, head_stride, slot_stride, dtype))
    return kBadSize;
  if (rows < 0 || rows > INT32_MAX || (!offsets && rows != sequences)) return kBadSize;
  if (!k_pages || !v_pages || !table || !lengths || !lengths_out || !err || (rows && (!k || !v))) return kBadSize;
  const bool scored = positions != 0;
  if (scored && (!positions_out || !scores || !scores_out || !seen || !seen_out)) return kBadSize;
  const int es = element_bytes(dtype);
  if ((k | v | k_pages | v_pages) & 15 || err & 7 ||
      (table | offsets | lengths | lengths_out | seen | seen_out | scores | scores_out | positions | positions_out) & 3)
    return kBadSize;
  if ((k_row_stride * es | k_head_stride * es | v_row_stride * es | v_head_stride * es) & 15) return kBadSize;
  PagedAppend a{};
  a.k = reinterpret_cast<const char*>(k);
  a.v = reinterpret_cast<const char*>(v);
  a.kp = reinterpret_cast<char*>(k_pages);
  a.vp = reinterpret_cast<char*>(v_pages);
  a.table = reinterpret_cast<const int32_t*>(table);
  a.offsets = reinterpret_cast<const int32_t*>(offsets);
  a.lengths = reinterpret_cast<const int32_t*>(lengths);
  a.lengths_out = reinterpret_cast<int32_t*>(lengths_out);
  a.seen = reinterpret_cast<const int32_t*>(seen);
  a.seen_out = reinterpret_cast<int32_t*>(seen_out);
  a.positions = reinterpret_cast<int32_t*>(positions);
  a.positions_out = reinterpret_cast<int32_t*>(positions_out);
  a.scores = reinterpret_cast<float*>(scores);
  a.scores_out = reinterpret_cast<float*>(scores_out);
  a.err = reinterpret_cast<unsigned*>(err);
  a.rows = rows;
  a.k_row = k_row_stride * es;
  a.k_head = k_head_stride * es;
  a.v_row = v_row_stride * es;
  a.v_head = v_head_stride * es;
  a.page_bytes = page_stride * es;
  a.head_bytes = head_stride * es;
  a.slot_bytes = slot_stride * es;
  a.div = page_div(page_size);
  a.sequences = sequences;
  a.kv_heads = kv_heads;
  a.row_bytes = head_dim * es;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.pages = (int)pages;
  a.slots = page_size * max_pages;
  const hipStream_t s = (hipStream_t)stream;
  if (!offsets) {
    hipLaunchKernelGGL(paged_append_kernel, dim3(sequences), dim3(kPT), 0, s, a);
    return (int)hipGetLastError();
  }
  if (rows) {
    hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)((rows + kAppendRows - 1) / kAppendRows)), dim3(kPT), 0, s, a);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  hipLaunchKernelGGL(paged_advance_kernel, dim3((sequences + kPT - 1) / kPT), dim3(kPT), 0, s, a);
  return (int)hipGetLastError();
}

size_t prismkv_paged_evict_work_bytes(int sequences, int kv_heads, int64_t slots) {
  if (sequences < 1 || kv_heads < 1 || slots < 1) return 0;
  return (size_t)sequences * kv_heads * (1 + 2 * (size_t)(slots / 2 + 1)) * sizeof(int32_t);
}

int prismkv_paged_evict(uint64_t k_pages, uint64_t v_pages, uint64_t table, uint64_t lengths, uint64_t lengths_out,
                        uint64_t seen, uint64_t seen_out, uint64_t scores, uint64_t scores_out, uint64_t positions,
                        uint64_t positions_out, uint64_t keeps, uint64_t paged_work, uint64_t err, int keep, int recent,
                        int sinks, int sequences, int kv_heads, int head_dim, int page_size, int max_pages, int64_t pages,
                        int64_t page_stride, int64_t head_stride, int64_t slot_stride, int dtype, size_t work_bytes,
                        uint64_t stream) {
  if (dtype < kBf16 || dtype > kFp32) return kBadMode;
  if (bad_cache(sequences, kv_heads, head_dim, page_size, max_pages, pages, page_stride, head_stride, slot_stride, dtype))
    return kBadSize;
  if (keep < 0 || recent < 0 || sinks < 0 || (keeps && keep)) return kBadSize;
  if (!k_pages || !v_pages || !table || !lengths || !lengths_out || !seen || !seen_out || !scores || !scores_out ||
      !positions || !positions_out || !paged_work || !err)
    return kBadSize;
  if ((k_pages | v_pages) & 15 || err & 7 ||
      (table | lengths | lengths_out | seen | seen_out | scores | scores_out | positions | positions_out | keeps |
       paged_work) & 3)
    return kBadSize;
  const int64_t slots = (int64_t)page_size * max_pages;
  if (work_bytes < prismkv_paged_evict_work_bytes(sequences, kv_heads, slots)) return kBadSize;
  const int es = element_bytes(dtype);
  PagedEvict a{};
  a.kp = reinterpret_cast<char*>(k_pages);
  a.vp = reinterpret_cast<char*>(v_pages);
  a.table = reinterpret_cast<const int32_t*>(table);
  a.lengths = reinterpret_cast<const int32_t*>(lengths);
  a.lengths_out = reinterpret_cast<int32_t*>(lengths_out);
  a.seen = reinterpret_cast<const int32_t*>(seen);
  a.seen_out = reinterpret_cast<int32_t*>(seen_out);
  a.scores = reinterpret_cast<const float*>(scores);
  a.scores_out = reinterpret_cast<float*>(scores_out);
  a.positions = reinterpret_cast<const int32_t*>(positions);
  a.positions_out = reinterpret_cast<int32_t*>(positions_out);
  a.keeps = reinterpret_cast<const int32_t*>(keeps);
  a.moves = slots / 2 + 1;
  a.count = reinterpret_cast<int32_t*>(paged_work);
  a.src = a.count + (size_t)sequences * kv_heads;
  a.dst = a.src + (size_t)sequences * kv_heads * a.moves;
  a.err = reinterpret_cast<unsigned*>(err);
  a.page_bytes = page_stride * es;
  a.head_bytes = head_stride * es;
  a.slot_bytes = slot_stride * es;
  a.div = page_div(page_size);
  a.sequences = sequences;
  a.kv_heads = kv_heads;
  a.row_bytes = head_dim * es;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.pages = (int)pages;
  a.slots = (int)slots;
  a.keep = keep;
  a.recent = recent;
  a.sinks = sinks;
  a.guard = recent > 0 || sinks > 0;
  const hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(paged_select_kernel, dim3(kv_heads, sequences), dim3(kET), 0, s, a);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  const int64_t pieces = (int64_t)(head_dim * es >> 4) * (slots / 2 + 1);
  const int64_t blocks = (pieces + kPT - 1) / kPT;
  hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)(blocks < 64 ? blocks : 64), kv_heads, sequences), dim3(kPT), 0, s,
                     a);
  return (int)hipGetLastError();
}

}  // extern "C"
