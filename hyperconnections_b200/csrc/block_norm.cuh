// block_norm.cuh — the norm kernels by eight columns a thread: for rows of whole
// chunks on 16-byte boundaries (D a multiple of 8), and, ragged, for any others.
//
// A token belongs to a group of W = ceil(D / 256) warps: a CTA for W > 1, one
// of a CTA's four warps for W = 1. A thread owns eight columns of every row,
// reads them once and writes its outputs once. The groups walk the tokens
// grid-strided.
//
// What bounds these kernels is HBM, as long as enough loads are in flight and
// the instructions keep up; both shaped the layout:
//   * a thread copies its own 16 bytes of every row of the next token to shared
//     memory (cp.async) while it works on this one. It reads nothing that
//     another thread copied, so the rows need no barrier, and they cost no
//     registers while they travel;
//   * the token's small matrices (R, or H, W and v) and its norm's statistics
//     are copied one token earlier still, so that the barrier between them and
//     their use is one that the group passes anyway;
//   * arithmetic is on pairs of float32 (fma.rn.f32x2); the small matrices'
//     entries lie in shared memory twice, as the pairs that it multiplies with;
//   * kernels exist for 1, 2, 4, 8 streams and 1, 2, 4 blocks. Rows and entries
//     past n and m are zeros in shared memory, never fetched and never stored,
//     so that no product asks for n or m;
//   * a warp folds k sums by halving exchanges (every exchange sends half of
//     the live values: about k + 5 - log k shuffles), writes them to shared
//     memory, and behind the group's barrier every thread adds the W warps' in
//     order. The backward's sums are the norm's two and the token's small
//     matrices'. The mix-write has all of them before its barrier and adds them
//     behind it; the read's second ones come out of the gradients, behind the
//     barrier, and are added behind the next token's. A token costs one barrier
//     (the mix-write's backward with a projection, whose matrices pass from
//     thread to thread, three).
// Ragged rows cost more instructions, not more bytes: they travel in 4-byte
// copies and are shifted when they are read, g x^T is summed on the FMA units,
// and outputs are put together in shared memory. (16,384 tokens, n = 4, bf16,
// forward and backward: 168 us at D = 769 against 95 at 768 for the read, 444
// against 180 for the mix-write.)
//
// The [m D] parameters' gradients are sums over tokens: a thread keeps its
// columns' sums in registers over all of its group's tokens and writes them
// once; block_capi.cu adds the groups' sums in order.
#pragma once

#include <type_traits>

#include "block_elem.cuh"
#include "pairs.cuh"

namespace hc {

constexpr int kColumns = 8;      // a thread's columns
constexpr int kSmallGroups = 4;  // groups of a CTA when a group is one warp
constexpr int kSmallSlots = 8;   // tokens whose small matrices are held (5 are live; a power of two)
constexpr int kCtaSmemMax = 227 * 1024;
constexpr int kNormSmemMax = 210 * 1024;  // dynamic; the sums of a token are static, up to 12.3 KB (n = 8, m = 4, 512 threads)

// Threads of a CTA at most, which bounds the registers of one. WIDE: kernels
// with room for 4096 columns, whose registers spill, for tokens that the others
// have too few threads for. (The mix-write's backward, n = 8, m = 2: 2,048 x 4096
// bf16 in 203 us, at 4104 columns element by element 2,302; 4,096 x 1024 fp16,
// which needs no such room, forward and backward in 192 against 152.)
constexpr int kWideThreads = 512;
constexpr int norm_bwd_threads(int N, int M, int esize, bool wide) {
  return wide ? kWideThreads : M >= 4 || (N == 8 && esize == 4) ? 256 : M == 2 || N == 8 ? 384 : 512;
}
// Chunks a thread may own in the forward (a token's rows then need fewer warps,
// down to one without barriers): as many as keep a block's rows in registers.
constexpr int norm_fwd_chunks(int N, int M, int esize) { return M == 1 && N <= 4 && esize == 2 ? 3 : 1; }
constexpr int norm_fwd_threads(int N, int M, int CH, int esize, bool wide) {
  return wide ? kWideThreads : M >= 4 ? 384 : CH > 1 ? 512 : 640;
}

// K pairs of a row of a small matrix, loaded where they are used: kept for both
// halves of the columns, a mix of 8 streams alone would fill the registers.
template <int K> __device__ __forceinline__ void pairs(const f2* p, f2 (&v)[K]) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  if constexpr (K == 1) {
    asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v[0]) : "r"(at));
  } else {
#pragma unroll
    for (int i = 0; i < K; i += 2) asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(v[i]), "=l"(v[i + 1]) : "r"(at + 8 * i));
  }
}

__device__ __forceinline__ bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

struct V8 {  // eight columns
  f2 v[4];
  __device__ __forceinline__ void fill(float a) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = both(a);
  }
};
__device__ __forceinline__ float dot(const V8& a, const V8& b) {
  f2 s = mul2(a.v[0], b.v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) s = fma2(a.v[i], b.v[i], s);
  return fold2(s);
}
__device__ __forceinline__ void axpy(f2 aa, const V8& x, V8& y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) y.v[i] = fma2(aa, x.v[i], y.v[i]);
}

template <typename T> constexpr int kWords = sizeof(T) / 2;  // 16-byte words of eight columns

// Four of the eight columns: the products with all rows at once are done by
// halves where N rows of eight would not leave registers for more warps.
struct V4 {
  f2 v[2];
};
__device__ __forceinline__ void axpy(f2 aa, const V4& x, V4& y) {
  y.v[0] = fma2(aa, x.v[0], y.v[0]);
  y.v[1] = fma2(aa, x.v[1], y.v[1]);
}
template <typename T> __device__ __forceinline__ void put4(T* p, const V4& r) {
  float f[4];
  split(r.v[0], f[0], f[1]);
  split(r.v[1], f[2], f[3]);
  if constexpr (sizeof(T) == 4) {
    st_v4(p, pack<float>(f));
  } else {
    const float g[8] = {f[0], f[1], f[2], f[3], 0.f, 0.f, 0.f, 0.f};
    const uint4 q = pack<T>(g);
    asm volatile("st.global.v2.u32 [%0], {%1, %2};" ::"l"(p), "r"(q.x), "r"(q.y) : "memory");
  }
}

template <typename T> __device__ __forceinline__ V8 expand(const uint4 (&q)[kWords<T>]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < kWords<T>; ++i) unpack<T>(q[i], f + i * (16 / sizeof(T)));
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = pair(f[2 * i], f[2 * i + 1]);
  return r;
}
template <typename T> __device__ __forceinline__ void put8(T* p, const V8& r) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(r.v[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
  for (int i = 0; i < kWords<T>; ++i) st_v4(p + i * (16 / sizeof(T)), pack<T>(f + i * (16 / sizeof(T))));
}
// Eight values of a float32 parameter, or `none`; of the first `cols` columns where rows are ragged.
template <bool RAGGED> __device__ __forceinline__ V8 param8(const float* p, int64_t c, int cols, float none) {
  V8 r;
  r.fill(none);
  if (!p || cols == 0) return r;
  if (RAGGED && (cols < kColumns || !on16(p + c))) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < cols ? __ldg(p + c + i) : none;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = pair(f[2 * i], f[2 * i + 1]);
  } else {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p + c)), b = __ldg(reinterpret_cast<const float4*>(p + c) + 1);
    r.v[0] = pair(a.x, a.y);
    r.v[1] = pair(a.z, a.w);
    r.v[2] = pair(b.x, b.y);
    r.v[3] = pair(b.z, b.w);
  }
  return r;
}

// ------------------------------------------------------------- async copies
__device__ __forceinline__ uint32_t shared_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int K> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(K) : "memory"); }

// ------------------------------------------------------------------- sums
constexpr int log2_of(int k) { return k <= 1 ? 0 : 1 + log2_of(k / 2); }

// Warp-wide sums of K values (a power of two up to 32): lane l ends with the
// sum of value l >> (5 - log2 K) in v[0].
template <int K, int O = 16> __device__ __forceinline__ void warp_fold(float* v, int lane) {
  if constexpr (O > 0) {
    if constexpr (K > 1) {
      tr_step<K>(v, lane, O);
      warp_fold<K / 2, O / 2>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(kFull, v[0], O);
      warp_fold<1, O / 2>(v, lane);
    }
  }
}
template <int K> __device__ __forceinline__ void fold_to(float* v, int lane, float* dst) {
  warp_fold<K>(v, lane);
  constexpr int shift = 5 - log2_of(K);
  if ((lane & ((1 << shift) - 1)) == 0) dst[lane >> shift] = v[0];
}

// Where a thread stands: its group, its warp in it, its columns.
struct Place {
  int W, group, warp, lane, tid;
  int64_t d0;
  bool live;  // owns columns of the row
  int cols, warp_cols;  // how many: of the thread's first chunk, and of its warp's
  __device__ __forceinline__ Place(int warps, int64_t D) {
    W = warps;
    lane = threadIdx.x & 31;
    const int w = threadIdx.x >> 5;
    group = W == 1 ? w : 0;
    warp = W == 1 ? 0 : w;
    tid = warp * 32 + lane;
    d0 = static_cast<int64_t>(tid) * kColumns;
    live = d0 < D;
    const int64_t w0 = static_cast<int64_t>(warp) * 256;
    cols = !live ? 0 : D - d0 < kColumns ? static_cast<int>(D - d0) : kColumns;
    warp_cols = D <= w0 ? 0 : D - w0 < 256 ? static_cast<int>(D - w0) : 256;
  }
  __device__ __forceinline__ void sync() const {
    if (W == 1)
      __syncwarp();
    else
      __syncthreads();
  }
  __device__ __forceinline__ int64_t first() const {
    return W == 1 ? static_cast<int64_t>(blockIdx.x) * kSmallGroups + group : blockIdx.x;
  }
  __device__ __forceinline__ int64_t stride() const {
    return W == 1 ? static_cast<int64_t>(gridDim.x) * kSmallGroups : gridDim.x;
  }
  __device__ __forceinline__ int slot() const { return threadIdx.x >> 5; }  // this warp's row of a shared buffer
  __device__ __forceinline__ int slot0() const { return W == 1 ? group : 0; }
};

// Chunks of eight columns that a thread owns, 32 W apart.
__device__ __forceinline__ int owned_chunks(const Place& p, int64_t D) {
  const int total = static_cast<int>((D + kColumns - 1) / kColumns), per = 32 * p.W;
  return p.tid < total ? (total - p.tid + per - 1) / per : 0;
}

// Mean and 1 / root of the group's values: u[c][k] of each chunk c that the
// thread owns (`chunks` of them) and each block k < m; columns that do not exist
// hold 0. `red` is one buffer, a float4 a warp; one barrier where W > 1, none
// where W = 1. The variance of a LayerNorm is merged from (count, mean, sum of
// squared deviations) triples pair by pair, which loses nothing where the mean
// is large against the deviations.
template <bool RAGGED, int CH, int M, int MAXW>
__device__ __forceinline__ void group_stats(const Place& p, const V8 (&u)[CH][M], int chunks, int m, int norm, float eps,
                                            float inv, float4 (&red)[MAXW], float& mean, float& rstd) {
  mean = 0.f;
  if (norm == HC_NORM_RMS) {
    f2 s2 = both(0.f);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int k = 0; k < M; ++k) {
        if (M > 2 && k >= m) break;  // three blocks of four: 0 x inf in the last one is not theirs
#pragma unroll
        for (int i = 0; i < 4; ++i) s2 = fma2(u[c][k].v[i], u[c][k].v[i], s2);
      }
    float s = fold2(s2);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
    if (p.W > 1) {
      if (p.lane == 0) red[p.slot()].x = s;
      p.sync();
      s = 0.f;
      for (int w = 0; w < p.W; ++w) s += red[w].x;
    }
    rstd = rsqrtf(fmaf(s, inv, eps));
    return;
  }
  float c = static_cast<float>((RAGGED ? p.cols : 8 * chunks) * m), mu = 0.f, m2 = 0.f;
  if (chunks > 0) {
    f2 s2 = both(0.f);
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int k = 0; k < M; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) s2 = add2(u[j][k].v[i], s2);
    mu = fold2(s2) / c;
    const f2 less = both(-mu);
    f2 q2 = both(0.f);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if (j >= chunks) break;
#pragma unroll
      for (int k = 0; k < M; ++k) {
        if (k >= m) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f2 d = add2(u[j][k].v[i], less);
          if (RAGGED && 2 * i + 2 > p.cols) {
            float lo, hi;
            split(d, lo, hi);
            d = pair(2 * i < p.cols ? lo : 0.f, 0.f);
          }
          q2 = fma2(d, d, q2);
        }
      }
    }
    m2 = fold2(q2);
  }
  auto merge = [&](float c2, float mu2, float m22) {
    const float n = c + c2;
    if (n > 0.f) {
      const float d = mu2 - mu, share = __fdividef(c2, n);
      mu = fmaf(d, share, mu);
      m2 += m22 + d * d * c * share;
      c = n;
    }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float c2 = __shfl_xor_sync(kFull, c, o), mu2 = __shfl_xor_sync(kFull, mu, o),
                m22 = __shfl_xor_sync(kFull, m2, o);
    // both partners take the pair in the same order, so that every lane gets the same bits
    if (p.lane & o) {
      const float c1 = c, mu1 = mu, m21 = m2;
      c = c2; mu = mu2; m2 = m22;
      merge(c1, mu1, m21);
    } else {
      merge(c2, mu2, m22);
    }
  }
  if (p.W > 1) {
    if (p.lane == 0) red[p.slot()] = make_float4(c, mu, m2, 0.f);
    p.sync();
    c = mu = m2 = 0.f;
    for (int w = 0; w < p.W; ++w) {
      const float4 r = red[w];
      merge(r.x, r.y, r.z);
    }
  }
  mean = mu;
  rstd = rsqrtf(fmaf(m2, inv, eps));
}

// ------------------------------------------------------ the token's rows
// A thread's words of ROWS rows of its CH chunks, at
// [warp][chunk][row][word][lane]. A row's lanes lie side by side (a warp's
// copies to scattered words took a quarter more time), and a row ends with 16
// bytes of padding, so that the same lane's words of eight rows lie in
// different banks (warp_gram). All of a thread's addresses are one register and
// a constant.
//
// RAGGED: rows begin where they like and end inside a chunk (one chunk a
// thread). They travel in 4-byte copies; of 16-bit values the words that hold
// them, four or, where the first begins inside one, five, the fifth behind the
// lanes' others, and are shifted when they are read. Outputs are put together
// in STAGE rows a warp, which it then stores side by side.
constexpr int kRowPitch = 32 * 16 + 16;
template <typename T, bool RAGGED> constexpr int kPitchOf = kRowPitch + (RAGGED && sizeof(T) == 2 ? 128 : 0);
template <typename T, int ROWS, int CH, bool RAGGED = false, int STAGE = 0> struct Rows {
  static constexpr int kPitch = kPitchOf<T, RAGGED>, kStageRow = 256 * sizeof(T);
  static_assert(!RAGGED || (CH == 1 && ROWS <= 32));
  uint8_t* mem;
  int base, cols;
  mutable uint32_t inside;  // bit i: row i's first value is the second of its word
  __device__ __forceinline__ Rows(uint8_t* smem, const Place& p)
      : mem(smem), base((threadIdx.x >> 5) * (CH * ROWS * kWords<T> * kPitch) + (threadIdx.x & 31) * 16), cols(p.cols), inside(0) {
    for (int i = 0; i < CH * ROWS * kWords<T>; ++i)
      *reinterpret_cast<uint4*>(mem + base + i * kPitch) = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ int at(int c, int row) const { return base + (c * ROWS + row) * kWords<T> * kPitch; }
  __device__ __forceinline__ int fifth(int row) const { return at(0, row) + kRowPitch - static_cast<int>(threadIdx.x & 31) * 12; }
  __device__ __forceinline__ int stage_base() const { return static_cast<int>(blockDim.x >> 5) * (CH * ROWS * kWords<T> * kPitch); }
  __device__ __forceinline__ int bytes() const {
    return stage_base() + (RAGGED ? static_cast<int>(blockDim.x >> 5) * STAGE * kStageRow : 0);
  }
  __device__ __forceinline__ void fetch(int c, int row, const T* src) const {
    const uint32_t dst = shared_addr(mem) + at(c, row);
    if constexpr (!RAGGED) {
#pragma unroll
      for (int i = 0; i < kWords<T>; ++i) copy16(dst + i * kPitch, src + i * (16 / sizeof(T)));
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < cols) copy4(dst + (i >> 2) * kPitch + (i & 3) * 4, src + i);
    } else {
      const uint32_t in = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src) >> 1) & 1u;
      inside = (inside & ~(1u << row)) | in << row;
      const T* word = src - in;
      const int count = cols + static_cast<int>(in);  // values from the first word's beginning on
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * i < count) copy4(dst + 4 * i, word + 2 * i);
      if (8 < count) copy4(shared_addr(mem) + fifth(row), word + 8);
    }
  }
  // Rows row .. row + K - 1 of a chunk, of which the first `count` exist, D elements apart.
  template <int K> __device__ __forceinline__ void fetch_rows(int c, int row, const T* src, int count, int64_t D) const {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (j < count) fetch(c, row + j, src);
      src += D;
    }
  }
  // Two words of 16-bit values of which the first is value `first` of the row; `next` is the word behind them.
  __device__ __forceinline__ uint2 settle(uint2 q, uint32_t next, int row, int first) const {
    if (inside >> row & 1u) q = make_uint2(__funnelshift_r(q.x, q.y, 16), __funnelshift_r(q.y, next, 16));
    const int left = cols - first;
    if (left < 4) {
      q.x = left >= 2 ? q.x : left == 1 ? q.x & 0xffffu : 0u;
      q.y = left == 3 ? q.y & 0xffffu : 0u;
    }
    return q;
  }
  __device__ __forceinline__ V4 half(int c, int row, int h) const {  // columns 4 h .. 4 h + 3
    float f[8];
    if constexpr (kWords<T> == 2) {
      unpack<T>(*reinterpret_cast<const uint4*>(mem + at(c, row) + h * kPitch), f);
    } else {
      uint2 q = *reinterpret_cast<const uint2*>(mem + at(c, row) + h * 8);
      if constexpr (RAGGED)
        q = settle(q, *reinterpret_cast<const uint32_t*>(mem + (h ? fifth(row) : at(c, row) + 8)), row, 4 * h);
      unpack<T>(make_uint4(q.x, q.y, 0u, 0u), f);
    }
    return V4{{pair(f[0], f[1]), pair(f[2], f[3])}};
  }
  __device__ __forceinline__ V8 get(int c, int row) const {
    uint4 q[kWords<T>];
#pragma unroll
    for (int i = 0; i < kWords<T>; ++i) q[i] = *reinterpret_cast<const uint4*>(mem + at(c, row) + i * kPitch);
    if constexpr (RAGGED && kWords<T> == 1) {
      const uint2 a = settle(make_uint2(q[0].x, q[0].y), q[0].z, row, 0);
      const uint2 b = settle(make_uint2(q[0].z, q[0].w), *reinterpret_cast<const uint32_t*>(mem + fifth(row)), row, 4);
      q[0] = make_uint4(a.x, a.y, b.x, b.y);
    }
    return expand<T>(q);
  }
  // Ragged outputs: columns into a staged row, then `count` of the staged rows, D elements apart in memory, from the
  // thread's column of the first on.
  __device__ __forceinline__ T* staged(int row) const {
    return reinterpret_cast<T*>(mem + stage_base() + ((threadIdx.x >> 5) * STAGE + row) * kStageRow);
  }
  __device__ __forceinline__ void stage8(int row, const V8& v) const {
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) split(v.v[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < kWords<T>; ++i)
      *reinterpret_cast<uint4*>(staged(row) + (threadIdx.x & 31) * 8 + i * (16 / sizeof(T))) = pack<T>(f + i * (16 / sizeof(T)));
  }
  __device__ __forceinline__ void stage4(int row, int h, const V4& v) const {
    float f[8] = {};
    split(v.v[0], f[0], f[1]);
    split(v.v[1], f[2], f[3]);
    const uint4 q = pack<T>(f);
    T* to = staged(row) + (threadIdx.x & 31) * 8 + 4 * h;
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<uint4*>(to) = q;
    else
      *reinterpret_cast<uint2*>(to) = make_uint2(q.x, q.y);
  }
  template <int K> __device__ __forceinline__ void unstage(T* dst, int count, int64_t D, int warp_cols) const {
    const int lane = threadIdx.x & 31;
    dst -= 8 * lane;
    __syncwarp();
#pragma unroll
    for (int r = 0; r < K; ++r) {
      if (r < count) {
        const T* from = staged(r);
#pragma unroll
        for (int e = 0; e < 256; e += 32)
          if (e + lane < warp_cols) dst[e + lane] = from[e + lane];
      }
      dst += D;
    }
    __syncwarp();
  }
};
__device__ __forceinline__ float one(f2 v) {
  float a, b;
  split(v, a, b);
  return a;
}

// The loop over a group's tokens. all(t) issues the copies of a token's rows,
// small(t, slot) those of its small matrices. work(t, next, slot, parity) does
// token t, whose rows have arrived and whose small matrices have since the
// barrier before; between two tokens' uses of a buffer, and between a token's
// wait for copies and another thread's use of them, it passes a barrier of the
// group (of a warp for W = 1, where a shuffle is none). Where next < T it asks
// for that token's rows, each as soon as it has read this token's.
template <typename All, typename Small, typename Start, typename Work>
__device__ __forceinline__ void walk_tokens(const Place& p, int64_t T, All all, Small small, Start start, Work work) {
  const int64_t t0 = p.first(), step = p.stride();
  if (t0 >= T) return;
  p.sync();  // the zeros of the rows and of the small matrices
  small(t0, 0);
  copy_commit();
  all(t0);
  if (t0 + step < T) small(t0 + step, 1);
  copy_commit();
  copy_wait<1>();
  p.sync();
  start(0);
  int i = 0;
  for (int64_t t = t0; t < T; t += step, ++i) {
    if (t + 2 * step < T) small(t + 2 * step, (i + 2) & (kSmallSlots - 1));
    copy_commit();
    copy_wait<1>();
    work(t, t + step, i & (kSmallSlots - 1), i & 1);
    copy_commit();
  }
}

// A group's small entries of a token, dealt to its threads once: R rounds of
// 32 W entries, each from src + t stride to entry dst of a slot.
template <int R> struct SmallCopies {
  const float* src[R];
  int stride[R], dst[R];
  template <typename Decode> __device__ __forceinline__ SmallCopies(const Place& p, int total, Decode decode) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int id = p.tid + r * 32 * p.W;
      src[r] = nullptr;
      stride[r] = 0;
      dst[r] = -1;
      if (id < total) decode(id, src[r], stride[r], dst[r]);
    }
  }
  __device__ __forceinline__ void fetch(f2* slot, int64_t t) const {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (dst[r] >= 0) {
        const float* s = src[r] + t * stride[r];
        const uint32_t d = shared_addr(slot + dst[r]);
        copy4(d, s);
        copy4(d + 4, s);
      }
  }
};

// Where the sums of a token's small gradients go, dealt to threads likewise;
// nullptr where nobody wants one.
template <int R> struct SmallGrads {
  float* out[R];
  int stride[R];
  template <typename Decode> __device__ __forceinline__ SmallGrads(const Place& p, int total, Decode decode) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int id = p.tid + r * 32 * p.W;
      out[r] = nullptr;
      stride[r] = 0;
      if (id < total) decode(id, out[r], stride[r]);
    }
  }
  // The W warps' sums of entry id, which lie `per` floats apart.
  template <typename Sums> __device__ __forceinline__ void store(const Place& p, int64_t t, Sums sums) const {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (out[r]) {
        const int id = p.tid + r * 32 * p.W;
        float s = 0.f;
        for (int q = 0; q < p.W; ++q) s += sums(q, id);
        out[r][t * stride[r]] = s;
      }
  }
};

// The groups' sums of the [m D] parameters' gradients; with several groups a
// CTA each adds its own row.
template <bool RAGGED, int CH, int M>
__device__ __forceinline__ void store_param_sums(const NormArgs& a, const Place& p, int chunks, const V8 (&A)[CH][M],
                                                 const V8 (&B)[CH][M]) {
  if (!a.partial) return;
  const int64_t E = a.D * a.m;
  const int64_t row = p.W == 1 ? static_cast<int64_t>(blockIdx.x) * kSmallGroups + p.group : blockIdx.x;
  float* dst = a.partial + row * 2 * E + p.d0;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (c >= chunks) break;
#pragma unroll
    for (int k = 0; k < M; ++k) {
      if (k >= a.m) break;
      if constexpr (RAGGED) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float s[2][2];
          split(A[c][k].v[i >> 1], s[0][0], s[0][1]);
          split(B[c][k].v[i >> 1], s[1][0], s[1][1]);
          if (i < p.cols) {
            dst[k * a.D + i] = s[0][i & 1];
            dst[E + k * a.D + i] = s[1][i & 1];
          }
        }
        continue;
      }
      put8<float>(dst + k * a.D + c * 256 * p.W, A[c][k]);
      put8<float>(dst + E + k * a.D + c * 256 * p.W, B[c][k]);
    }
  }
}

// The group's small matrices, all slots, to zero.
template <int K> __device__ __forceinline__ void clear_small(const Place& p, f2 (&s)[kSmallSlots][K]) {
  for (int i = p.tid; i < kSmallSlots * K; i += 32 * p.W) (&s[0][0])[i] = 0ull;
}

// A group's part of dynamic shared memory, behind the rows.
template <int N, int M> struct ReadMemory {
  static constexpr int kEntries = N * M + 2;
  alignas(16) f2 R[kSmallSlots][kEntries];  // R [N][M], and for the backward mean and 1 / root
};
template <typename Memory>
__device__ __forceinline__ Memory& group_memory(uint8_t* dyn, const Place& p, int row_bytes) {
  return reinterpret_cast<Memory*>(dyn + row_bytes)[p.group];
}

// ------------------------------------------------------------------- read
template <typename T, int N, int M, int CH, bool RAGGED, bool WIDE>
__global__ void __launch_bounds__(norm_fwd_threads(N, M, CH, sizeof(T), WIDE))
    read_norm_fwd_kernel(const __grid_constant__ NormArgs a, int warps) {
  constexpr int MAXW = norm_fwd_threads(N, M, CH, sizeof(T), WIDE) / 32;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ float4 red[2][MAXW];
  const Place p(warps, a.D);
  const int n = a.n, m = a.m, chunks = owned_chunks(p, a.D), step = 256 * p.W;
  const int64_t D = a.D, E = D * m;
  const float inv = 1.f / static_cast<float>(E);
  const Rows<T, N, CH, RAGGED, M> rows(dyn, p);
  auto& sR = group_memory<ReadMemory<N, M>>(dyn, p, rows.bytes()).R;
  clear_small(p, sR);
  const SmallCopies<(N * M + 31) / 32> copies(p, n * m, [&](int id, const float*& src, int& stride, int& dst) {
    src = a.R + id;
    stride = n * m;
    dst = id % n * M + id / n;
  });
  auto fetch = [&](int64_t t, int c) {
    if (c >= chunks) return;
    const T* x = static_cast<const T*>(a.x) + t * n * D + p.d0 + c * step;
    rows.template fetch_rows<N>(c, 0, x, n, D);
  };
  walk_tokens(
      p, a.T,
      [&](int64_t t) {
#pragma unroll
        for (int c = 0; c < CH; ++c) fetch(t, c);
      },
      [&](int64_t t, int slot) { copies.fetch(sR[slot], t); }, [](int) {},
      [&](int64_t t, int64_t next, int slot, int parity) {
        const f2* R = sR[slot];
        V8 u[CH][M];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
          for (int k = 0; k < M; ++k) u[c][k].fill(0.f);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const V8 x = rows.get(c, j);
#pragma unroll
            for (int k = 0; k < M; ++k) axpy(R[j * M + k], x, u[c][k]);
          }
          if (next < a.T) fetch(next, c);
        }
        float mean, rstd;
        group_stats<RAGGED, CH, M, MAXW>(p, u, chunks, m, a.norm, a.eps, inv, red[parity], mean, rstd);
        if (a.stats && p.tid == 0) *reinterpret_cast<float2*>(a.stats + 2 * t) = make_float2(mean, rstd);
        T* y = static_cast<T*>(a.out) + t * E + p.d0;
        const f2 less = both(-mean), r2 = both(rstd);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          if (!RAGGED && c >= chunks) break;
          const int cols = RAGGED ? p.cols : kColumns;
#pragma unroll
          for (int k = 0; k < M; ++k) {
            if (k >= m) break;
            const int64_t col = k * D + c * step;
            const V8 w = param8<RAGGED>(a.weight, col + p.d0, cols, 1.f), b = param8<RAGGED>(a.bias, col + p.d0, cols, 0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[c][k].v[i] = fma2(mul2(add2(u[c][k].v[i], less), r2), w.v[i], b.v[i]);
            if constexpr (RAGGED)
              rows.stage8(k, u[c][k]);
            else
              put8<T>(y + col, u[c][k]);
          }
        }
        if constexpr (RAGGED) rows.template unstage<M>(y, m, D, p.warp_cols);
        __syncwarp();
      });
}

template <typename T, int N, int M, int CH, bool RAGGED, bool WIDE>
__global__ void __launch_bounds__(norm_bwd_threads(N, M, sizeof(T), WIDE))
    read_norm_bwd_kernel(const __grid_constant__ NormArgs a, int warps) {
  static_assert(CH == 1, "the backward's threads own one chunk");
  constexpr int MAXW = norm_bwd_threads(N, M, sizeof(T), WIDE) / 32, G = N * M;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ float red[2][MAXW][2], gram[2][MAXW][G];
  static_assert(kNormSmemMax + sizeof(red) + sizeof(gram) <= kCtaSmemMax);
  const Place p(warps, a.D);
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  const float inv = 1.f / static_cast<float>(E);
  const Rows<T, N + M, 1, RAGGED, N> rows(dyn, p);
  auto& sR = group_memory<ReadMemory<N, M>>(dyn, p, rows.bytes()).R;
  clear_small(p, sR);
  const SmallCopies<(G + 33) / 32> copies(p, n * m + 2, [&](int id, const float*& src, int& stride, int& dst) {
    const bool st = id >= n * m;
    src = st ? a.stats + (id - n * m) : a.R + id;
    stride = st ? 2 : n * m;
    dst = st ? G + id - n * m : id % n * M + id / n;
  });
  const SmallGrads<(G + 31) / 32> grads(p, G, [&](int id, float*& out, int& stride) {  // [stream][block]
    const int j = id / M, k = id % M;
    if (a.grad_R && j < n && k < m) out = a.grad_R + k * n + j;
    stride = n * m;
  });
  V8 A[1][M], B[1][M];
#pragma unroll
  for (int k = 0; k < M; ++k) {
    A[0][k].fill(0.f);
    B[0][k].fill(0.f);
  }
  int64_t last = -1;
  int last_parity = 0;
  // grad_R of the last token, whose warps' sums lie in the other buffer
  auto flush = [&] {
    if (last >= 0) grads.store(p, last, [&](int q, int id) { return gram[last_parity][p.slot0() + q][id]; });
  };
  auto fetch_x = [&](int64_t t) {
    if (!p.live) return;
    const T* x = static_cast<const T*>(a.x) + t * n * D + p.d0;
    rows.template fetch_rows<N>(0, 0, x, n, D);
  };
  auto fetch_g = [&](int64_t t) {
    if (!p.live) return;
    const T* g = static_cast<const T*>(a.g) + t * E + p.d0;
    rows.template fetch_rows<M>(0, N, g, m, D);
  };
  walk_tokens(
      p, a.T,
      [&](int64_t t) {
        fetch_x(t);
        fetch_g(t);
      },
      [&](int64_t t, int slot) { copies.fetch(sR[slot], t); }, [](int) {},
      [&](int64_t t, int64_t next, int slot, int parity) {
        const f2* R = sR[slot];
        const f2 less = both(-one(R[G])), r2 = R[G + 1];
        f2 s1 = both(0.f), s2 = both(0.f);
        V8 u[M], q[M];
#pragma unroll
        for (int k = 0; k < M; ++k) u[k].fill(0.f);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const V8 x = rows.get(0, j);
#pragma unroll
          for (int k = 0; k < M; ++k) axpy(R[j * M + k], x, u[k]);
        }
#pragma unroll
        for (int k = 0; k < M; ++k) {
          const V8 g = rows.get(0, N + k);
          const V8 w = param8<RAGGED>(a.weight, k * D + p.d0, k < m ? (RAGGED ? p.cols : p.live ? kColumns : 0) : 0, 1.f);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[k].v[i] = mul2(add2(u[k].v[i], less), r2);  // xhat
            q[k].v[i] = mul2(g.v[i], w.v[i]);
            s1 = fma2(q[k].v[i], u[k].v[i], s1);
            s2 = add2(q[k].v[i], s2);
            A[0][k].v[i] = fma2(g.v[i], u[k].v[i], A[0][k].v[i]);
            B[0][k].v[i] = add2(g.v[i], B[0][k].v[i]);
          }
        }
        if (next < a.T) fetch_g(next);
        float s[2] = {fold2(s1), fold2(s2)};  // g is 0 where there are no columns
        fold_to<2>(s, p.lane, red[parity][p.slot()]);
        p.sync();
        flush();
        float c1 = 0.f, c2 = 0.f;
        for (int i = 0; i < p.W; ++i) {
          c1 += red[parity][p.slot0() + i][0];
          c2 += red[parity][p.slot0() + i][1];
        }
        const f2 k1 = both(-c1 * inv), k2 = both(a.norm == HC_NORM_LAYER ? -c2 * inv : 0.f);
#pragma unroll
        for (int k = 0; k < M; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) u[k].v[i] = mul2(r2, fma2(u[k].v[i], k1, add2(q[k].v[i], k2)));  // du
        float acc[G];
        T* gx = static_cast<T*>(a.grad_x) + t * n * D + p.d0;
        const bool store = a.grad_x && p.live;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          V8 r;
          r.fill(0.f);
#pragma unroll
          for (int k = 0; k < M; ++k) axpy(R[j * M + k], u[k], r);
          if constexpr (RAGGED) {
            rows.stage8(j, r);
          } else {
            if (store && j < n) put8<T>(gx, r);
            gx += D;
          }
          const V8 x = rows.get(0, j);  // 0 where there are no columns
#pragma unroll
          for (int k = 0; k < M; ++k) acc[j * M + k] = dot(u[k], x);
        }
        if constexpr (RAGGED) {
          if (a.grad_x) rows.template unstage<N>(gx, n, D, p.warp_cols);
        }
        if (next < a.T) fetch_x(next);
        fold_to<G>(acc, p.lane, gram[parity][p.slot()]);
        last = t;
        last_parity = parity;
      });
  p.sync();
  flush();
  store_param_sums<RAGGED, 1, M>(a, p, p.live ? 1 : 0, A, B);
}

// -------------------------------------------------------------- mix-write
// All ones where one of eight columns is kept, the first a multiple of 8.
__device__ __forceinline__ void keep8(const DropArgs& d, const DropKey& key, uint64_t element, uint32_t (&mask)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 w = philox4(key, (element >> 2) + h);
    mask[4 * h] = w.x > d.below ? 0xffffffffu : 0u;
    mask[4 * h + 1] = w.y > d.below ? 0xffffffffu : 0u;
    mask[4 * h + 2] = w.z > d.below ? 0xffffffffu : 0u;
    mask[4 * h + 3] = w.w > d.below ? 0xffffffffu : 0u;
  }
}
// v / (1 - p) where kept, else 0 whatever v is.
__device__ __forceinline__ void keep_mul(V8& v, float scale, const uint32_t (&mask)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x, y;
    split(mul2(v.v[i], both(scale)), x, y);
    v.v[i] = pair(__uint_as_float(__float_as_uint(x) & mask[2 * i]), __uint_as_float(__float_as_uint(y) & mask[2 * i + 1]));
  }
}
// The same of eight columns that begin inside a block of four.
__device__ __forceinline__ void keep_ragged(const DropArgs& d, const DropKey& key, uint64_t element, uint32_t (&mask)[8]) {
  uint32_t bits = 0;
#pragma unroll
  for (int h = 0; h < 3; ++h) {
    const uint4 w = philox4(key, (element >> 2) + h);
    bits |= ((w.x > d.below ? 1u : 0u) | (w.y > d.below ? 2u : 0u) | (w.z > d.below ? 4u : 0u) | (w.w > d.below ? 8u : 0u)) << (4 * h);
  }
  bits >>= static_cast<uint32_t>(element) & 3u;
#pragma unroll
  for (int i = 0; i < 8; ++i) mask[i] = bits >> i & 1u ? 0xffffffffu : 0u;
}
// act(a) of a gate, and act'(a).
__device__ __forceinline__ void gate8(int act, const V8& a, V8& val, V8& der) {
  if (act == HC_ACT_SIGMOID) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x, y;
      split(a.v[i], x, y);
      x = __fdividef(1.f, 1.f + __expf(-x));
      y = __fdividef(1.f, 1.f + __expf(-y));
      val.v[i] = pair(x, y);
      der.v[i] = fma2(val.v[i], pair(-x, -y), val.v[i]);  // s - s^2
    }
  } else {
    val = a;
    der.fill(1.f);
  }
}

// A token's small matrices in shared memory: H [column][row] (TRANSPOSED) or
// [row][column], W [N][M], v, then mean and 1 / root.
template <int N, int M, bool TRANSPOSED> struct Small {
  static constexpr int kW = N * N, kV = kW + N * M, kStats = kV + N, kEntries = (kStats + 3) / 2 * 2;
  static constexpr int kRounds = (kStats + 2 + 31) / 32;
  __device__ static __forceinline__ int h(int r, int c) { return TRANSPOSED ? c * N + r : r * N + c; }
  __device__ static __forceinline__ SmallCopies<kRounds> copies(const NormArgs& a, const Place& p, bool stats) {
    const int n = a.n, m = a.m, w0 = n * n, v0 = w0 + n * m, s0 = a.v ? v0 + n : v0;
    return SmallCopies<kRounds>(p, stats ? s0 + 2 : s0, [&](int id, const float*& src, int& stride, int& dst) {
      if (id < w0) {
        src = a.H + id;
        stride = w0;
        dst = h(id / n, id % n);
      } else if (id < v0) {
        src = a.W + (id - w0);
        stride = n * m;
        dst = kW + (id - w0) / m * M + (id - w0) % m;
      } else if (id < s0) {
        src = a.v + (id - v0);
        stride = n;
        dst = kV + id - v0;
      } else {
        src = a.stats + (id - s0);
        stride = 2;
        dst = kStats + id - s0;
      }
    });
  }
  // H + (v - H v) v^T, by the group's first threads.
  __device__ static __forceinline__ void project(const Place& p, const f2* s, f2* dst) {
    for (int i = p.tid; i < N * N; i += 32 * p.W) {
      const int r = i / N, c = i % N;
      float q = one(s[kV + r]);
      for (int k = 0; k < N; ++k) q -= one(s[h(r, k)]) * one(s[kV + k]);
      dst[h(r, c)] = both(one(s[h(r, c)]) + q * one(s[kV + c]));
    }
  }
  // grad_H and grad_v of the token from G = dL/d(H + (v - H v) v^T), [row][column].
  __device__ static __forceinline__ void grads(const NormArgs& a, const Place& p, const f2* s, const float* G, int64_t t) {
    const int n = a.n;
    for (int i = p.tid; i < N * N; i += 32 * p.W) {
      const int r = i / N, c = i % N;
      if (r >= n || c >= n || !a.grad_H) continue;
      float dq = 0.f;
      for (int j = 0; j < n; ++j) dq += G[r * N + j] * one(s[kV + j]);
      a.grad_H[t * n * n + r * n + c] = G[i] - dq * one(s[kV + c]);
    }
    if (a.grad_v && p.tid < n) {
      const int c = p.tid;
      float g = 0.f;
      for (int r = 0; r < n; ++r) {
        float q = one(s[kV + r]), dq = 0.f;
        for (int j = 0; j < n; ++j) {
          q -= one(s[h(r, j)]) * one(s[kV + j]);
          dq += G[r * N + j] * one(s[kV + j]);
        }
        g += q * G[r * N + c] + (r == c ? dq : 0.f) - one(s[h(r, c)]) * dq;
      }
      a.grad_v[t * n + c] = g;
    }
  }
};

template <int N, int M> struct WriteMemory {
  alignas(16) f2 small[kSmallSlots][Small<N, M, true>::kEntries];
  alignas(16) f2 mixed[2][N * N];  // H + (v - H v) v^T of this token and the next
  float G[N * N];
};

// g x^T of a warp's 256 columns by mma.m16n8k16 (products of 16-bit values are
// exact in float32): a lane's 16 bytes of a row are a row of an 8 x 8 tile, so
// that the tiles g and x of two lanes' columns are one ldmatrix, and the sums
// over the lanes come out of the products instead of exchanges. Rows past N
// repeat the others and are not stored; dst is [column][row].
template <typename T, int N, typename R>
__device__ __forceinline__ void warp_gram(const R& rows, float (&c)[4]) {
  const int lane = threadIdx.x & 31;
  // matrices 0, 1: rows g of an even and an odd lane's columns; 2, 3: rows x
  const uint32_t addr = shared_addr(rows.mem) + rows.at(0, 0) - lane * 16 + ((lane >> 3) & 1) * 16 +
                        static_cast<uint32_t>(((lane >> 4) * N + (lane & 7) % N) * kRowPitch);
#pragma unroll
  for (int l = 0; l < 32; l += 2) {
    uint32_t g0, g1, x0, x1;
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(g0), "=r"(g1), "=r"(x0), "=r"(x1)
                 : "r"(addr + l * 16)
                 : "memory");
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      asm volatile(
          "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(g0), "r"(0), "r"(g1), "r"(0), "r"(x0), "r"(x1));
    else
      asm volatile(
          "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(g0), "r"(0), "r"(g1), "r"(0), "r"(x0), "r"(x1));
  }
}
template <int N> __device__ __forceinline__ void store_gram(const float (&c)[4], int lane, float* dst) {
  const int r = lane >> 2, col = (lane & 3) * 2;  // c[0], c[1]: row r, columns col and col + 1
  if (r < N) {
    if (col < N) dst[col * N + r] = c[0];
    if (col + 1 < N) dst[(col + 1) * N + r] = c[1];
  }
}

// scale * weight and scale * bias of eight columns from c on.
template <bool RAGGED>
__device__ __forceinline__ void scaled_params(const NormArgs& a, int64_t c, int cols, V8& ws, V8& bs) {
  const V8 sc = param8<RAGGED>(a.scale, c, cols, 1.f);
  ws = param8<RAGGED>(a.weight, c, cols, 1.f);
  bs = param8<RAGGED>(a.bias, c, cols, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ws.v[i] = mul2(ws.v[i], sc.v[i]);
    bs.v[i] = mul2(bs.v[i], sc.v[i]);
  }
}

template <typename T, int N, int M, int CH, bool RAGGED, bool WIDE>
__global__ void __launch_bounds__(norm_fwd_threads(N, M, CH, sizeof(T), WIDE))
    write_norm_fwd_kernel(const __grid_constant__ NormArgs a, int warps) {
  constexpr int MAXW = norm_fwd_threads(N, M, CH, sizeof(T), WIDE) / 32;
  using S = Small<N, M, false>;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ float4 red[2][MAXW];
  const Place p(warps, a.D);
  const int n = a.n, m = a.m, chunks = owned_chunks(p, a.D), step = 256 * p.W;
  const int64_t D = a.D, E = D * m;
  const float inv = 1.f / static_cast<float>(E);
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  const Rows<T, N + 2 * M, CH, RAGGED, N> rows(dyn, p);  // x, f, gate
  auto& memory = group_memory<WriteMemory<N, M>>(dyn, p, rows.bytes());
  auto& small = memory.small;
  auto& mixed = memory.mixed;
  clear_small(p, small);
  const auto copies = S::copies(a, p, false);
  auto fetch_f = [&](int64_t t, int c) {
    if (c >= chunks) return;
    const T* f = static_cast<const T*>(a.f) + t * E + p.d0 + c * step;
    rows.template fetch_rows<M>(c, N, f, m, D);
  };
  auto fetch_rest = [&](int64_t t, int c) {  // gate and x
    if (c >= chunks) return;
    const T* x = static_cast<const T*>(a.x) + t * n * D + p.d0 + c * step;
    if (a.gate) rows.template fetch_rows<M>(c, N + M, static_cast<const T*>(a.gate) + t * E + p.d0 + c * step, m, D);
    rows.template fetch_rows<N>(c, 0, x, n, D);
  };
  walk_tokens(
      p, a.T,
      [&](int64_t t) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          fetch_f(t, c);
          fetch_rest(t, c);
        }
      },
      [&](int64_t t, int slot) { copies.fetch(small[slot], t); },
      [&](int slot) {
        if (a.v) S::project(p, small[slot], mixed[0]);
      },
      [&](int64_t t, int64_t next, int slot, int parity) {
        V8 z[CH][M];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
          for (int k = 0; k < M; ++k) z[c][k] = rows.get(c, N + k);
          if (next < a.T) fetch_f(next, c);
        }
        float mean = 0.f, rstd = 1.f;
        if (a.norm != HC_NORM_NONE) {
          group_stats<RAGGED, CH, M, MAXW>(p, z, chunks, m, a.norm, a.eps, inv, red[parity], mean, rstd);
          if (a.stats && p.tid == 0) *reinterpret_cast<float2*>(a.stats + 2 * t) = make_float2(mean, rstd);
        } else {
          p.sync();
        }
        // a group of one warp has passed no barrier in group_stats: what its lanes copied (the next token's matrices) and
        // wrote (this token's mix) is read by one another below
        if (p.W == 1) __syncwarp();
        const f2* s = small[slot];
        if (a.v) S::project(p, small[(slot + 1) & (kSmallSlots - 1)], mixed[parity ^ 1]);
        const f2* H = a.v ? mixed[parity] : s;
        const f2 less = both(-mean), r2 = both(rstd);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
          for (int k = 0; k < M; ++k) {
            if (M > 1 && k >= m) {  // a block that does not exist
              z[c][k].fill(0.f);
              continue;
            }
            const int64_t col = k * D + p.d0 + c * step;
            V8 ws, bs;
            scaled_params<RAGGED>(a, col, RAGGED ? p.cols : c < chunks ? kColumns : 0, ws, bs);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[c][k].v[i] = fma2(mul2(add2(z[c][k].v[i], less), r2), ws.v[i], bs.v[i]);
            if (a.gate) {
              V8 val, der;
              gate8(a.gate_act, rows.get(c, N + M + k), val, der);
#pragma unroll
              for (int i = 0; i < 4; ++i) z[c][k].v[i] = mul2(z[c][k].v[i], val.v[i]);
            }
            if (a.drop.on) {
              uint32_t keep[8];
              if constexpr (RAGGED)
                keep_ragged(a.drop, key, static_cast<uint64_t>(t * E + col), keep);
              else
                keep8(a.drop, key, static_cast<uint64_t>(t * E + col), keep);
              keep_mul(z[c][k], a.drop.scale, keep);
            }
          }
          T* out = static_cast<T*>(a.out) + t * n * D + p.d0 + c * step;
#pragma unroll 1  // one half's registers at a time
          for (int h = 0; h < 2; ++h) {
            V4 x[N], zh[M];
#pragma unroll
            for (int k = 0; k < M; ++k) {
              zh[k].v[0] = h ? z[c][k].v[2] : z[c][k].v[0];
              zh[k].v[1] = h ? z[c][k].v[3] : z[c][k].v[1];
            }
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = rows.half(c, j, h);
            T* dst = out + 4 * h;
#pragma unroll
            for (int i = 0; i < N; ++i) {
              V4 r{{both(0.f), both(0.f)}};
              f2 hi[N], wi[M];
              pairs<N>(H + i * N, hi);
              pairs<M>(s + S::kW + i * M, wi);
#pragma unroll
              for (int j = 0; j < N; ++j) axpy(hi[j], x[j], r);
#pragma unroll
              for (int k = 0; k < M; ++k) axpy(wi[k], zh[k], r);
              if constexpr (RAGGED) {
                rows.stage4(i, h, r);
              } else {
                if (c < chunks && i < n) put4<T>(dst, r);
                dst += D;
              }
            }
          }
          if constexpr (RAGGED) rows.template unstage<N>(out, n, D, p.warp_cols);
          if (next < a.T) fetch_rest(next, c);
        }
        __syncwarp();
      });
}

template <typename T, int N, int M, int CH, bool RAGGED, bool WIDE>
__global__ void __launch_bounds__(norm_bwd_threads(N, M, sizeof(T), WIDE))
    write_norm_bwd_kernel(const __grid_constant__ NormArgs a, int warps) {
  static_assert(CH == 1, "the backward's threads own one chunk");
  constexpr int MAXW = norm_bwd_threads(N, M, sizeof(T), WIDE) / 32;
  constexpr int GB = N * N < 32 ? N * N : 32, G = N * N + N * M;  // H's sums [column][row] by batches of GB, then W's
  using S = Small<N, M, true>;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ float red[2][MAXW][2], gram[2][MAXW][G];
  static_assert(kNormSmemMax + sizeof(red) + sizeof(gram) <= kCtaSmemMax);
  const Place p(warps, a.D);
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  const float inv = 1.f / static_cast<float>(E);
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  const Rows<T, 2 * N + 2 * M, 1, RAGGED, N> rows(dyn, p);  // g, x, f, gate
  auto& memory = group_memory<WriteMemory<N, M>>(dyn, p, rows.bytes());
  auto& small = memory.small;
  auto& mixed = memory.mixed;
  clear_small(p, small);
  const auto copies = S::copies(a, p, a.norm != HC_NORM_NONE);
  const SmallGrads<(G + 31) / 32> grads(p, G, [&](int id, float*& out, int& stride) {
    if (id < N * N) {
      const int c = id / N, r = id % N;
      if (a.grad_H && r < n && c < n) out = a.grad_H + r * n + c;
      stride = n * n;
      if (a.v) {  // first to the projection's gradients
        out = memory.G + r * N + c;
        stride = 0;
      }
    } else {
      const int r = (id - N * N) / M, k = (id - N * N) % M;
      if (a.grad_W && r < n && k < m) out = a.grad_W + r * m + k;
      stride = n * m;
    }
  });
  V8 A[1][M], B[1][M];
#pragma unroll
  for (int k = 0; k < M; ++k) {
    A[0][k].fill(0.f);
    B[0][k].fill(0.f);
  }
  // grad_H, grad_v and grad_W of the token whose warps' sums lie in gram[parity], behind the barrier that completes
  // them: the next sums to go there are those of the token after next, behind one more barrier
  auto add_sums = [&](int64_t t, int slot, int parity) {
    grads.store(p, t, [&](int q, int id) { return gram[parity][p.slot0() + q][id]; });
    if (a.v) {
      p.sync();
      S::grads(a, p, small[slot], memory.G, t);
    }
  };
  auto fetch_outer = [&](int64_t t) {  // g, x and gate
    if (!p.live) return;
    const int64_t xo = t * n * D + p.d0;
    const T *g = static_cast<const T*>(a.g) + xo, *x = static_cast<const T*>(a.x) + xo;
    rows.template fetch_rows<N>(0, 0, g, n, D);
    if (a.gate) rows.template fetch_rows<M>(0, 2 * N + M, static_cast<const T*>(a.gate) + t * E + p.d0, m, D);
    rows.template fetch_rows<N>(0, N, x, n, D);
  };
  auto fetch_f = [&](int64_t t) {
    if (!p.live) return;
    const T* f = static_cast<const T*>(a.f) + t * E + p.d0;
    rows.template fetch_rows<M>(0, 2 * N, f, m, D);
  };
  walk_tokens(
      p, a.T,
      [&](int64_t t) {
        fetch_outer(t);
        fetch_f(t);
      },
      [&](int64_t t, int slot) { copies.fetch(small[slot], t); },
      [&](int slot) {
        if (a.v) {
          S::project(p, small[slot], mixed[0]);
          p.sync();
        }
      },
      [&](int64_t t, int64_t next, int slot, int parity) {
        const f2* s = small[slot];
        const f2* H = a.v ? mixed[parity] : s;
        const f2 less = a.norm == HC_NORM_NONE ? both(0.f) : both(-one(s[S::kStats]));
        const f2 r2 = a.norm == HC_NORM_NONE ? both(1.f) : s[S::kStats + 1];
        __syncwarp();  // the other lanes' copies have arrived
        // dz, from W^T g; a column of the mix at a time, grad_x_j = sum_i Heff_ij g_i
        V8 q[M];
        T* gx = static_cast<T*>(a.grad_x) + t * n * D + p.d0;
        const bool store = a.grad_x && p.live;
#pragma unroll 1  // one half's registers at a time
        for (int h = 0; h < 2; ++h) {
          V4 g[N], d[M];
#pragma unroll
          for (int k = 0; k < M; ++k) d[k].v[0] = d[k].v[1] = both(0.f);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            g[i] = rows.half(0, i, h);
            f2 wi[M];
            pairs<M>(s + S::kW + i * M, wi);
#pragma unroll
            for (int k = 0; k < M; ++k) axpy(wi[k], g[i], d[k]);
          }
#pragma unroll
          for (int k = 0; k < M; ++k) {
            q[k].v[0] = h ? q[k].v[0] : d[k].v[0];
            q[k].v[1] = h ? q[k].v[1] : d[k].v[1];
            q[k].v[2] = d[k].v[0];  // the second half stays
            q[k].v[3] = d[k].v[1];
          }
          T* dst = gx + 4 * h;
#pragma unroll
          for (int j = 0; j < N; ++j) {
            V4 r{{both(0.f), both(0.f)}};
            f2 hj[N];
            pairs<N>(H + j * N, hj);
#pragma unroll
            for (int i = 0; i < N; ++i) axpy(hj[i], g[i], r);
            if constexpr (RAGGED) {
              rows.stage4(j, h, r);
            } else {
              if (store && j < n) put4<T>(dst, r);
              dst += D;
            }
          }
        }
        if constexpr (RAGGED) {
          if (a.grad_x) rows.template unstage<N>(gx, n, D, p.warp_cols);
        }
        if constexpr (sizeof(T) == 4 || RAGGED) {  // g x^T of float32 streams, and of rows that are shifted when they are read
          float acc[GB];
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const V8 x = rows.get(0, N + j);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[(j * N + i) % GB] = dot(rows.get(0, i), x);
            if ((j + 1) * N % GB == 0) fold_to<GB>(acc, p.lane, &gram[parity][p.slot()][(j + 1) * N - GB]);
          }
        }
        if constexpr (sizeof(T) == 2 && !RAGGED) {
          float gsum[4] = {0.f, 0.f, 0.f, 0.f};
          warp_gram<T, N>(rows, gsum);
          store_gram<N>(gsum, p.lane, gram[parity][p.slot()]);
        }
        // dropout's and the gate's backward; z
        f2 s1 = both(0.f), s2 = both(0.f);
        V8 z[M];
#pragma unroll
        for (int k = 0; k < M; ++k) {
          if (M > 1 && k >= m) {
            z[k].fill(0.f);
            continue;
          }
          const int64_t col = k * D + p.d0;
          uint32_t keep[8];
          if (a.drop.on) {
            if constexpr (RAGGED)
                keep_ragged(a.drop, key, static_cast<uint64_t>(t * E + col), keep);
              else
                keep8(a.drop, key, static_cast<uint64_t>(t * E + col), keep);
            keep_mul(q[k], a.drop.scale, keep);
          }
          V8 ws, bs, xh = rows.get(0, 2 * N + k);
          scaled_params<RAGGED>(a, col, RAGGED ? p.cols : p.live ? kColumns : 0, ws, bs);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            xh.v[i] = mul2(add2(xh.v[i], less), r2);
            z[k].v[i] = fma2(xh.v[i], ws.v[i], bs.v[i]);  // scale (weight xhat + bias)
          }
          if (a.gate) {
            V8 val, der;
            gate8(a.gate_act, rows.get(0, 2 * N + M + k), val, der);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              der.v[i] = mul2(der.v[i], mul2(q[k].v[i], z[k].v[i]));
              q[k].v[i] = mul2(q[k].v[i], val.v[i]);
              z[k].v[i] = mul2(z[k].v[i], val.v[i]);
            }
            if constexpr (RAGGED)
              rows.stage8(k, der);
            else if (a.grad_gate && p.live)
              put8<T>(static_cast<T*>(a.grad_gate) + t * E + col, der);
          }
          if (a.drop.on) keep_mul(z[k], a.drop.scale, keep);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            A[0][k].v[i] = fma2(q[k].v[i], xh.v[i], A[0][k].v[i]);
            B[0][k].v[i] = add2(q[k].v[i], B[0][k].v[i]);
            q[k].v[i] = mul2(q[k].v[i], ws.v[i]);
            s1 = fma2(q[k].v[i], xh.v[i], s1);
            s2 = add2(q[k].v[i], s2);
          }
        }
        if constexpr (RAGGED) {
          if (a.gate && a.grad_gate)
            rows.template unstage<M>(static_cast<T*>(a.grad_gate) + t * E + p.d0, m, D, p.warp_cols);
        }
        float sums[2] = {fold2(s1), fold2(s2)};  // g is 0 where there are no columns
        fold_to<2>(sums, p.lane, red[parity][p.slot()]);
        float accW[N * M];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const V8 g = rows.get(0, i);  // again: held over the block's part above it costs the registers of two warps in five
#pragma unroll
          for (int k = 0; k < M; ++k) accW[i * M + k] = dot(g, z[k]);
        }
        fold_to<N * M>(accW, p.lane, &gram[parity][p.slot()][N * N]);
        __syncwarp();  // warp_gram's reads are done before the next token's copies overwrite the rows
        if (next < a.T) fetch_outer(next);
        p.sync();
        add_sums(t, slot, parity);
        if (a.v) {  // the next token's mix, which its work begins with
          S::project(p, small[(slot + 1) & (kSmallSlots - 1)], mixed[parity ^ 1]);
          p.sync();
        }
        float c1 = 0.f, c2 = 0.f;
        for (int i = 0; i < p.W; ++i) {
          c1 += red[parity][p.slot0() + i][0];
          c2 += red[parity][p.slot0() + i][1];
        }
        const f2 k1 = both(-c1 * inv), k2 = both(a.norm == HC_NORM_LAYER ? -c2 * inv : 0.f);
        if (a.grad_f && (RAGGED || p.live)) {
#pragma unroll
          for (int k = 0; k < M; ++k) {
            if (k >= m) break;
            if (a.norm != HC_NORM_NONE) {  // without a norm f's value plays no part, be it a NaN
              const V8 f = rows.get(0, 2 * N + k);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                q[k].v[i] = mul2(r2, fma2(mul2(add2(f.v[i], less), r2), k1, add2(q[k].v[i], k2)));
            }
            if constexpr (RAGGED)
              rows.stage8(k, q[k]);
            else
              put8<T>(static_cast<T*>(a.grad_f) + t * E + k * D + p.d0, q[k]);
          }
          if constexpr (RAGGED) rows.template unstage<M>(static_cast<T*>(a.grad_f) + t * E + p.d0, m, D, p.warp_cols);
        }
        if (next < a.T) fetch_f(next);
      });
  store_param_sums<RAGGED, 1, M>(a, p, p.live ? 1 : 0, A, B);
}

// ------------------------------------------------------------------- host
using NormKernel = void (*)(NormArgs, int);

// Rows of whole chunks have kernels for 1, 2, 4 and 8 streams, ragged ones for 4
// and 8; none for fewer streams than blocks. Numbers between are cheap to read
// and dear to mix (16,384 x n x 768 bf16, forward and backward, n = 3, 4, 5, 6, 7,
// 8: read 86, 95, 110, 120, 128, 136 us, mix-write 173, 180, 283, 291, 297, 303;
// m = 3 and 4 at n = 4: read 187, 199, mix-write 449, 525): the work of the mix
// is the larger kernel's.
inline int padded_blocks(int m) { return m <= 1 ? 1 : m <= 2 ? 2 : 4; }
inline int padded_streams(int n, int M, bool ragged) {
  const int least = ragged ? 4 : M > n ? M : n;
  return least <= 1 && n <= 1 ? 1 : least <= 2 && n <= 2 ? 2 : n <= 4 ? 4 : 8;
}

// Shared memory of a CTA: its threads' rows and its groups' small matrices.
inline int64_t norm_smem_bytes(bool write, bool bwd, bool ragged, int N, int M, int chunks, int threads, int groups, int esize) {
  const int rows = write ? (bwd ? 2 * N : N) + 2 * M : N + (bwd ? M : 0);
  const int pitch = ragged && esize == 2 ? kPitchOf<__half, true> : kRowPitch, stage = !ragged ? 0 : write || bwd ? N : M;
  const int64_t entries = write ? (N * N + N * M + N + 3) / 2 * 2 : N * M + 2;
  const int64_t group = (entries * 8 * kSmallSlots + (write ? N * N * 20 : 0) + 15) / 16 * 16;
  const int64_t warp = static_cast<int64_t>(rows * esize / 2) * chunks * pitch + stage * 256 * esize;
  return warp * (threads / 32) + groups * group;
}
static_assert(sizeof(ReadMemory<8, 4>) == (34 * 8 * kSmallSlots + 15) / 16 * 16);
static_assert(sizeof(WriteMemory<8, 4>) == (106 * 8 * kSmallSlots + 64 * 20 + 15) / 16 * 16);
static_assert(sizeof(WriteMemory<1, 1>) == (6 * 8 * kSmallSlots + 20 + 15) / 16 * 16);

// The kernel for n streams, m blocks and ch chunks a thread: the next larger of
// 1, 2, 4, 8 and of 1, 2, 4 (rows past n and m are neither read nor written).
template <typename T, bool WRITE, bool BWD, int N, int M, int CH, bool RAGGED, bool WIDE> NormKernel norm_kernel_of() {
  if constexpr (WRITE && BWD) return write_norm_bwd_kernel<T, N, M, CH, RAGGED, WIDE>;
  if constexpr (WRITE && !BWD) return write_norm_fwd_kernel<T, N, M, CH, RAGGED, WIDE>;
  if constexpr (!WRITE && BWD) return read_norm_bwd_kernel<T, N, M, CH, RAGGED, WIDE>;
  if constexpr (!WRITE && !BWD) return read_norm_fwd_kernel<T, N, M, CH, RAGGED, WIDE>;
}
template <typename T, bool WRITE, int N, int M, bool RAGGED> NormKernel norm_kernel_for(bool bwd, bool wide, int ch) {
  if (bwd) {
    if constexpr (norm_bwd_threads(N, M, sizeof(T), false) < kWideThreads)
      if (wide) return norm_kernel_of<T, WRITE, true, N, M, 1, RAGGED, true>();
    return norm_kernel_of<T, WRITE, true, N, M, 1, RAGGED, false>();
  }
  if constexpr (norm_fwd_threads(N, M, 1, sizeof(T), false) < kWideThreads)
    if (wide) return norm_kernel_of<T, WRITE, false, N, M, 1, RAGGED, true>();
  if constexpr (!RAGGED && norm_fwd_chunks(N, M, sizeof(T)) >= 3) {
    if (ch == 3) return norm_kernel_of<T, WRITE, false, N, M, 3, false, false>();
    if (ch == 2) return norm_kernel_of<T, WRITE, false, N, M, 2, false, false>();
  }
  return norm_kernel_of<T, WRITE, false, N, M, 1, RAGGED, false>();
}
template <typename T, bool WRITE> NormKernel norm_kernel(const NormGeometry& geo, bool bwd, int N, int M) {
#define HC_NM(N, M, RAGGED) norm_kernel_for<T, WRITE, N, M, RAGGED>(bwd, geo.wide, geo.chunks)
  if (geo.ragged) {
    if (N == 4) return M == 1 ? HC_NM(4, 1, true) : M == 2 ? HC_NM(4, 2, true) : HC_NM(4, 4, true);
    return M == 1 ? HC_NM(8, 1, true) : M == 2 ? HC_NM(8, 2, true) : HC_NM(8, 4, true);
  }
  if (N == 1) return HC_NM(1, 1, false);
  if (N == 2) return M == 1 ? HC_NM(2, 1, false) : HC_NM(2, 2, false);
  if (N == 4) return M == 1 ? HC_NM(4, 1, false) : M == 2 ? HC_NM(4, 2, false) : HC_NM(4, 4, false);
  return M == 1 ? HC_NM(8, 1, false) : M == 2 ? HC_NM(8, 2, false) : HC_NM(8, 4, false);
#undef HC_NM
}

// Warps of a token's group, and for the forward the chunks a thread owns; 0
// warps where the 8-column kernels do not take the shape (rows that do not fit a
// CTA: a backward's threads own one chunk, so from 4104 columns on; 4,096 tokens,
// n = 4, bf16: backward of 4096, 5120 and 8192 columns in 81, 706 and 1,183 us for
// the read, 151, 3,062 and 5,052 for the mix-write). `aligned`: streams and
// parameters on 16-byte boundaries.
inline NormGeometry norm_geometry(bool write, bool bwd, int n, int m, int64_t D, int esize, bool aligned) {
  NormGeometry g{};
  g.ragged = !aligned || D % kColumns != 0;
  const int M = padded_blocks(m), N = padded_streams(n, M, g.ragged);
  const int64_t lines = (D + 32 * kColumns - 1) / (32 * kColumns);  // warps with a chunk a thread
  const int most = bwd || g.ragged ? 1 : norm_fwd_chunks(N, M, esize);
  g.chunks = static_cast<int>(lines < most ? lines : most);
  const int64_t warps = (lines + g.chunks - 1) / g.chunks;
  const int groups = warps == 1 ? kSmallGroups : 1;
  const int64_t threads = 32 * warps * groups;
  const int most_threads = bwd ? norm_bwd_threads(N, M, esize, false) : norm_fwd_threads(N, M, g.chunks, esize, false);
  g.wide = threads > most_threads && most_threads < kWideThreads;
  if (threads > (g.wide ? kWideThreads : most_threads) ||
      norm_smem_bytes(write, bwd, g.ragged, N, M, g.chunks, static_cast<int>(threads), groups, esize) > kNormSmemMax)
    return g;
  g.warps = static_cast<int>(warps);
  return g;
}

// CTAs of a kernel that an SM holds, 0 on an error; the kernel is made ready for
// that much shared memory. The driver is asked once a kernel, size and device on
// each thread (a decoding step's read + pre-norm 10.8 -> 10.5 us a call).
inline int ctas_per_sm(const void* kernel, int threads, int smem) {
  struct Known {
    const void* kernel;
    int threads, smem, device, ctas;
  };
  thread_local Known known[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  Known& at = known[(reinterpret_cast<uintptr_t>(kernel) / 16 + threads / 32) % 64];
  if (at.kernel == kernel && at.threads == threads && at.smem == smem && at.device == device) return at.ctas;
  int ctas = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormSmemMax) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, threads, smem) != cudaSuccess || ctas < 1) {
    cudaGetLastError();
    return 0;
  }
  at = Known{kernel, threads, smem, device, ctas};
  return ctas;
}

template <typename T, bool WRITE>
int norm_launch(bool bwd, NormGeometry& geo, const NormArgs& a, cudaStream_t s) {
  if (geo.warps == 0) return norm_launch_elem<T>(WRITE, bwd, geo, a, s);
  const int groups = geo.warps == 1 ? kSmallGroups : 1, threads = 32 * geo.warps * groups;
  const int M = padded_blocks(a.m), N = padded_streams(a.n, M, geo.ragged);
  const NormKernel k = norm_kernel<T, WRITE>(geo, bwd, N, M);
  const int smem = static_cast<int>(norm_smem_bytes(WRITE, bwd, geo.ragged, N, M, geo.chunks, threads, groups, sizeof(T)));
  const int per_sm = ctas_per_sm(reinterpret_cast<const void*>(k), threads, smem);
  if (per_sm < 1) return HC_ERR_LAUNCH;
  const int64_t want = (a.T + groups - 1) / groups, most = static_cast<int64_t>(per_sm) * sm_count();
  geo.grid = static_cast<int>(want < most ? want : most);
  geo.rows = geo.grid * groups;
  k<<<geo.grid, threads, smem, s>>>(a, geo.warps);
  return launch_status();
}

}  // namespace hc
