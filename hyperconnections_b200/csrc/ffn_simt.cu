// ffn_simt.cu — the gated feed-forward's float32 products on the FMA units (the
// tensor cores have no float32 inputs): any size and order.
//
// 256 threads make a 64 x 64 tile of the result (for h: 64 x 32 of a and of b)
// in four groups, each of which sums every fourth stage of 16 steps on its own
// and over the whole tile; the groups' sums are added in their order at the end.
// So a few hundred rows fill the device's schedulers, and a thread still makes 8
// x 8 values: four 16-byte reads of shared memory for 64 FMAs, where 4 x 4
// values take two for 16 and the reads bound the kernel. A warp's lanes are 4
// rows x 8 columns of such blocks, whose reads of a step are 64 and 128
// consecutive bytes; columns go in pairs through fma.rn.f32x2, which halves the
// instructions. Stages arrive by 4-byte asynchronous copies, which take any
// alignment, stride and order, two of the group's stages ahead. Products with
// few tiles also split their sum over CTAs, whose parts one more kernel adds in
// order.
//
// Forward and backward of 4096 x 1024 x 2048: 48 TFLOP/s (3,217 us; 3,788 with
// single FMAs), two thirds of the FMA units' peak: the reads of shared memory
// return 128 bytes a cycle, as long as the FMAs they feed take. Of 517 x 333 x
// 887: 133 us (204 with 4 x 4 values and no groups): five products of 20-39 us,
// two thirds of them waits for the first stages and for each other's last ones.
//
// A few rows, at most 24, take tiles of 8 x 64, a thread all rows of four
// columns for four of a stage's sixteen steps: the weights' way through shared
// memory bounds it. The forward of at most 4 rows streams the weights.
#include "ffn.cuh"
#include "mix_warp.cuh"  // smem_u32
#include "pairs.cuh"

namespace hc {
namespace {

constexpr int kTile = 64, kDepth = 16, kPitch = kTile + 4, kStages = 3;
constexpr int kGroup = 64, kGroups = 4, kThreads = kGroup * kGroups;
constexpr int kFewRows = 8;  // of a tile for a few tokens

// Shared memory by the tile's rows of A: a group's stages are A's [step][row] and B's.
template <int TM> struct Layout {
  static constexpr int kPitchA = TM + 4, kStageA = kDepth * kPitchA, kStage = kStageA + kDepth * kPitch;
  static constexpr int kGroupFloats = kStages * kStage, kBytes = kGroups * kGroupFloats * 4;
  static constexpr int kPerSm = TM == kTile ? 2 : 3;
  static constexpr int kSums = TM == kTile ? kTile * kTile : 4 * TM * kTile;  // of a group, which take its stages' place
  static_assert(kGroupFloats >= kSums);
};

__device__ __forceinline__ void copy4(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// 4 bytes, or zeros with nothing read.
__device__ __forceinline__ void copy4_or_zero(uint32_t dst, const float* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}

// Where the lanes of a copy lie along the sum, two steps 8 apart would meet in
// a bank (8 x the pitch is a multiple of 32): the pairs of four rows change places
// in the later one.
__device__ __forceinline__ constexpr int swap(bool along, int k) { return along && k >= 8 ? 2 : 0; }

// ROWS rows of an operand, 16 steps at a time by the 64 threads of a group,
// neighbouring threads along its unit stride (ALONG: the sum's), into a
// [step][row] buffer. Rows and steps past the operand's end count as 0.
template <int ROWS, bool ALONG, int PITCH> struct Loader {
  static constexpr int kLoads = ROWS * kDepth / kGroup;
  static constexpr int kRowStep = ALONG ? kGroup / kDepth : 0, kStep = ALONG ? 0 : kGroup / ROWS;  // from load to load
  const float* p;
  int64_t step, advance;  // from one of a thread's loads to the next; from the group's stage to its next
  uint32_t rows;          // bit i: the row of load i exists
  static_assert(kRowStep % 4 == 0);  // swap() works within four rows
  __device__ __forceinline__ static int row(int tid) { return ALONG ? tid / kDepth : tid % ROWS; }
  __device__ __forceinline__ static int k(int tid) { return ALONG ? tid % kDepth : tid / ROWS; }
  __device__ __forceinline__ void start(const FfnOperand& o, int64_t row0, int64_t k0, int tid) {
    const int64_t ld = ALONG ? o.row_stride : o.k_stride, r = row0 + row(tid);
    p = static_cast<const float*>(o.p) + (ALONG ? r * ld + k0 + k(tid) : r + (k0 + k(tid)) * ld);
    step = (ALONG ? kRowStep : kStep) * ld;
    advance = kGroups * kDepth * (ALONG ? 1 : ld);
    rows = 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) rows |= (r + i * kRowStep < o.rows ? 1u : 0u) << i;
  }
  __device__ __forceinline__ void fetch(uint32_t buffer, int64_t left, int tid) {  // `left` steps of the sum from this stage on
    const float* q = p;
    const uint32_t dst = buffer + 4 * (k(tid) * PITCH + (row(tid) ^ swap(ALONG, k(tid))));
    constexpr int to = 4 * (kStep * PITCH + kRowStep);
    if (left >= kDepth && rows == (1u << kLoads) - 1) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i, q += step) copy4(dst + i * to, q);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i, q += step) {
        const bool there = (rows >> i & 1u) && k(tid) + i * kStep < left;
        copy4_or_zero(dst + i * to, there ? q : p, there);
      }
    }
    p += advance;
  }
};

// Products of one launch, the jobs' tiles one after the other in blockIdx.x.
struct Jobs {
  FfnProduct p[kFfnMaxJobs];
  float* parts[kFfnMaxJobs];
  int run[kFfnMaxJobs], first[kFfnMaxJobs];  // tiles a row (a few tokens: a column) of tiles, and before the job
  int count, splits;
};

// Four neighbouring values, their pairs changed back.
__device__ __forceinline__ void read4(const float* p, int swapped, float* r) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  r[swapped] = v.x; r[swapped + 1] = v.y; r[2 - swapped] = v.z; r[3 - swapped] = v.w;
}
__device__ __forceinline__ void read_pairs(const float* p, int swapped, f2* r) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  r[swapped / 2] = v.x;
  r[1 - swapped / 2] = v.y;
}
__device__ __forceinline__ bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Four neighbouring values, of which the first `count` exist; `wide`: p is 16-byte aligned.
__device__ __forceinline__ void write4(float* p, const float* v, int64_t count, bool wide) {
  if (wide && count >= 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) p[i] = v[i];
  }
}

// TM: the tile's rows. AK, BK: whether A's and B's unit stride is the sum's.
template <int EPI, int TM, bool AK, bool BK>
__global__ void __launch_bounds__(kThreads, Layout<TM>::kPerSm) ffn_simt_kernel(const __grid_constant__ Jobs jobs) {
  using L = Layout<TM>;
  extern __shared__ __align__(16) float smem[];
  constexpr int kTileN = EPI == kGlu ? kTile / 2 : kTile;
  constexpr bool few = TM == kFewRows;
  int job = 0;
#pragma unroll
  for (int j = 1; j < kFfnMaxJobs; ++j)
    if (j < jobs.count && static_cast<int>(blockIdx.x) >= jobs.first[j]) job = j;
  const FfnProduct& p = jobs.p[job];
  const int tile = static_cast<int>(blockIdx.x) - jobs.first[job], line = tile / jobs.run[job];
  const int at = tile - line * jobs.run[job];
  const int64_t m0 = static_cast<int64_t>(few ? at : line) * TM, n0 = static_cast<int64_t>(few ? line : at) * kTileN;
  const int group = threadIdx.x / kGroup, tid = threadIdx.x % kGroup, lane = threadIdx.x & 31;
  // 64 rows: a thread's 4 + 4 rows and columns begin at ty and tx. A few: all rows, four columns from tx, every fourth
  // block of four steps.
  const int ty = (tid >> 5) * 32 + 4 * (lane >> 3), tx = few ? 4 * (tid & 15) : 4 * (lane & 7);
  const int quarter = tid >> 4;
  float* const mine = smem + group * L::kGroupFloats;
  constexpr int kPairs = few ? 2 : 4;
  f2 acc[8][kPairs] = {};  // pairs of columns

  // the CTA's stages of each term's sum, dealt out to the groups
  const int per_term = static_cast<int>((p.K + kDepth - 1) / kDepth), stages = per_term * p.terms;
  const int s0 = static_cast<int>(static_cast<int64_t>(stages) * blockIdx.y / jobs.splits);
  const int s1 = static_cast<int>(static_cast<int64_t>(stages) * (blockIdx.y + 1) / jobs.splits);
  Loader<TM, AK, L::kPitchA> la;
  Loader<kTileN, BK, kPitch> lb, lu;  // kGlu: rows of w_gate and of w_up
  int term = -1, into = 0;
  auto fetch = [&](int st) {
    if (st < s1) {
      const int t = st >= per_term ? 1 : 0, k0 = (st - t * per_term) * kDepth;
      if (t != term) {
        term = t;
        la.start(p.A[t], m0, k0, tid);
        lb.start(p.B[t], n0, k0, tid);
        if constexpr (EPI == kGlu) lu.start(p.B[1], n0, k0, tid);
      }
      const int64_t left = p.K - k0;
      const uint32_t a = smem_u32(mine + into * L::kStage), b = a + 4 * L::kStageA;
      la.fetch(a, left, tid);
      lb.fetch(b, left, tid);
      if constexpr (EPI == kGlu) lu.fetch(b + 4 * kTileN, left, tid);
      if (++into == kStages) into = 0;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // one group of copies a stage, empty behind the last
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(s0 + group + i * kGroups);
  int slot = 0;
  for (int st = s0 + group; st < s1; st += kGroups) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(kGroup) : "memory");  // arrived, and the one before it has been read
    fetch(st + (kStages - 1) * kGroups);
    const float *sA = mine + slot * L::kStage, *sB = sA + L::kStageA;
#pragma unroll
    for (int step = 0; step < (few ? kDepth / 4 : kDepth); ++step) {
      float a[8];
      f2 b[kPairs];
      if constexpr (few) {
        const int k = 4 * quarter + step;
        read4(&sA[k * L::kPitchA], 0, a);
        read4(&sA[k * L::kPitchA + 4], 0, a + 4);
        read_pairs(&sB[k * kPitch + tx], 0, b);
      } else {
        const int k = step;
        read4(&sA[k * L::kPitchA + ty], swap(AK, k), a);
        read4(&sA[k * L::kPitchA + ty + 16], swap(AK, k), a + 4);
        read_pairs(&sB[k * kPitch + tx], swap(BK, k), b);
        read_pairs(&sB[k * kPitch + tx + 32], swap(BK, k), b + 2);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const f2 aa = both(a[i]);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) acc[i][j] = fma2(aa, b[j], acc[i][j]);
      }
    }
    if (++slot == kStages) slot = 0;
  }

  // the groups' sums in their order
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(kGroup) : "memory");
  if constexpr (few) {  // [quarter][row][column]; a thread finishes one or two results
    const bool back_a = AK && quarter >= 2, back_b = BK && quarter >= 2;  // swap() of steps 8 to 15
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<ulonglong2*>(&mine[(quarter * 8 + (back_a ? i ^ 2 : i)) * kTile + tx]) =
          make_ulonglong2(back_b ? acc[i][1] : acc[i][0], back_b ? acc[i][0] : acc[i][1]);
    __syncthreads();
    const auto sum = [&](int row, int col) {
      float r = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int q = 0; q < 4; ++q) r += smem[g * L::kGroupFloats + (q * 8 + row) * kTile + col];
      return r;
    };
    for (int o = threadIdx.x; o < 8 * kTileN; o += kThreads) {
      const int row = o / kTileN, col = o % kTileN;
      const int64_t m = m0 + row, n = n0 + col, to = m * p.ldo + n;
      if (m >= p.M || n >= p.N) continue;
      const float v = sum(row, col);
      if constexpr (EPI == kStore) {
        if (float* parts = jobs.parts[job]) parts[(blockIdx.y * p.M + m) * p.N + n] = v;
        else static_cast<float*>(p.out)[to] = v;
      } else if constexpr (EPI == kGlu) {
        const float b = sum(row, col + kTileN);
        float val, der;
        ffn_act(p.act, v, val, der);
        static_cast<float*>(p.out)[to] = val * b;
        if (p.slope_gate) {
          static_cast<float*>(p.slope_gate)[to] = der * b;
          static_cast<float*>(p.slope_up)[to] = val;
        }
      } else {
        static_cast<float*>(p.out)[to] = v * static_cast<const float*>(p.slope_gate)[to];
        static_cast<float*>(p.out2)[to] = v * static_cast<const float*>(p.slope_up)[to];
      }
    }
  } else {  // two rows of each thread's eight a group
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float lo, hi;
        hc::split(acc[i][j], lo, hi);
        mine[(8 * i + 2 * j) * kGroup + tid] = lo;
        mine[(8 * i + 2 * j + 1) * kGroup + tid] = hi;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 8 / kGroups; ++r) {
      const int i = 8 / kGroups * group + r;
      float sum[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[j] = smem[(8 * i + j) * kGroup + tid];
#pragma unroll
        for (int g = 1; g < kGroups; ++g) sum[j] += smem[g * L::kGroupFloats + (8 * i + j) * kGroup + tid];
      }
      const int64_t m = m0 + ty + (i & 3) + 16 * (i >> 2);
      if (m >= p.M) continue;
      if constexpr (EPI == kStore) {
        float* parts = jobs.parts[job];
        float* row = parts ? parts + (blockIdx.y * p.M + m) * p.N : static_cast<float*>(p.out) + m * p.ldo;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t n = n0 + tx + 32 * h;
          write4(row + n, sum + 4 * h, p.N - n, on16(row));
        }
      } else {
        const bool wide = on16(p.out) && on16(p.out2) && on16(p.slope_gate) && on16(p.slope_up);  // rows are of whole 32 bytes
        if constexpr (EPI == kGlu) {
          const int64_t n = n0 + tx, to = m * p.ldo + n;
          float h[4], sg[4], su[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float der;
            ffn_act(p.act, sum[j], su[j], der);
            h[j] = su[j] * sum[4 + j];
            sg[j] = der * sum[4 + j];
          }
          write4(static_cast<float*>(p.out) + to, h, p.N - n, wide);
          if (p.slope_gate) {
            write4(static_cast<float*>(p.slope_gate) + to, sg, p.N - n, wide);
            write4(static_cast<float*>(p.slope_up) + to, su, p.N - n, wide);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t n = n0 + tx + 32 * h, to = m * p.ldo + n;
            float da[4], db[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bool there = n + j < p.N;
              da[j] = there ? sum[4 * h + j] * static_cast<const float*>(p.slope_gate)[to + j] : 0.f;
              db[j] = there ? sum[4 * h + j] * static_cast<const float*>(p.slope_up)[to + j] : 0.f;
            }
            write4(static_cast<float*>(p.out) + to, da, p.N - n, wide);
            write4(static_cast<float*>(p.out2) + to, db, p.N - n, wide);
          }
        }
      }
    }
  }
}

// The forward's products for at most 4 rows of A, bound by the weights: a CTA
// takes four rows of them (two of w_gate and the same two of w_up), its lanes 16
// bytes of each at a time and its warps every eighth 512 bytes, straight into
// registers; x comes from L1. No stage, no barrier until the sums meet. (Forward
// of 2048 x 8192: 46 us, 4.3 TB/s of weights, for one token and 57 for four, against
// 75 and 77 with tiles; for eight, whose x costs more loads than the weights, 81
// against 78.)
constexpr int kStreamThreads = 256, kStreamWarps = kStreamThreads / 32, kStreamTokens = 4;

__device__ __forceinline__ float4 weight4(const float* p) {
  float4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

template <int MATS> __global__ void __launch_bounds__(kStreamThreads, 3) ffn_stream_kernel(const __grid_constant__ FfnProduct p) {
  constexpr int kRows = 4 / MATS;
  __shared__ float sums[kStreamWarps][4 * kStreamTokens];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  const int tokens = static_cast<int>(p.M);
  const float* w[4];
  bool there[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const FfnOperand& b = p.B[v / kRows];
    const int64_t row = row0 + v % kRows;
    there[v] = row < b.rows;
    w[v] = static_cast<const float*>(b.p) + (there[v] ? row : 0) * b.row_stride;
  }
  const float* x = static_cast<const float*>(p.A[0].p);
  const int64_t ldx = p.A[0].row_stride;
  f2 acc[4][kStreamTokens] = {};  // of even and odd steps
  constexpr int64_t kStep = 4 * kStreamThreads;
  const int64_t first = 4 * threadIdx.x;
  float4 next[4];
  const auto load = [&](int64_t k) {
#pragma unroll
    for (int v = 0; v < 4; ++v) next[v] = k < p.K && there[v] ? weight4(w[v] + k) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  load(first);
  for (int64_t k = first; k < p.K; k += kStep) {  // K is a multiple of 4
    f2 lo[4], hi[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      lo[v] = pair(next[v].x, next[v].y);
      hi[v] = pair(next[v].z, next[v].w);
    }
    load(k + kStep);
#pragma unroll
    for (int t = 0; t < kStreamTokens; ++t) {
      if (t >= tokens) break;
      const float4 xv = __ldg(reinterpret_cast<const float4*>(x + t * ldx + k));
      const f2 x0 = pair(xv.x, xv.y), x1 = pair(xv.z, xv.w);
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[v][t] = fma2(hi[v], x1, fma2(lo[v], x0, acc[v][t]));
    }
  }
  // the lanes' sums: every exchange sends half of the live values, lanes l and l + 16 end with value l (row l / 4, token
  // l % 4)
  constexpr int kValues = 4 * kStreamTokens;
  float s[kValues];
#pragma unroll
  for (int i = 0; i < kValues; ++i) s[i] = fold2(acc[i / kStreamTokens][i % kStreamTokens]);
#pragma unroll
  for (int o = kValues / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = lane & o ? s[i + o] : s[i], give = lane & o ? s[i] : s[i + o];
      s[i] = keep + __shfl_xor_sync(kFull, give, o);
    }
  s[0] += __shfl_xor_sync(kFull, s[0], kValues);
  if (lane < kValues) sums[warp][lane] = s[0];
  __syncthreads();
  if (warp != 0) return;
  float r = 0.f;
#pragma unroll
  for (int i = 0; i < kStreamWarps; ++i) r += sums[i][lane % kValues];
  const float b = __shfl_down_sync(kFull, r, kValues / 2);  // MATS 2: of w_up
  const int64_t t = lane % kStreamTokens, n = row0 + lane / kStreamTokens, to = t * p.ldo + n;
  if (lane >= kValues / MATS || t >= tokens || n >= p.N) return;
  if constexpr (MATS == 2) {
    float val, der;
    ffn_act(p.act, r, val, der);
    static_cast<float*>(p.out)[to] = val * b;
    if (p.slope_gate) {
      static_cast<float*>(p.slope_gate)[to] = der * b;
      static_cast<float*>(p.slope_up)[to] = val;
    }
  } else {
    static_cast<float*>(p.out)[to] = r;
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether the streaming kernel takes a product: rows of whole 16 bytes, summed along them.
bool streams(const FfnProduct& p) {
  if (p.M > kStreamTokens || p.terms != 1 || p.epilogue == kGluBwd || p.K % 4 != 0) return false;
  for (const FfnOperand* o : {&p.A[0], &p.B[0], &p.B[p.epilogue == kGlu ? 1 : 0]})
    if (o->k_stride != 1 || o->row_stride % 4 != 0 || !aligned16(o->p)) return false;
  return true;
}
int stream_launch(const FfnProduct& p, cudaStream_t s) {
  if (p.epilogue == kGlu)
    ffn_stream_kernel<2><<<static_cast<unsigned>(ceil_div(p.N, 2)), kStreamThreads, 0, s>>>(p);
  else
    ffn_stream_kernel<1><<<static_cast<unsigned>(ceil_div(p.N, 4)), kStreamThreads, 0, s>>>(p);
  return launch_status();
}

template <int TM> void (*kernel_of(int epilogue, bool ak, bool bk))(Jobs) {  // the orders that occur: see ffn.cuh
  if (epilogue == kGlu) return ffn_simt_kernel<kGlu, TM, true, true>;
  if (epilogue == kGluBwd) return ffn_simt_kernel<kGluBwd, TM, true, false>;
  if (ak) return bk ? ffn_simt_kernel<kStore, TM, true, true> : ffn_simt_kernel<kStore, TM, true, false>;
  return ffn_simt_kernel<kStore, TM, false, false>;
}

}  // namespace

// Tiles of 8 rows rather than 64: the forward of 2048 x 8192 takes 78 us against
// 182 at 8 rows, 128 against 183 at 16, 201 against 185 at 32; of 512 x 2048, 27
// against 34 at 32. On either side of the limit, 24 and 25 rows from cold caches:
// 175 and 188 us, 384 x 1536 23.5 and 33.8.
bool ffn_simt_few(int64_t M) { return M <= 24; }

int64_t ffn_simt_tiles(int64_t M, int64_t N, bool few) { return ceil_div(M, few ? kFewRows : kTile) * ceil_div(N, kTile); }

// CTAs that share the sum of one tile: until an SM has as many as it can hold,
// each with at least 8 stages (128 steps), two a group.
int ffn_simt_splits(int64_t tiles, int64_t K, int terms, bool few) {
  const int per_sm = few ? Layout<kFewRows>::kPerSm : Layout<kTile>::kPerSm;
  const int64_t by_sms = per_sm * sm_count() / tiles, by_depth = ceil_div(K, kDepth) * terms / (2 * kGroups);
  const int64_t s = by_sms < by_depth ? by_sms : by_depth;
  return static_cast<int>(s < 1 ? 1 : s > 32 ? 32 : s);
}

int ffn_simt_launch(const FfnProduct* ps, int count, float* parts, cudaStream_t s) {
  const int epilogue = ps[0].epilogue, tile_n = epilogue == kGlu ? kTile / 2 : kTile;
  if (count == 1 && streams(ps[0])) return stream_launch(ps[0], s);
  bool few = true;
  for (int j = 0; j < count; ++j) few = few && ffn_simt_few(ps[j].M);
  Jobs jobs{};
  jobs.count = count;
  int64_t total = 0;
  for (int j = 0; j < count; ++j) {
    const int64_t rows = ceil_div(ps[j].M, few ? kFewRows : kTile), cols = ceil_div(ps[j].N, tile_n);
    jobs.p[j] = ps[j];
    jobs.run[j] = static_cast<int>(few ? rows : cols);
    jobs.first[j] = static_cast<int>(total);
    total += rows * cols;
    if (total > INT_MAX) return HC_ERR_BAD_SIZE;
  }
  jobs.splits = epilogue == kStore ? ffn_simt_splits(total, ps[0].K, ps[0].terms, few) : 1;
  if (jobs.splits > 1) {
    if (!parts) return HC_ERR_SCRATCH;
    float* at = parts;
    for (int j = 0; j < count; ++j) {
      jobs.parts[j] = at;
      at += jobs.splits * ps[j].M * ps[j].N;
    }
  }
  const bool ak = ps[0].A[0].k_stride == 1, bk = ps[0].B[0].k_stride == 1;
  const auto kernel = few ? kernel_of<kFewRows>(epilogue, ak, bk) : kernel_of<kTile>(epilogue, ak, bk);
  const int bytes = few ? Layout<kFewRows>::kBytes : Layout<kTile>::kBytes;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return HC_ERR_LAUNCH;
  }
  // plain launches: CTAs that come up early crowd the SMs with room (8 tokens, 2048 x 8192, forward: 88 us against 78)
  kernel<<<dim3(static_cast<unsigned>(total), jobs.splits), kThreads, bytes, s>>>(jobs);
  if (int rc = launch_status()) return rc;
  if (jobs.splits == 1) return HC_OK;
  FfnParts sums[kFfnMaxJobs];
  for (int j = 0; j < count; ++j) sums[j] = {jobs.parts[j], ps[j].out, ps[j].M * ps[j].N, false};
  return ffn_add_parts(sums, count, jobs.splits, HC_DTYPE_F32, s);
}

}  // namespace hc
