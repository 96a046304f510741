// ffn_tc.cu — the gated feed-forward's products on the 5th-generation tensor
// cores, bf16 and fp16.
//
// A pair of CTAs (a cluster of two, on two SMs) owns a 256 x 256 tile of a
// result: tcgen05.mma with cta_group::2, each CTA holding 128 rows of A, 128
// rows of B and its 128 x 256 half of the float32 accumulator in tensor
// memory. Against a CTA of its own with a 128 x 256 tile this halves the bytes
// of B that an SM fetches: 32 KB for every 512 cycles of the tensor cores.
// Clusters are persistent and walk the tiles; per CTA
//
//   warp 0      fetches: one lane issues the TMA copies of the CTA's halves of
//               A and B into a ring of 32 KB stages (64 deep); both CTAs'
//               copies are counted on the leader's barrier
//   warp 1      multiplies (in the leader CTA): one lane issues the four
//               16-deep steps of a stage for both CTAs
//   warp 2      owns the tensor memory, and (for da, db) stores what is finished
//   warp 3      (for da, db) fetches the tile's slopes, 32 columns of a quarter
//               at a time, into six slots of 16 KB that go round
//   warps 4-19  finish: four groups of four warps read the accumulator out of
//               tensor memory, a quarter of the columns each, and write the
//               result while the next tile is multiplied into the other half of
//               tensor memory (2 x 256 of its 512 columns)
//
// Results leave through shared memory and TMA stores, and slopes come by TMA
// loads: a warp holds a row a lane, so its own loads and stores would touch 32
// lines each (da and db of 32,768 tokens, 384 x 1536, fp16: 134 us that way, 88
// with the copies). da and db take their slopes' places; a warp of its own stores
// them, so that the finishing warps need not wait for their slots to empty.
//
// What bounds the products: the wide ones (16,384 tokens, 2048 x 8192, bf16) keep
// the tensor pipe 58-91% active, under the power limit. In the narrow ones of the
// shape above (101, 48, 88, 91 and 131 us under the profiler for h and the slopes,
// y, da and db, dx, the weights' gradients) no unit is full: tensor pipe 42, 45,
// 23, 49 and 66%, L2 44, 28, 49, 33 and 37%, what the SMs read from it 17-30%. Of
// each some 13 us are its start and end, and y and dx have tiles for 3.5 rounds of
// the clusters, which take four. Fetching the next blocks into L2 ahead of their
// copies made every product 20-30% slower; a sixth stage and a release fence less
// changed nothing (the fence is there), and 128-byte lines for slopes and results
// cost the first shape what they gave the other.
//
// An operand is read as it lies: summed along its unit stride ("K-major", x
// and the weights of the forward) or across it ("MN-major", the weights of dx
// and both operands of the weights' gradients); both come as boxes of 128-byte
// lines with the 128-byte swizzle, and the matrix descriptor says which of the
// two they are. For h, the CTAs of a pair fetch different weights: the leader
// w_gate's 128 rows, its peer w_up's, so a accumulates in columns 0-127, b in
// columns 128-255 of the same rows, and a thread that finishes a row holds
// both.
//
// Products with few tiles and a long sum (the weights' gradients of a narrow
// model, a few tokens) split the sum over several clusters, which write
// float32 parts that one more kernel adds in order.
//
// Every wait is bounded (poll limit of status.cu): a warp that gives up
// reports it, tells both CTAs to stop, and the pair leaves together after its
// copies in flight have landed.
#include <cstring>

#include "ffn.cuh"
#include "mix_warp.cuh"
#include "pairs.cuh"

namespace hc {
namespace {

__device__ unsigned int g_ffn_wait_timeouts;

constexpr int kRows = 128;         // rows of A, and of B, that one CTA holds
constexpr int kTileM = 2 * kRows;  // a pair's tile
constexpr int kTileN = 2 * kRows;
constexpr int kDepth = 64;         // elements of the sum in a stage: 128 bytes
constexpr int kOperandBytes = kRows * kDepth * 2;
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kFinishWarp = 4;    // the first of the finishing warps
constexpr int kFinishWarps = 16;  // four a scheduler: with two, the activation's chains left it idle two cycles in three
constexpr int kThreads = 32 * (kFinishWarp + kFinishWarps);
constexpr int kSlotBytes = kOperandBytes;  // kGluBwd: 32 columns of both slopes, and of da and db in their place
constexpr int kSlots = 6;
constexpr int kUses = 8;  // of slots by a tile: the quarters' first 32 columns, then their second ones
// The ring's stages, and where results are put together: kStore's warps have 32
// rows of 64 bytes each, kGlu's three of them (h and the slopes).
constexpr int kMostStages = 6;
constexpr int stages_of(int epi) { return epi == kStore ? kMostStages : 4; }
constexpr int kBoxBytes = 32 * 64;
constexpr int warp_bytes_of(int epi) { return epi == kGlu ? 3 * kBoxBytes : kBoxBytes; }
constexpr int staging_of(int epi) { return epi == kGluBwd ? kSlots * kSlotBytes : kFinishWarps * warp_bytes_of(epi); }
constexpr int kSmemBytes = kMostStages * kStageBytes + staging_of(kStore) + 1024;
static_assert(kSmemBytes == stages_of(kGlu) * kStageBytes + staging_of(kGlu) + 1024);
static_assert(kSmemBytes == stages_of(kGluBwd) * kStageBytes + staging_of(kGluBwd) + 1024);
constexpr int kGroupM = 8;  // tiles of A that neighbouring clusters share B with

// Operands by term of a sum of two products, or by job of a launch of several.
struct alignas(64) TcMaps {
  CUtensorMap a[kFfnMaxJobs], b[kFfnMaxJobs];
  CUtensorMap out[kFfnMaxJobs];  // kStore: by job; kGlu: h and the slopes; kGluBwd: da and db
  CUtensorMap in[2];             // kGluBwd: the slopes
};

// One result. A launch of several shares the depth of the sum and the operands'
// order.
struct TcJob {
  int64_t M, N, ldo;
  void* out;
  float* parts;  // float32 parts [splits][M][N], or nullptr
  int tiles_m, tiles_n;
  int tma;  // the result's rows start on 16-byte boundaries: TMA stores
};

struct TcArgs {
  TcJob job[kFfnMaxJobs];
  const void* slope_gate;  // kGlu: whether the slopes are written
  int jobs, tiles, splits;  // tiles of all jobs
  int blocks_term, blocks;  // 64-deep blocks of one term, and of all
  int a_mn, b_mn;           // operands whose unit stride is their rows
  int tile_n;               // columns of a tile's accumulator
  uint32_t maps;            // bit i: the i-th of TcMaps is in use
  int act;
  uint32_t wait_limit;
  unsigned int* status;
};

struct Shared {
  uint64_t full[kMostStages], empty[kMostStages];
  uint64_t acc_full[2], acc_empty[2], drain;
  // By a tile's use of a slot: its slopes have arrived, its da and db are in place. By use and not by slot, so that who
  // waits for a phase has itself waited for the one before it; a slot passes from one quarter to another.
  uint64_t use_full[kUses], use_ready[kUses];
  uint64_t slot_done[kSlots];  // its results have left
  uint32_t tmem;
  volatile int stop;
};

// ------------------------------------------------------------------- PTX
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of a shared variable of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
// An arrival on a barrier of either CTA of the pair. Release: it gives back tensor memory whose reads (tcgen05.ld,
// waited for and fenced) have to come before the other side's next products. A relaxed one, which no rule of the memory
// model orders so, was no faster in any product.
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// The wait that goes with it.
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok;
}
// A box of a matrix into this CTA, counted on a barrier of the pair.
__device__ __forceinline__ void fetch_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// A box into this CTA, counted on its own barrier.
__device__ __forceinline__ void fetch_own(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// Until all but the last K groups of this thread's stores have read their source.
template <int K> __device__ __forceinline__ void store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(K) : "memory");
}
__device__ __forceinline__ void store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void put16(uint32_t at, const uint32_t* w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
__device__ __forceinline__ uint4 get16(uint32_t at) {
  uint4 q;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(at));
  return q;
}
// 16-byte word c of line r of a box of 64-byte lines as the TMA swizzles it: the
// line's number over two modulo 4 mixed in.
__device__ __forceinline__ uint32_t word64(uint32_t base, int r, int c) { return base + r * 64 + ((c ^ ((r >> 1) & 3)) << 4); }

__device__ __forceinline__ void mma_pair(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(acc),
      "l"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
// The barrier at this offset in both CTAs is arrived at when the products issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 16 consecutive columns of this thread's accumulator row.
__device__ __forceinline__ void acc_load16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
// Until the loads issued so far are done; r is theirs, so that no use of it moves up.
__device__ __forceinline__ void acc_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// Shared-memory matrix descriptor with the 128-byte swizzle. K-major: groups of
// 8 rows are 1024 bytes apart. MN-major: groups of 8 steps of the sum are 1024
// bytes apart, and the next 64 rows begin a whole box (64 lines) on.
__device__ __forceinline__ uint64_t matrix_desc(uint32_t addr, bool mn) {
  const uint64_t lead = mn ? (kDepth * 128) >> 4 : 1, step = 1024 >> 4;
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (lead << 16) | (step << 32) | (1ull << 46) | (2ull << 61);
}

// Bounded wait that also ends when the pair has been told to stop. CLUSTER: for threads of both CTAs.
template <bool CLUSTER = false>
__device__ __forceinline__ bool pair_wait(Shared& sh, uint64_t* bar, uint32_t parity, uint32_t limit) {
  for (uint32_t i = 0; i < limit; ++i) {
    if (CLUSTER ? try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
    if (sh.stop) return false;
  }
  return false;
}

__device__ __forceinline__ void tell_stop(Shared& sh, const TcArgs& a) {
  if (!sh.stop) report_timeout(&g_ffn_wait_timeouts, a.status);
  for (uint32_t r = 0; r < 2; ++r)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(const_cast<int*>(&sh.stop), r)), "r"(1)
                 : "memory");
}

// ------------------------------------------------------------------ tiles
struct Item {
  int job, m, n;       // result, and tile of it
  int split, k0, k1;   // blocks of the sum
};
// Item i of the walk: the splits one after the other, in each the jobs, in each
// kGroupM tiles of A for each tile of B, so that the clusters at work share
// rows of both through L2.
__device__ __forceinline__ Item item_at(const TcArgs& a, int i) {
  Item it;
  it.split = i / a.tiles;
  int t = i - it.split * a.tiles;
  it.job = 0;
#pragma unroll
  for (int j = 0; j + 1 < kFfnMaxJobs; ++j) {
    const int n = a.job[j].tiles_m * a.job[j].tiles_n;
    if (it.job == j && j + 1 < a.jobs && t >= n) {
      t -= n;
      it.job = j + 1;
    }
  }
  const int tiles_m = a.job[it.job].tiles_m, tiles_n = a.job[it.job].tiles_n;
  const int per_group = kGroupM * tiles_n;
  const int g = t / per_group;
  t -= g * per_group;
  const int rows = min(kGroupM, tiles_m - g * kGroupM);
  it.n = t / rows;
  it.m = g * kGroupM + (t - it.n * rows);
  it.k0 = static_cast<int>(static_cast<int64_t>(a.blocks) * it.split / a.splits);
  it.k1 = static_cast<int>(static_cast<int64_t>(a.blocks) * (it.split + 1) / a.splits);
  return it;
}

// ------------------------------------------------------------------ stores
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ uint32_t pack2(f2 v) {
  float a, b;
  split(v, a, b);
  return pack2<T>(a, b);
}
__device__ __forceinline__ void st_v8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float inverse_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// act(a) and act'(a) of two values with the approximate exponential and
// inverse: their errors, a few 2^-22 relative, and that of the exponent's
// argument (at most 36 for |a| <= 6: some 125 2^-24 of the result) are far below
// the half steps 2^-8 and 2^-11 of the types they go to.
__device__ __forceinline__ f2 sigmoid_of(f2 x) {  // 1 / (1 + 2^x)
  float e0, e1;
  split(x, e0, e1);
  split(add2(pair(exp2_fast(e0), exp2_fast(e1)), both(1.f)), e0, e1);
  return pair(inverse_fast(e0), inverse_fast(e1));
}
__device__ __forceinline__ void fast_act(int act, f2 a, f2& val, f2& der) {
  constexpr float kLog2e = 1.4426950408889634f;
  if (act == HC_ACT_SILU) {
    const f2 s = sigmoid_of(mul2(a, both(-kLog2e)));
    val = mul2(a, s);
    der = fma2(val, fma2(s, both(-1.f), both(1.f)), s);
  } else {  // a / (1 + e^-2u), see ffn_act
    constexpr float c2 = 2.f * 0.7978845608028654f;
    float q0, q1;
    split(mul2(a, a), q0, q1);
    const f2 a2 = pair(fminf(q0, 1e4f), fminf(q1, 1e4f));
    const f2 s = sigmoid_of(mul2(mul2(a, both(-c2 * kLog2e)), fma2(a2, both(0.044715f), both(1.f))));
    val = mul2(a, s);
    der = fma2(mul2(val, fma2(s, both(-1.f), both(1.f))), fma2(a2, both(3.f * 0.044715f * c2), both(c2)), s);
  }
}

// A finishing warp's part of a tile: 32 rows (one a lane), a quarter of the
// columns. `acc` is the warp's lanes of the accumulator at its columns, `release`
// gives the accumulator back once it has been read.
template <typename T> struct Part {
  const TcArgs& a;
  const TcJob& job;
  const TcMaps& maps;
  int lane, split, job_id;
  int64_t row0, n0;
  bool inside;  // any of it lies in the result
  __device__ __forceinline__ Part(const TcArgs& args, const TcMaps& m, const Item& it, int rank, int quad, int tile_n, int col)
      : a(args), job(args.job[it.job]), maps(m), lane(threadIdx.x & 31), split(it.split), job_id(it.job) {
    row0 = static_cast<int64_t>(it.m) * kTileM + rank * kRows + 32 * quad;
    n0 = static_cast<int64_t>(it.n) * tile_n + col;
    inside = row0 < job.M && n0 < job.N;
  }

  // 64 columns of the result, or of a part of its sum.
  template <typename Release> __device__ __forceinline__ void store(uint32_t acc, uint32_t mine, Release release) {
    const bool boxes = job.tma && !job.parts;
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      if (boxes && (st & 1) == 0) {
        if (lane == 0) store_wait_read<0>();  // the last 32 columns have left
        __syncwarp();
      }
      uint32_t r[16];
      acc_load16(acc + 16 * st, r);
      acc_wait(r);
      if (st == 3) release();
      const int64_t row = row0 + lane, n = n0 + 16 * st;
      if (job.parts) {
        if (row < job.M && n < job.N) {
          float* p = job.parts + (static_cast<int64_t>(split) * job.M + row) * job.N + n;
          if ((job.N & 7) == 0) {
            if (n + 8 <= job.N) st_v8(p, r);
            if (n + 16 <= job.N) st_v8(p + 8, r + 8);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (n + i < job.N) p[i] = __uint_as_float(r[i]);
          }
        }
      } else if (job.tma) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = pack2<T>(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
        put16(word64(mine, lane, 2 * (st & 1)), w);
        put16(word64(mine, lane, 2 * (st & 1) + 1), w + 4);
        if (st & 1) {
          fence_proxy_async_smem();
          __syncwarp();
          const int64_t x = n0 + 32 * (st >> 1);
          if (lane == 0) {
            if (row0 < job.M && x < job.N) store_box(&maps.out[job_id], static_cast<int>(x), static_cast<int>(row0), mine);
            store_commit();
          }
        }
      } else if (row < job.M) {
        T* p = static_cast<T*>(job.out) + row * job.ldo + n;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (n + i < job.N) p[i] = Elem<T>::from_f(__uint_as_float(r[i]));
      }
      __syncwarp();  // the next load is the whole warp's
    }
  }

  // 32 columns of h, act'(a) b and act(a); a at acc, b at acc + 128.
  template <typename Release> __device__ __forceinline__ void glu(uint32_t acc, uint32_t mine, Release release) {
    const bool keep = a.slope_gate != nullptr;
    if (lane == 0) store_wait_read<0>();  // the last tile's results have left
    __syncwarp();
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      uint32_t r[16], q[16];
      acc_load16(acc + 16 * st, r);
      acc_load16(acc + kRows + 16 * st, q);
      acc_wait(r);
      acc_wait(q);
      if (st == 1) release();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t h[4], sg[4], su[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = 8 * c + 2 * i;
          const f2 b = pair(__uint_as_float(q[k]), __uint_as_float(q[k + 1]));
          f2 v, d;
          fast_act(a.act, pair(__uint_as_float(r[k]), __uint_as_float(r[k + 1])), v, d);
          h[i] = pack2<T>(mul2(v, b));
          sg[i] = pack2<T>(mul2(d, b));
          su[i] = pack2<T>(v);
        }
        put16(word64(mine, lane, 2 * st + c), h);
        if (keep) {
          put16(word64(mine + kBoxBytes, lane, 2 * st + c), sg);
          put16(word64(mine + 2 * kBoxBytes, lane, 2 * st + c), su);
        }
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (inside) {
        const int x = static_cast<int>(n0), y = static_cast<int>(row0);
        store_box(&maps.out[0], x, y, mine);
        if (keep) {
          store_box(&maps.out[1], x, y, mine + kBoxBytes);
          store_box(&maps.out[2], x, y, mine + 2 * kBoxBytes);
        }
      }
      store_commit();
    }
  }

  // 32 columns (the part's first or second) of da and db, from dh and the slopes in the warp's lines of a slot, where
  // the results take their place.
  __device__ __forceinline__ void glu_bwd(uint32_t acc, int half, uint32_t gate, uint32_t up) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      uint32_t r[16];
      acc_load16(acc + 32 * half + 16 * st, r);
      acc_wait(r);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t at = word64(k ? up : gate, lane, 2 * st + c);
          float x[8];
          unpack<T>(get16(at), x);
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = pack2<T>(x[2 * i] * __uint_as_float(r[8 * c + 2 * i]), x[2 * i + 1] * __uint_as_float(r[8 * c + 2 * i + 1]));
          put16(at, w);
        }
      }
      __syncwarp();
    }
  }
};

template <typename T, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    ffn_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ TcArgs a) {
  extern __shared__ uint8_t raw[];
  __shared__ Shared sh;
  constexpr int kStages = stages_of(EPI), kWarpBytes = warp_bytes_of(EPI);
  const uint32_t ring = (smem_u32(raw) + 1023) & ~1023u, staging = ring + kStages * kStageBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int items = a.tiles * a.splits;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  pdl_launch_dependents();
  if (warp == 3 && lane < static_cast<int>(sizeof(TcMaps) / sizeof(CUtensorMap)) && (a.maps >> lane & 1u))
    prefetch_map(reinterpret_cast<const CUtensorMap*>(&maps) + lane);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh.acc_full[b], 1);
      mbar_init(&sh.acc_empty[b], 2 * kFinishWarps);  // of both CTAs
    }
    for (int u = 0; u < kUses; ++u) {
      mbar_init(&sh.use_full[u], 1);
      mbar_init(&sh.use_ready[u], 4);  // the quarter's warps
    }
    for (int q = 0; q < kSlots; ++q) mbar_init(&sh.slot_done[q], 1);
    mbar_init(&sh.drain, 1);
    sh.stop = 0;
    fence_mbar_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  pdl_wait_prior_grid();  // no memory is touched before the launches before this one are done

  if (warp == 0) {
    if (lane == 0) {
      // both CTAs' boxes; B's across the sum are 64 columns wide, be there 96 or 128
      const uint32_t stage_bytes =
          2 * (kOperandBytes + (a.b_mn ? (a.tile_n > 128 ? 2 : 1) * (kOperandBytes / 2) : a.tile_n / 2 * kDepth * 2));
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = first; i < items && ok; i += step) {
        const Item it = item_at(a, i);
        const int row_a = it.m * kTileM + static_cast<int>(rank) * kRows;
        const int row_b = EPI == kGlu ? it.n * kRows : it.n * a.tile_n + static_cast<int>(rank) * (a.tile_n / 2);
        for (int kb = it.k0; kb < it.k1; ++kb) {
          if (!pair_wait(sh, &sh.empty[s], ph ^ 1, a.wait_limit)) {
            ok = false;
            break;
          }
          const int term = kb >= a.blocks_term ? 1 : 0;
          const int k = (kb - term * a.blocks_term) * kDepth;
          const CUtensorMap* ma = &maps.a[it.job + term];
          const CUtensorMap* mb = &maps.b[EPI == kGlu ? static_cast<int>(rank) : it.job + term];
          const uint32_t bar = cluster_addr(&sh.full[s], 0);
          const uint32_t da = ring + s * kStageBytes, db = da + kOperandBytes;
          if (rank == 0) mbar_expect_tx(&sh.full[s], stage_bytes);
          if (a.a_mn) {
            fetch_box(da, ma, row_a, k, bar);
            fetch_box(da + kOperandBytes / 2, ma, row_a + 64, k, bar);
          } else {
            fetch_box(da, ma, k, row_a, bar);
          }
          if (a.b_mn) {
            fetch_box(db, mb, row_b, k, bar);
            if (a.tile_n > 128) fetch_box(db + kOperandBytes / 2, mb, row_b + 64, k, bar);
          } else {
            fetch_box(db, mb, k, row_b, bar);
          }
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // every stage's last release has arrived before the CTA leaves
      for (int j = 0; j < kStages && ok; ++j) {
        ok = pair_wait(sh, &sh.empty[s], ph ^ 1, a.wait_limit);
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok) tell_stop(sh, a);
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      // float32 sums of bf16 (format 1) or fp16 (0) operands, 256 x tile_n
      constexpr uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(a.a_mn) << 15) |
                             (static_cast<uint32_t>(a.b_mn) << 16) | (static_cast<uint32_t>(a.tile_n >> 3) << 17) |
                             ((kTileM >> 4) << 24);
      const uint64_t step_a = (a.a_mn ? 16 * 128 : 32) >> 4, step_b = (a.b_mn ? 16 * 128 : 32) >> 4;
      int s = 0, buf = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int i = first; i < items && ok; i += step) {
        const Item it = item_at(a, i);
        if (!pair_wait<true>(sh, &sh.acc_empty[buf], acc_ph ^ 1, a.wait_limit)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kb = it.k0; kb < it.k1; ++kb) {
          if (!pair_wait(sh, &sh.full[s], ph, a.wait_limit)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint64_t da = matrix_desc(ring + s * kStageBytes, a.a_mn);
          uint64_t db = matrix_desc(ring + s * kStageBytes + kOperandBytes, a.b_mn);
#pragma unroll
          for (int k = 0; k < kDepth / 16; ++k) {
            mma_pair(tmem + buf * kTileN, da, db, idesc, kb > it.k0 || k > 0);
            da += step_a;
            db += step_b;
          }
          commit_pair(&sh.empty[s]);
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        commit_pair(&sh.acc_full[buf]);
        buf ^= 1;
        if (buf == 0) acc_ph ^= 1;
      }
      if (!ok) {  // stop, and let the products in flight end before the tensor memory goes
        tell_stop(sh, a);
        commit_pair(&sh.drain);
        for (uint32_t i = 0; i < kWaitPolls && !mbar_try_wait(&sh.drain, 0); ++i) {
        }
      }
    }
  } else if (EPI == kGluBwd && warp == 3) {
    if (lane == 0) {  // the tiles' uses, one after the other, go round the slots
      bool ok = true;
      uint32_t slot = 0, ph = 0;
      for (int i = first; i < items && ok; i += step) {
        const Item it = item_at(a, i);
        const int row = it.m * kTileM + static_cast<int>(rank) * kRows;
        for (int use = 0; use < kUses; ++use) {
          if (!pair_wait(sh, &sh.slot_done[slot], ph ^ 1, a.wait_limit)) {
            ok = false;
            break;
          }
          const uint32_t dst = staging + slot * kSlotBytes;
          const int n = it.n * kTileN + (use & 3) * 64 + (use >> 2) * 32;
          mbar_expect_tx(&sh.use_full[use], kSlotBytes);
          fetch_own(dst, &maps.in[0], n, row, &sh.use_full[use]);
          fetch_own(dst + kSlotBytes / 2, &maps.in[1], n, row, &sh.use_full[use]);
          if (++slot == kSlots) {
            slot = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) tell_stop(sh, a);
    }
  } else if (EPI == kGluBwd && warp == 2) {
    if (lane == 0) {  // da and db leave; a slot is given back when the one behind it is on its way
      bool ok = true;
      uint32_t slot = 0, ph = 0;
      int last = -1;
      for (int i = first; i < items && ok; i += step, ph ^= 1) {
        const Item it = item_at(a, i);
        const int row = it.m * kTileM + static_cast<int>(rank) * kRows;
        for (int use = 0; use < kUses; ++use) {
          if (!pair_wait(sh, &sh.use_ready[use], ph, a.wait_limit)) {
            ok = false;
            break;
          }
          const uint32_t src = staging + slot * kSlotBytes;
          const int n = it.n * kTileN + (use & 3) * 64 + (use >> 2) * 32;
          if (n < a.job[0].N && row < a.job[0].M) {
            store_box(&maps.out[0], n, row, src);
            store_box(&maps.out[1], n, row, src + kSlotBytes / 2);
          }
          store_commit();
          store_wait_read<1>();
          if (last >= 0) mbar_arrive(&sh.slot_done[last]);
          last = static_cast<int>(slot);
          if (++slot == kSlots) slot = 0;
        }
      }
      store_wait_all();
      if (!ok) tell_stop(sh, a);
    }
  } else if (warp >= kFinishWarp) {
    const int quad = warp & 3, part = (warp - kFinishWarp) >> 2;
    const int tile_n = EPI == kGlu ? kRows : a.tile_n;
    constexpr int kPart = EPI == kGlu ? 32 : 64;  // columns of a quarter; a narrow tile has none for the last ones
    int buf = 0;
    uint32_t acc_ph = 0, uses = 0;  // of the slots, by the tiles before this one
    for (int i = first; i < items; i += step) {
      Part<T> tile(a, maps, item_at(a, i), static_cast<int>(rank), quad, tile_n, part * kPart);
      bool ok = pair_wait(sh, &sh.acc_full[buf], acc_ph, a.wait_limit);
      if (!__all_sync(kFull, ok)) {
        if (lane == 0) tell_stop(sh, a);
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + buf * kTileN + (static_cast<uint32_t>(32 * quad) << 16) + part * kPart;
      const auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(cluster_addr(&sh.acc_empty[buf], 0));
      };
      if constexpr (EPI == kGlu) {
        tile.glu(acc, staging + (warp - kFinishWarp) * kWarpBytes, release);
      } else if constexpr (EPI == kGluBwd) {
        for (int half = 0; half < 2; ++half) {
          const int use = 4 * half + part;
          ok = pair_wait(sh, &sh.use_full[use], uses / kUses & 1, a.wait_limit);
          if (!__all_sync(kFull, ok)) break;
          const uint32_t gate = staging + (uses + use) % kSlots * kSlotBytes + quad * 32 * 64;
          tile.glu_bwd(acc, half, gate, gate + kSlotBytes / 2);
          if (half) release();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.use_ready[use]);
        }
        if (!__all_sync(kFull, ok)) {
          if (lane == 0) tell_stop(sh, a);
          break;
        }
        uses += kUses;
      } else if (part * kPart >= tile_n) {
        release();
      } else {
        tile.store(acc, staging + (warp - kFinishWarp) * kWarpBytes, release);
      }
      buf ^= 1;
      if (buf == 0) acc_ph ^= 1;
    }
    if (lane == 0) store_wait_all();
  }
  __syncwarp();
  __syncthreads();
  if (sh.stop && threadIdx.x == 0)  // copies in flight may be counted on the other CTA's barrier: give them 4 ms
    for (int i = 0; i < 4096; ++i) __nanosleep(1000);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  __syncthreads();
  cluster_sync();
}

// ----------------------------------------------------- parts of a split sum
struct AddJobs {
  FfnParts job[kFfnMaxJobs];
  int jobs, splits;
};
template <typename T> __device__ __forceinline__ void put_sum(T* p, float4 s) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4*>(p) = s;
  else
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
}
template <typename T> __global__ void __launch_bounds__(256) add_parts_kernel(const __grid_constant__ AddJobs a) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256, first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
#pragma unroll
  for (int j = 0; j < kFfnMaxJobs; ++j) {
    if (j >= a.jobs) break;
    const float* parts = a.job[j].parts;
    T* out = static_cast<T*>(a.job[j].out);
    const int64_t count = a.job[j].count;
    if (a.job[j].fours) {
      for (int64_t i = 4 * first; i < count; i += 4 * stride) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < a.splits; ++p) {
          const float4 v = *reinterpret_cast<const float4*>(parts + p * count + i);
          s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
        }
        put_sum<T>(out + i, s);
      }
    } else {
      for (int64_t i = first; i < count; i += stride) {
        float s = 0.f;
        for (int p = 0; p < a.splits; ++p) s += parts[p * count + i];
        out[i] = Elem<T>::from_f(s);
      }
    }
  }
}

// ------------------------------------------------------------------- host
int pairs_resident() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sm_count() / 2;
  if (cached[dev] > 0) return cached[dev];
  int n = 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * (sm_count() / 2));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  auto* k = ffn_tc_kernel<__nv_bfloat16, kStore>;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, k, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = sm_count() / 2;
  }
  cached[dev] = n;
  return n;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The matrix of an operand as a tensor map: 128-byte lines along its unit
// stride; `rows` of it in a box whose lines lie along the sum.
bool encode_operand(CUtensorMap* map, const FfnOperand& o, int64_t K, int rows) {
  const auto encode = tensor_map_encoder();
  if (!encode) return false;
  const bool mn = o.k_stride != 1;
  const int64_t inner = mn ? o.rows : K, outer = mn ? K : o.rows, ld = mn ? o.k_stride : o.row_stride;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(mn ? kDepth : rows)};
  const cuuint32_t ones[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(o.p), dims, strides, box, ones,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A result or slopes in boxes of `rows` x 32, the lines of 64 bytes swizzled.
bool encode_rows(CUtensorMap* map, void* p, int64_t M, int64_t N, int64_t ld, int rows) {
  const auto encode = tensor_map_encoder();
  if (!encode) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(M)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[2] = {32, static_cast<cuuint32_t>(rows)};
  const cuuint32_t ones[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

using Kernel = void (*)(TcMaps, TcArgs);
template <typename T> Kernel kernel_of(int epi) {
  return epi == kStore ? ffn_tc_kernel<T, kStore> : epi == kGlu ? ffn_tc_kernel<T, kGlu> : ffn_tc_kernel<T, kGluBwd>;
}

}  // namespace

// The width of a launch's tiles and the clusters that share the sum of one: as
// many as there are for every tile, each with at least 4 blocks (256 deep) of
// its own. A narrower tile where it leaves the clusters less to do: a block
// takes about 2 tile_n + 64 cycles. (fp16, y of 32,768 tokens from 1536: 128
// columns in 27.9 us with tiles of 128 against 29.1 with 256; 384 columns in
// 47.2 with 192 against 48.8.)
FfnTcPlan ffn_tc_plan(const FfnSize* sizes, int jobs, int64_t K, int terms) {
  const int64_t pairs = pairs_resident(), blocks = ceil_div(K, kDepth) * terms;
  FfnTcPlan best{};
  int64_t least = 0;
  for (int tile_n = kTileN; tile_n >= 128; tile_n -= 64) {
    int64_t tiles = 0;
    for (int j = 0; j < jobs; ++j) tiles += ceil_div(sizes[j].M, kTileM) * ceil_div(sizes[j].N, tile_n);
    int64_t splits = pairs / tiles < blocks / 4 ? pairs / tiles : blocks / 4;
    splits = splits < 1 ? 1 : splits > 32 ? 32 : splits;
    const int64_t cost = ceil_div(tiles * splits, pairs) * ceil_div(blocks, splits) * (2 * tile_n + 64);
    if (tile_n == kTileN || cost < least) {
      least = cost;
      best = {tile_n, static_cast<int>(splits)};
    }
  }
  return best;
}

int ffn_tc_launch(const FfnProduct* ps, int jobs, int dtype, float* parts, cudaStream_t s) {
  const FfnProduct& p = ps[0];
  const bool bf = dtype == HC_DTYPE_BF16;
  const Kernel kernel = bf ? kernel_of<__nv_bfloat16>(p.epilogue) : kernel_of<__half>(p.epilogue);
  // A call of the runtime before the first one of the driver's encoder: on a
  // thread that has made none (autograd's), the encoder finds no context.
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) != cudaSuccess) {
    cudaGetLastError();
    return HC_ERR_LAUNCH;
  }
  FfnSize sizes[kFfnMaxJobs];
  for (int j = 0; j < jobs; ++j) sizes[j] = {ps[j].M, ps[j].N};
  const FfnTcPlan plan = p.epilogue == kStore ? ffn_tc_plan(sizes, jobs, p.K, p.terms) : FfnTcPlan{kTileN, 1};
  const int rows_b = plan.tile_n / 2;
  TcMaps maps{};
  TcArgs a{};
  a.jobs = jobs;
  a.tile_n = plan.tile_n;
  a.splits = plan.splits;
  for (int j = 0; j < jobs; ++j) {
    const int nb = ps[j].epilogue == kGlu ? 2 : ps[j].terms;
    for (int t = 0; t < ps[j].terms; ++t)
      if (!encode_operand(&maps.a[j + t], ps[j].A[t], p.K, kRows)) return HC_ERR_LAUNCH;
    for (int t = 0; t < nb; ++t)
      if (!encode_operand(&maps.b[j + t], ps[j].B[t], p.K, rows_b)) return HC_ERR_LAUNCH;
    TcJob& job = a.job[j];
    job.M = ps[j].M; job.N = ps[j].N; job.ldo = ps[j].ldo; job.out = ps[j].out;
    job.tiles_m = static_cast<int>(ceil_div(job.M, kTileM));
    job.tiles_n = static_cast<int>(ceil_div(job.N, p.epilogue == kGlu ? kRows : plan.tile_n));
    // the hidden tensors' rows always start on 16-byte boundaries
    job.tma = job.ldo % 8 == 0;
    if (job.tma) {
      const FfnProduct& q = ps[j];
      void* const outs[3] = {q.out, q.epilogue == kGlu ? q.slope_gate : q.out2, q.epilogue == kGlu ? q.slope_up : nullptr};
      for (int k = 0; k < (q.epilogue == kStore ? 1 : 3); ++k)
        if (outs[k] && !encode_rows(&maps.out[j + k], outs[k], job.M, job.N, job.ldo, q.epilogue == kGluBwd ? kRows : 32))
          return HC_ERR_LAUNCH;
    }
    if (static_cast<int64_t>(job.tiles_m) * job.tiles_n > (int64_t(1) << 24)) return HC_ERR_BAD_SIZE;
    a.tiles += job.tiles_m * job.tiles_n;
  }
  if (p.epilogue == kGluBwd && (!encode_rows(&maps.in[0], p.slope_gate, p.M, p.N, p.ldo, kRows) ||
                                !encode_rows(&maps.in[1], p.slope_up, p.M, p.N, p.ldo, kRows)))
    return HC_ERR_LAUNCH;
  const CUtensorMap* all = reinterpret_cast<const CUtensorMap*>(&maps);
  for (size_t i = 0; i < sizeof(TcMaps) / sizeof(CUtensorMap); ++i) {
    const CUtensorMap none{};
    if (memcmp(all + i, &none, sizeof(none)) != 0) a.maps |= 1u << i;
  }
  a.slope_gate = p.slope_gate;
  if (a.splits > 1) {
    if (!parts) return HC_ERR_SCRATCH;
    float* at = parts;
    for (int j = 0; j < jobs; ++j) {
      a.job[j].parts = at;
      at += a.splits * ps[j].M * ps[j].N;
    }
  }
  a.blocks_term = static_cast<int>(ceil_div(p.K, kDepth));
  a.blocks = a.blocks_term * p.terms;
  a.a_mn = p.A[0].k_stride != 1;
  a.b_mn = p.B[0].k_stride != 1;
  a.act = p.act;
  a.wait_limit = wait_poll_limit();
  a.status = timeout_word(s);
  const int items = a.tiles * a.splits, pairs = items < pairs_resident() ? items : pairs_resident();
  if (int rc = ffn_launch(kernel, dim3(2 * pairs), kThreads, kSmemBytes, s, maps, a)) return rc;
  if (a.splits == 1) return HC_OK;
  FfnParts sums[kFfnMaxJobs];
  for (int j = 0; j < jobs; ++j) sums[j] = {a.job[j].parts, ps[j].out, ps[j].M * ps[j].N, false};
  return ffn_add_parts(sums, jobs, a.splits, dtype, s);
}

int ffn_add_parts(const FfnParts* jobs, int count, int splits, int dtype, cudaStream_t s) {
  AddJobs a{};
  a.jobs = count;
  a.splits = splits;
  int64_t most = 0;
  for (int j = 0; j < count; ++j) {
    a.job[j] = jobs[j];
    a.job[j].fours = jobs[j].count % 4 == 0 && aligned16(jobs[j].parts) && aligned16(jobs[j].out);
    const int64_t items = a.job[j].fours ? jobs[j].count / 4 : jobs[j].count;
    if (items > most) most = items;
  }
  const int64_t want = ceil_div(most, 256), cap = 8 * static_cast<int64_t>(sm_count());
  const int grid = static_cast<int>(want < cap ? want : cap);
  const auto kernel = dtype == HC_DTYPE_F32 ? add_parts_kernel<float> : dtype == HC_DTYPE_F16 ? add_parts_kernel<__half>
                                                                                              : add_parts_kernel<__nv_bfloat16>;
  return ffn_launch(kernel, dim3(grid), 256, 0, s, a);
}

unsigned int ffn_take_timeouts(bool reset) {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_ffn_wait_timeouts, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (reset && v != 0) {
    const unsigned int z = 0;
    cudaMemcpyToSymbol(g_ffn_wait_timeouts, &z, sizeof(z));
  }
  return v;
}

}  // namespace hc
