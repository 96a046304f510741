// block.cuh — what the kernels of a layer's block share: arguments of the
// norm kernels (hc_read_norm, hc_mix_write_norm), the dropout bits, and the
// per-dtype launchers that block_capi.cu dispatches to.
#pragma once

#include "common.cuh"

namespace hc {

constexpr int kBlockMaxN = 8;  // streams
constexpr int kBlockMaxM = 4;  // backbone blocks

// ------------------------------------------------------------ dropout bits
// Philox 4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten rounds on a
// 128-bit counter with a 64-bit key that grows by two Weyl constants. The
// counter is (element / 4, offset), the key the seed, and element i takes word
// i % 4, so the bits depend on nothing but the element's place: the forward,
// the backward and every split of the work over threads draw the same ones.
struct DropArgs {
  const int64_t* state;  // device (seed, offset), or nullptr for the two below
  uint64_t seed, offset;
  uint32_t below;      // floor(p 2^32) - 1: an element is kept when its word is above
  float scale;         // 1 / (1 - p); 0 at p = 1
  int on;              // floor(p 2^32) > 0; else nothing is dropped
};

struct DropKey {
  uint32_t k0, k1, o0, o1;
};

__device__ __forceinline__ DropKey drop_key(const DropArgs& a) {
  uint64_t seed = a.seed, offset = a.offset;
  if (a.state) {
    seed = static_cast<uint64_t>(a.state[0]);
    offset = static_cast<uint64_t>(a.state[1]);
  }
  return DropKey{static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), static_cast<uint32_t>(offset),
                 static_cast<uint32_t>(offset >> 32)};
}

// The ten round keys. A kernel that draws many blocks makes them once.
struct RoundKeys {
  uint32_t a[10], b[10];
  __device__ __forceinline__ explicit RoundKeys(const DropKey& k) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      a[r] = k.k0 + r * 0x9E3779B9u;
      b[r] = k.k1 + r * 0xBB67AE85u;
    }
  }
};

__device__ __forceinline__ uint4 philox4(const RoundKeys& k, uint32_t o0, uint32_t o1, uint64_t block) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = o0, c3 = o1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c0, p1 = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k.a[r];
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k.b[r];
    c3 = static_cast<uint32_t>(p0);
  }
  return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ uint4 philox4(const DropKey& key, uint64_t block) {
  return philox4(RoundKeys(key), key.o0, key.o1, block);
}

// The word of one element.
__device__ __forceinline__ uint32_t philox_word(const DropKey& key, uint64_t i) {
  const uint4 w = philox4(key, i >> 2);
  const uint32_t r = static_cast<uint32_t>(i) & 3u;
  return r == 0 ? w.x : r == 1 ? w.y : r == 2 ? w.z : w.w;
}

// A dropped value is 0 whatever it was (an infinity or a NaN too), so it is
// selected, not multiplied.
__device__ __forceinline__ float drop_value(const DropArgs& a, uint32_t word, float v) {
  return word > a.below ? v * a.scale : 0.f;
}

// ------------------------------------------------------------ norm kernels
struct NormArgs {
  const void* x;     // [T, n, D]
  const void* g;     // upstream gradient: [T, m, D] (read), [T, n, D] (mix-write)
  const void* f;     // [T, m, D] (mix-write)
  const void* gate;  // [T, m, D] or nullptr
  const float* R;    // [T, m, n] (read)
  const float* H;    // [T, n, n] (mix-write)
  const float* W;    // [T, n, m] (mix-write)
  const float* v;    // [T, n] or nullptr
  const float *weight, *bias, *scale;  // [m D] or nullptr
  void* out;                           // y (read) or x' (mix-write)
  float* stats;                        // [T, 2]: mean, 1 / root
  void *grad_x, *grad_f, *grad_gate;
  float *grad_R, *grad_H, *grad_W, *grad_v;
  float* partial;  // [rows][2][m D]: the groups' sums over their tokens, or nullptr
  int64_t T, D;
  int n, m, norm, gate_act;
  float eps;
  DropArgs drop;
};

// Which kernels a call takes, and over how many CTAs.
struct NormGeometry {
  int warps;   // warps of one token's group (the 8-column kernels); 0 = element by element
  int chunks;  // 8-column chunks a thread owns (forward)
  bool ragged; // rows that are not whole chunks on 16-byte boundaries
  bool wide;   // kernels for more threads
  int grid;    // CTAs
  int rows;    // rows of `partial` that are written
};

// Launchers of one stream dtype; the 8-column ones set grid and rows.
#define HC_BLOCK_DECL(SFX)                                                                     \
  int read_norm_launch_##SFX(bool bwd, NormGeometry& g, const NormArgs& a, cudaStream_t s);     \
  int write_norm_launch_##SFX(bool bwd, NormGeometry& g, const NormArgs& a, cudaStream_t s);    \
  int dropout_launch_##SFX(const void* x, void* y, int64_t N, const DropArgs& d, cudaStream_t s);
HC_BLOCK_DECL(f32)
HC_BLOCK_DECL(f16)
HC_BLOCK_DECL(bf16)
#undef HC_BLOCK_DECL

// grad_weight, grad_bias and grad_scale from the CTAs' sums (block_capi.cu).
int norm_param_grads(const float* partial, int rows, int64_t E, const float* weight, const float* bias,
                     const float* scale, float* grad_weight, float* grad_bias, float* grad_scale, cudaStream_t s);

}  // namespace hc
