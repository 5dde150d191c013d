// Corrections of a row of logits before a token is picked: nd_logits_adjust.
// The engine's constrained text path masks and picks on the host one row at a
// time; this is the device form for many rows.
#include <cooperative_groups.h>

#include "kernels.hpp"
#include "launch_util.hpp"

namespace nb {
namespace {

namespace cg = cooperative_groups;

constexpr int LG_THREADS = 256;
constexpr int LG_CHUNK = 4096;      // ids a block corrects at a time
constexpr uint32_t LG_SEEN = 1u << 31;  // token of the history; the low bits count the generated ones

struct LogitArgs {
  const float* x;
  float* y;
  long ldx, ldy;
  int vocab, chunk, loops;
  const int *hist, *hist_off, *gen_from;
  const float *rep, *pres, *freq;
  const int* bias_ids;
  const float* bias_vals;
  const int* bias_off;
  const uint32_t* mask;
  long mask_ld;
  float masked;
  uint32_t* picks;
};

// One row's value: penalties of a seen token, then its bias.
__device__ __forceinline__ float adjust(float x, uint32_t n, float bias, float rep, float pres, float freq) {
  if (n) {
    x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
    const uint32_t c = n & ~LG_SEEN;
    if (c) x -= (float)c * freq + pres;
  }
  return x + bias;
}

// Grid (cluster size, rows): the blocks of a cluster share a row. Per chunk of
// ids a block counts the row's history and sums its biases in shared memory
// (counts are whole numbers, so their atomics' order is no matter; biases are
// added in list order by one warp), then streams the logits once: 8 bytes per
// logit bound it, the mask is one bit and the history 4 bytes per chunk.
template <bool BIAS>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const LogitArgs A) {
  extern __shared__ __align__(16) uint32_t cnt[];  // [chunk + 4], then the biases
  __shared__ unsigned long long best_of[LG_THREADS / 32];
  __shared__ unsigned long long block_best;
  float* bias = reinterpret_cast<float*>(cnt + A.chunk + 4);
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const float* x = A.x + (size_t)row * A.ldx;
  float* y = A.y + (size_t)row * A.ldy;
  const uint32_t* mask = A.mask ? A.mask + (size_t)row * A.mask_ld : nullptr;
  const float rep = A.rep ? A.rep[row] : 1.f, pres = A.pres ? A.pres[row] : 0.f, freq = A.freq ? A.freq[row] : 0.f;
  const int h0 = A.hist ? A.hist_off[row] : 0, h1 = A.hist ? A.hist_off[row + 1] : 0;
  const int gen = A.hist && A.gen_from ? A.gen_from[row] : h0;
  const int b0 = BIAS ? A.bias_off[row] : 0, b1 = BIAS ? A.bias_off[row + 1] : 0;
  // Row elements before the first 16-byte boundary of x; wide accesses need y
  // to have as many.
  const int skew = (int)(((uintptr_t)x >> 2) & 3);
  const bool wide = skew == (int)(((uintptr_t)y >> 2) & 3);
  float best = -INFINITY;
  int at = 0x7fffffff;

  for (int l = 0; l < A.loops; ++l) {
    const long c0l = ((long)l * gridDim.x + blockIdx.x) * A.chunk;
    if (c0l >= A.vocab) break;  // block-uniform; the cluster meets again below
    const int c0 = (int)c0l, c1 = min(A.vocab, c0 + A.chunk);
    __syncthreads();
    for (int i = tid; i < (A.chunk + 4) / 4; i += LG_THREADS) {
      reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
      if (BIAS) reinterpret_cast<float4*>(bias)[i] = make_float4(0, 0, 0, 0);
    }
    __syncthreads();
    // Shared index of id c0 + j is j + skew (chunks are multiples of 4, so the
    // wide accesses below are aligned in both).
    for (int i = h0 + tid; i < h1; i += LG_THREADS) {
      const uint32_t j = (uint32_t)A.hist[i] - (uint32_t)c0;
      if (j < (uint32_t)(c1 - c0)) {
        if (i >= gen) atomicAdd(&cnt[j + skew], 1u);
        else atomicOr(&cnt[j + skew], LG_SEEN);
      }
    }
    if (BIAS && tid < 32) {
      for (int i0 = b0; i0 < b1; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t j = i < b1 ? (uint32_t)A.bias_ids[i] - (uint32_t)c0 : 0xffffffffu;
        bool todo = i < b1 && j < (uint32_t)(c1 - c0);
        const float val = todo ? A.bias_vals[i] : 0.f;
        // One id several times: one entry a turn, the earliest first.
        while (__any_sync(0xffffffffu, todo)) {
          const unsigned same = __match_any_sync(0xffffffffu, todo ? j : 0xffffffffu);
          if (todo && __ffs(same) - 1 == lane) {
            bias[j + skew] += val;
            todo = false;
          }
          __syncwarp();
        }
      }
    }
    __syncthreads();
    auto one = [&](int id) {
      const int s = id - c0 + skew;
      float v = adjust(x[id], cnt[s], BIAS ? bias[s] : 0.f, rep, pres, freq);
      if (mask && !((__ldg(mask + (id >> 5)) >> (id & 31)) & 1)) v = A.masked;
      y[id] = v;
      if (v > best) best = v, at = id;
    };
    if (wide) {
      // Chunk piece j covers ids c0 - skew + 4j .. + 3; those outside [c0, c1)
      // go one by one.
      const int n4 = (c1 - c0 + skew + 3) / 4;
#pragma unroll 2
      for (int j = tid; j < n4; j += LG_THREADS) {
        const int id = c0 - skew + 4 * j;
        if (id < c0 || id + 4 > c1) {
          for (int e = max(id, c0); e < min(id + 4, c1); ++e) one(e);
          continue;
        }
        const float4 f = *reinterpret_cast<const float4*>(x + id);
        const uint4 n = *reinterpret_cast<const uint4*>(cnt + 4 * j);
        float4 b = make_float4(0, 0, 0, 0);
        if (BIAS) b = *reinterpret_cast<const float4*>(bias + 4 * j);
        float r[4] = {adjust(f.x, n.x, b.x, rep, pres, freq), adjust(f.y, n.y, b.y, rep, pres, freq),
                      adjust(f.z, n.z, b.z, rep, pres, freq), adjust(f.w, n.w, b.w, rep, pres, freq)};
        if (mask) {
          const int w = id >> 5, sh = id & 31;
          const uint32_t lo = __ldg(mask + w), hi = sh > 28 ? __ldg(mask + w + 1) : 0u;
          const uint32_t bits = __funnelshift_r(lo, hi, sh);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((bits >> e) & 1)) r[e] = A.masked;
        }
        *reinterpret_cast<float4*>(y + id) = make_float4(r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r[e] > best) best = r[e], at = id + e;
      }
    } else {
      for (int id = c0 + tid; id < c1; id += LG_THREADS) one(id);
    }
  }
  if (!A.picks) return;
  // First maximum of the row: the largest key over the block, then the cluster.
  unsigned long long key = at != 0x7fffffff ? argmax_key(best, (uint32_t)at) : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
    key = other > key ? other : key;
  }
  if (lane == 0) best_of[tid >> 5] = key;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < LG_THREADS / 32; ++w) key = best_of[w] > key ? best_of[w] : key;
    block_best = key;
  }
  if (gridDim.x == 1) {
    if (tid == 0) A.picks[row] = argmax_pick(key);
    return;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  if (blockIdx.x == 0 && tid == 0) {
    for (unsigned r = 1; r < gridDim.x; ++r) {
      const unsigned long long other = *cl.map_shared_rank(&block_best, r);
      key = other > key ? other : key;
    }
    A.picks[row] = argmax_pick(key);
  }
  cl.sync();  // no block leaves while its key may be read
}

}  // namespace

cudaError_t launch_logits_adjust(const float* x, int ldx, int rows, int vocab, float* y, int ldy, const int* hist,
                                 const int* hist_off, const int* gen_from, const float* rep, const float* pres,
                                 const float* freq, const int* bias_ids, const float* bias_vals, const int* bias_off,
                                 const uint32_t* mask, int mask_ld, float masked, uint32_t* picks, cudaStream_t st) {
  if (rows <= 0) return cudaSuccess;
  LogitArgs A{x, y, ldx, ldy, vocab, 0, 0, hist, hist_off, gen_from, rep, pres, freq,
              bias_ids, bias_vals, bias_off, mask, mask_ld, masked, picks};
  // Blocks per row: one per 1024 ids, at most 8 (a portable cluster); each
  // takes its share in equal chunks of at most LG_CHUNK ids.
  int blocks = 1;
  while (blocks < 8 && vocab > 1024 * blocks) blocks *= 2;
  A.loops = (int)((vocab + (long)LG_CHUNK * blocks - 1) / ((long)LG_CHUNK * blocks));
  const long parts = (long)A.loops * blocks;
  A.chunk = (int)(((vocab + parts - 1) / parts + 3) / 4 * 4);
  const size_t smem = (size_t)(A.chunk + 4) * 4 * (bias_ids ? 2 : 1);
  auto kern = bias_ids ? logits_kernel<true> : logits_kernel<false>;
  for (int r0 = 0; r0 < rows; r0 += 65535) {  // grid limit of the row axis
    const int n = rows - r0 < 65535 ? rows - r0 : 65535;
    LogitArgs B = A;
    B.x += (size_t)r0 * ldx;
    B.y += (size_t)r0 * ldy;
    if (hist) B.hist_off += r0;
    if (gen_from) B.gen_from += r0;
    if (rep) B.rep += r0;
    if (pres) B.pres += r0;
    if (freq) B.freq += r0;
    if (bias_off) B.bias_off += r0;
    if (mask) B.mask += (size_t)r0 * mask_ld;
    if (picks) B.picks += r0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, n);
    cfg.blockDim = dim3(LG_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = blocks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, B);
    if (e != cudaSuccess) return e;
  }
  return cudaGetLastError();
}

}  // namespace nb
