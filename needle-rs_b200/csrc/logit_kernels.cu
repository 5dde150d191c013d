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
constexpr int LG_FLIGHT = 2;        // pieces of four logits a thread holds
constexpr int LG_CHUNK = 12800;     // ids a block corrects at a time: four blocks' marks fit an SM
// Marks of an id: in the history, with a bias (and which entry of the list in
// shared memory holds its sum); the low bits count its generated occurrences.
constexpr uint32_t LG_SEEN = 1u << 31, LG_BIASED = 1u << 30, LG_COUNT = (1u << 22) - 1;
constexpr int LG_ENTRY = 22;  // bit of the entry's number
constexpr int LG_LIST = 256;  // biases of a row that shared memory holds (eight bits of a mark)

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

// One row's value: the penalties of a seen token, then the sum of its biases
// (bval; with more than LG_LIST in the row, summed from the list itself).
template <bool BIAS>
__device__ __forceinline__ float adjust(float x, uint32_t n, int id, float rep, float pres, float freq, const float* bval,
                                     const int* list, const float* vals, int nb) {
  const uint32_t c = n & LG_COUNT;
  if (c || (n & LG_SEEN)) x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
  if (c) x -= (float)c * freq + pres;
  if (BIAS && (n & LG_BIASED)) {
    float sum = 0.f;
    if (nb <= LG_LIST)
      sum = bval[(n >> LG_ENTRY) & (LG_LIST - 1)];
    else
      for (int k = 0; k < nb; ++k)
        if (list[k] == id) sum += vals[k];
    x += sum;
  }
  return x;
}

// Grid (cluster size, rows): the blocks of a cluster share a row. Per chunk of
// ids a block counts the row's history in shared memory (whole numbers: the
// order of their atomics is no matter) and marks the ids with a bias, then
// streams the logits, LG_FLIGHT pieces of four a thread on their way while the
// ones before are stored, the first while the marks are made. The stream masks
// only: the marked ids, which are few, follow, each by the thread that takes its
// mark away, and until then stay out of the running maximum. 8 bytes per logit
// bound it, the mask is one bit; the history costs 8 bytes per id and block. 256
// rows of 100003: 72 us (2.9 TB/s), of which the stream alone takes 51; 8 rows of
// 8192: 8.
template <bool BIAS>
__global__ void __launch_bounds__(LG_THREADS, 4) logits_kernel(const LogitArgs A) {
  extern __shared__ __align__(16) uint32_t cnt[];  // [chunk + 32], none without history and biases
  __shared__ unsigned long long best_of[LG_THREADS / 32];
  __shared__ unsigned long long of_rank[8];  // block 0 of a cluster: every block's best
  __shared__ __align__(16) int bid[BIAS ? LG_LIST : 4];
  __shared__ __align__(16) float braw[BIAS ? LG_LIST : 4];
  __shared__ float bval[BIAS ? LG_LIST : 1];  // an id's sum at its first entry
  if (gridDim.x > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const float* x = A.x + (size_t)row * A.ldx;
  float* y = A.y + (size_t)row * A.ldy;
  const uint32_t* mask = A.mask ? A.mask + (size_t)row * A.mask_ld : nullptr;
  const float rep = A.rep ? A.rep[row] : 1.f, pres = A.pres ? A.pres[row] : 0.f, freq = A.freq ? A.freq[row] : 0.f;
  const int h0 = A.hist ? A.hist_off[row] : 0, h1 = A.hist ? A.hist_off[row + 1] : 0;
  const int gen = A.hist && A.gen_from ? A.gen_from[row] : h0;
  const int b0 = BIAS ? A.bias_off[row] : 0, nb = BIAS ? A.bias_off[row + 1] - b0 : 0;
  const int* list = BIAS ? A.bias_ids + b0 : nullptr;
  const float* vals = BIAS ? A.bias_vals + b0 : nullptr;
  const bool marks = A.hist || BIAS;
  // Row elements after the last 128-byte boundary before x, so that a warp's
  // accesses are whole lines; wide ones need y on a 16-byte boundary with it.
  const int skew = (int)(((uintptr_t)x >> 2) & 31);
  const bool wide = (skew & 3) == (int)(((uintptr_t)y >> 2) & 3);
  float best = -INFINITY;
  int at = 0x7fffffff;

  for (int l = 0; l < A.loops; ++l) {
    const long c0l = ((long)l * gridDim.x + blockIdx.x) * A.chunk;
    if (c0l >= A.vocab) break;  // block-uniform; the cluster meets again below
    const int c0 = (int)c0l, c1 = min(A.vocab, c0 + A.chunk);
    // Piece j covers ids c0 - skew + 4j .. + 3; those outside [c0, c1) go one by one.
    const int n4 = wide ? (c1 - c0 + skew + 3) / 4 : 0;
    float4 f[LG_FLIGHT];
    uint32_t lo[LG_FLIGHT], hi[LG_FLIGHT];  // the mask's words around a piece's bits
    auto load = [&](int j0) {  // nothing here waits for a load
#pragma unroll
      for (int u = 0; u < LG_FLIGHT; ++u) {
        const int id = c0 - skew + 4 * (j0 + u * LG_THREADS);
        const bool whole = id >= c0 && id + 4 <= c1;
        f[u] = whole ? *reinterpret_cast<const float4*>(x + id) : make_float4(0.f, 0.f, 0.f, 0.f);
        if (mask) {
          const int w = max(min(id, A.vocab - 1), 0) >> 5;
          lo[u] = __ldg(mask + w);
          hi[u] = __ldg(mask + min(w + 1, (A.vocab - 1) >> 5));
        }
      }
    };
    load(tid);
    if (marks) {
      if (l) __syncthreads();
      for (int i = tid; i < (A.chunk + 32) / 4; i += LG_THREADS) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
      if (BIAS && l == 0 && tid < nb && nb <= LG_LIST) bid[tid] = list[tid], braw[tid] = vals[tid];
      __syncthreads();
      // Shared index of id c0 + j is j + skew (chunks are multiples of 32, so the
      // wide accesses below are aligned in both).
      for (int i = h0 + tid; i < h1; i += LG_THREADS) {
        const uint32_t j = (uint32_t)A.hist[i] - (uint32_t)c0;
        if (j < (uint32_t)(c1 - c0)) {
          if (i >= gen) atomicAdd(&cnt[j + skew], 1u);
          else atomicOr(&cnt[j + skew], LG_SEEN);
        }
      }
      if (BIAS) {
        static_assert(LG_LIST <= LG_THREADS, "a thread an entry");
        if (nb <= LG_LIST) {
          // The first entry of an id sums them in list order (all threads read the same entries).
          if (tid < nb) {
            const int id = bid[tid];
            bool first = true;
            float sum = 0.f;
            for (int k = 0; k < nb; k += 4) {
              const int4 o = *reinterpret_cast<const int4*>(bid + k);
              const float4 w = *reinterpret_cast<const float4*>(braw + k);
              first &= !(o.x == id && k < tid) && !(o.y == id && k + 1 < tid) && !(o.z == id && k + 2 < tid) &&
                       !(o.w == id && k + 3 < tid);
              if (o.x == id) sum += w.x;
              if (o.y == id && k + 1 < nb) sum += w.y;
              if (o.z == id && k + 2 < nb) sum += w.z;
              if (o.w == id && k + 3 < nb) sum += w.w;
            }
            const uint32_t j = (uint32_t)id - (uint32_t)c0;
            if (first && j < (uint32_t)(c1 - c0)) {
              bval[tid] = sum;
              atomicOr(&cnt[j + skew], LG_BIASED | (uint32_t)tid << LG_ENTRY);
            }
          }
        } else {
          for (int i = tid; i < nb; i += LG_THREADS) {
            const uint32_t j = (uint32_t)list[i] - (uint32_t)c0;
            if (j < (uint32_t)(c1 - c0)) atomicOr(&cnt[j + skew], LG_BIASED);
          }
        }
      }
      __syncthreads();
    }
    auto allowed = [&](int id) { return !mask || ((__ldg(mask + (id >> 5)) >> (id & 31)) & 1); };
    auto one = [&](int id) {
      const float v = allowed(id) ? x[id] : A.masked;
      y[id] = v;
      if (v > best && !(marks && cnt[id - c0 + skew])) best = v, at = id;  // a thread's ids ascend
    };
    for (int j0 = tid; j0 < n4; j0 += LG_THREADS * LG_FLIGHT) {
      float4 g[LG_FLIGHT];
      uint32_t ok[LG_FLIGHT];
#pragma unroll
      for (int u = 0; u < LG_FLIGHT; ++u)
        g[u] = f[u], ok[u] = __funnelshift_r(lo[u], hi[u], (c0 - skew + 4 * (j0 + u * LG_THREADS)) & 31);
      load(j0 + LG_THREADS * LG_FLIGHT);
#pragma unroll
      for (int u = 0; u < LG_FLIGHT; ++u) {
        const int j = j0 + u * LG_THREADS, id = c0 - skew + 4 * j;
        if (j >= n4) continue;
        if (id < c0 || id + 4 > c1) {
          for (int e = max(id, c0); e < min(id + 4, c1); ++e) one(e);
          continue;
        }
        if (mask) {
          g[u].x = ok[u] & 1 ? g[u].x : A.masked;
          g[u].y = ok[u] & 2 ? g[u].y : A.masked;
          g[u].z = ok[u] & 4 ? g[u].z : A.masked;
          g[u].w = ok[u] & 8 ? g[u].w : A.masked;
        }
        *reinterpret_cast<float4*>(y + id) = g[u];
        if (marks) {
          const uint4 n = *reinterpret_cast<const uint4*>(cnt + 4 * j);
          g[u].x = n.x ? -INFINITY : g[u].x;
          g[u].y = n.y ? -INFINITY : g[u].y;
          g[u].z = n.z ? -INFINITY : g[u].z;
          g[u].w = n.w ? -INFINITY : g[u].w;
        }
        const float top = fmaxf(fmaxf(g[u].x, g[u].y), fmaxf(g[u].z, g[u].w));
        if (top > best) {
          best = top;
          at = id + (g[u].x == top ? 0 : g[u].y == top ? 1 : g[u].z == top ? 2 : 3);
        }
      }
    }
    if (!wide)
      for (int id = c0 + tid; id < c1; id += LG_THREADS) one(id);
    if (marks) {
      __syncthreads();
      auto marked = [&](int id) {  // the first to come takes the mark and the id
        const uint32_t j = (uint32_t)id - (uint32_t)c0;
        if (j >= (uint32_t)(c1 - c0)) return;
        const uint32_t n = atomicExch(&cnt[j + skew], 0u);
        if (!n) return;
        float v = y[id];
        if (allowed(id)) {
          v = adjust<BIAS>(v, n, id, rep, pres, freq, bval, list, vals, nb);
          y[id] = v;
        }
        if (v > best || (v == best && id < at && at != 0x7fffffff)) best = v, at = id;
      };
      for (int i = h0 + tid; i < h1; i += LG_THREADS) marked(A.hist[i]);
      if (BIAS)
        for (int i = tid; i < nb; i += LG_THREADS) marked(nb <= LG_LIST ? bid[i] : list[i]);
    }
  }
  // First maximum of the row: the largest key over the block, then the cluster.
  unsigned long long key = at != 0x7fffffff ? argmax_key(best, (uint32_t)at) : 0ull;
  if (A.picks) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      key = other > key ? other : key;
    }
    if (lane == 0) best_of[tid >> 5] = key;
    __syncthreads();
    if (tid == 0)
      for (int w = 1; w < LG_THREADS / 32; ++w) key = best_of[w] > key ? best_of[w] : key;
  }
  if (gridDim.x == 1) {
    if (A.picks && tid == 0) A.picks[row] = argmax_pick(key);
    return;
  }
  // Every block of the cluster runs (the arrival at the top): its key goes to
  // block 0, which alone waits for the others'.
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (!A.picks) return;
  cg::cluster_group cl = cg::this_cluster();
  if (tid == 0) *cl.map_shared_rank(&of_rank[blockIdx.x], 0) = key;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if (blockIdx.x != 0) return;
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid == 0) {
    for (unsigned r = 0; r < gridDim.x; ++r) key = of_rank[r] > key ? of_rank[r] : key;
    A.picks[row] = argmax_pick(key);
  }
}

}  // namespace

cudaError_t launch_logits_adjust(const float* x, int ldx, int rows, int vocab, float* y, int ldy, const int* hist,
                                 const int* hist_off, const int* gen_from, const float* rep, const float* pres,
                                 const float* freq, const int* bias_ids, const float* bias_vals, const int* bias_off,
                                 const uint32_t* mask, int mask_ld, float masked, uint32_t* picks, cudaStream_t st) {
  if (rows <= 0) return cudaSuccess;
  LogitArgs A{x, y, ldx, ldy, vocab, 0, 0, hist, hist_off, gen_from, rep, pres, freq,
              bias_ids, bias_vals, bias_off, mask, mask_ld, masked, picks};
  // Blocks per row, at most 8 (a portable cluster), each with its share in equal
  // chunks of at most LG_CHUNK ids: every one reads the row's history, so more
  // only while SMs are free (two a SM of 1024 ids, four of 8192) or the turns
  // become many. Measured (blocks: us):
  //     8 x 8192     1: 10.0  2: 8.5   4: 8.3   8: 7.8
  //    64 x 8192     1: 10.5  2: 8.5   4: 8.5   8: 9.7
  //   256 x 8192     1: 10.5  2: 12.3  4: 16.6  8: 25.0
  //    64 x 100003   1: 74.0  2: 40.9  4: 26.3  8: 20.8
  //   256 x 100003   1: 112   2: 73.5  4: 73.7  8: 75.8
  int blocks = 1;
  while (blocks < 8 && ((2l * rows * blocks <= 296 && vocab > 1024 * blocks) ||
                        (2l * rows * blocks <= 592 && vocab > 8192 * blocks) || vocab > 2 * LG_CHUNK * blocks))
    blocks *= 2;
  A.loops = (int)((vocab + (long)LG_CHUNK * blocks - 1) / ((long)LG_CHUNK * blocks));
  const long parts = (long)A.loops * blocks;
  A.chunk = (int)(((vocab + parts - 1) / parts + 31) / 32 * 32);
  const size_t smem = hist || bias_ids ? (size_t)(A.chunk + 32) * 4 : 0;
  auto kern = bias_ids ? logits_kernel<true> : logits_kernel<false>;
  cudaError_t e = allow_smem((const void*)kern, smem, true);
  if (e != cudaSuccess) return e;
  for (long r0 = 0; r0 < rows; r0 += 65535) {  // grid limit of the row axis
    const int n = (int)(rows - r0 < 65535 ? rows - r0 : 65535);
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
    e = cudaLaunchKernelEx(&cfg, kern, B);
    if (e != cudaSuccess) return e;
  }
  return cudaGetLastError();
}

}  // namespace nb
