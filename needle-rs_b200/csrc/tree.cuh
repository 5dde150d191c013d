// What the two forms of the tree attention share (tree_kernels.cu, mma.sync;
// tree_umma.cu, tcgen05).
#pragma once
#include <cuda_runtime.h>

#include "common.cuh"
#include "fastdiv.hpp"

namespace nb {

struct TreeArgs {
  const float* q;
  long ldq;
  const char *k, *v;       // ring [B][slots][kvh][qk | vh]
  const float *ks, *vs;    // [B][slots][kvh]
  const char *tk, *tv;     // draft [B][T][kvh][qk | vh]
  const float *tks, *tvs;  // [B][T][kvh]
  const int *lo, *hi;      // [B][T]
  const uint32_t* mask;    // [B][T][words] or null: a chain
  int slots, T, heads, kvh, rep, qk, vh, words;
  int drafted;             // T when the draft's keys are given, else 0
  int nsplit;
  float scale;             // log2(e) / sqrt(qk)
  FastDiv by_rep;
  float* out;              // [B][T][heads][vh]
  float* part;             // [B][kvh][nsplit][T * rep][vh + 2] when nsplit > 1
};

// A product of a scaled query and codes is up to 2^28: times a key scale above this
// it could pass the range before the query's power of two is taken back.
constexpr float KEY_SCALE_FAR = 0x1p96f;

// 2^x, relative error about 2^-22; arguments here are <= 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The arguments of the sessions from b0 on (a grid axis holds 65535 of them).
inline TreeArgs tree_sessions(const TreeArgs& A, int b0, int es) {
  TreeArgs C = A;
  const size_t ring = (size_t)b0 * A.slots * A.kvh, draft = (size_t)b0 * A.T * A.kvh;
  C.q += (size_t)b0 * A.T * A.ldq;
  C.k += ring * A.qk * es, C.v += ring * A.vh * es;
  if (A.ks) C.ks += ring, C.vs += ring;
  if (A.drafted) {
    C.tk += draft * A.qk * es, C.tv += draft * A.vh * es;
    if (A.tks) C.tks += draft, C.tvs += draft;
  }
  C.lo += (size_t)b0 * A.T, C.hi += (size_t)b0 * A.T;
  if (A.mask) C.mask += (size_t)b0 * A.T * A.words;
  C.out += (size_t)b0 * A.T * A.heads * A.vh;
  if (A.part) C.part += (size_t)b0 * A.kvh * A.nsplit * A.T * A.rep * (A.vh + 2);
  return C;
}

// Bits [a, b) of a 32-bit word.
__device__ __forceinline__ uint32_t bit_range(int a, int b) {
  const uint32_t hi = b >= 32 ? 0xffffffffu : b <= 0 ? 0u : (1u << b) - 1u;
  const uint32_t lo = a >= 32 ? 0xffffffffu : a <= 0 ? 0u : (1u << a) - 1u;
  return hi & ~lo;
}

// Where position v of a call lies: the draft's nodes come first, the ring's
// offsets after them.
struct TreePlace {
  size_t ring, draft;  // first row (position * kvh + kh) of the session in each
  int drafted, slot0, slots, kvh, total;
  __device__ __forceinline__ bool in_draft(int v) const { return v < drafted; }
  __device__ __forceinline__ size_t row(int v) const {
    if (v < drafted) return draft + (size_t)v * kvh;
    int s = slot0 + (v - drafted);
    if (s >= slots) s -= slots;
    return ring + (size_t)s * kvh;
  }
  // Whether positions v .. v + n - 1 are ring places one after another.
  __device__ __forceinline__ bool plain(int v, int n) const {
    const int s = slot0 + (v - drafted);
    return v >= drafted && v + n <= total && (s + n <= slots || s >= slots);
  }
};

// What row `node` sees of positions v0 .. v0 + 31.
__device__ __forceinline__ uint32_t tree_sees(const TreeArgs& A, size_t node_at, int node, int start, int cnt,
                                              int n_ring, int v0) {
  uint32_t w = 0;
  if (v0 < A.drafted) {
    w = A.mask ? __ldg(A.mask + node_at * A.words + (v0 >> 5)) : bit_range(0, node - v0 + 1);
    w &= bit_range(0, A.drafted - v0);
  }
  const int o = A.drafted - v0;  // ring offset 0 is bit o
  if (o < 32) {
    w |= bit_range(o + start, o + min(start + cnt, n_ring));
    if (start + cnt > A.slots) w |= bit_range(o, (int)((uint32_t)o + start + cnt - A.slots));  // the sum may pass 2^31
  }
  return w;
}

// One row over positions [v0, v1) by a warp, in f32 from the cache itself: the
// rows whose keys, values or scales split operands cannot hold. Adds them to the
// row's running log2 max, sum, and dims lane + 32 j of the output.
template <bool I8>
__device__ __forceinline__ void tree_slow_row(const TreeArgs& A, const TreePlace& P, size_t node_at, int node,
                                              int head, int start, int cnt, int n_ring, int v0, int v1, float* m_run,
                                              float* l_run, float (&o)[4]) {
  const int lane = threadIdx.x & 31;
  const float* q = A.q + node_at * A.ldq + (size_t)head * A.qk;
  float m = *m_run, l = *l_run;
  for (int base = v0 & ~31; base < v1; base += 32) {
    const int v = base + lane;
    const bool on = v >= v0 && v < v1 && ((tree_sees(A, node_at, node, start, cnt, n_ring, base) >> lane) & 1);
    float s = -INFINITY;
    if (on) {
      const size_t r = P.row(v);
      const bool d = P.in_draft(v);
      s = 0.f;
      if (I8) {
        const int8_t* k = (const int8_t*)(d ? A.tk : A.k) + r * A.qk;
        const float sc = (d ? A.tks : A.ks)[r];
        for (int i = 0; i < A.qk; ++i) s = fmaf(q[i], (float)k[i], s);
        s *= sc;
      } else {
        const float* k = (const float*)(d ? A.tk : A.k) + r * A.qk;
        for (int i = 0; i < A.qk; ++i) s = fmaf(q[i], k[i], s);
      }
      s *= A.scale;
    }
    const float mn = fmaxf(m, warp_max(s));
    const float mz = mn == -INFINITY ? 0.f : mn;
    const float corr = ex2(m - mz), p = on ? ex2(s - mz) : 0.f;
    m = mn;
    l = l * corr + warp_sum(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] *= corr;
    for (int i = 0; i < 32; ++i) {
      const float w = __shfl_sync(0xffffffffu, p, i);
      if (w == 0.f) continue;  // the same for every lane
      const size_t r = P.row(base + i);
      const bool d = P.in_draft(base + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = lane + 32 * j;
        if (e >= A.vh) continue;
        const float x = I8 ? (float)((const int8_t*)(d ? A.tv : A.v))[r * A.vh + e] * (d ? A.tvs : A.vs)[r]
                           : ((const float*)(d ? A.tv : A.v))[r * A.vh + e];
        o[j] = fmaf(w, x, o[j]);
      }
    }
  }
  *m_run = m;
  *l_run = l;
}

// Whether the tcgen05 form takes heads of these widths, and its launch.
bool tree_umma_takes(int int8, int rows, int qk, int vh, int piece);
int tree_umma_nsplit(int int8, int B, int rows, int kvh, int qk, int vh, int span);
cudaError_t launch_tree_umma(const TreeArgs& A, int int8, int B, cudaStream_t st);

}  // namespace nb
