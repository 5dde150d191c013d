// What the two forms of the tree attention share (tree_kernels.cu, mma.sync;
// tree_umma.cu, tcgen05).
#pragma once
#include <cuda_runtime.h>

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

// Whether the tcgen05 form takes heads of these widths, and its launch.
bool tree_umma_takes(int int8, int rows, int qk, int vh, int piece);
int tree_umma_nsplit(int int8, int B, int rows, int kvh, int qk, int vh, int span);
cudaError_t launch_tree_umma(const TreeArgs& A, int int8, int B, cudaStream_t st);

}  // namespace nb
