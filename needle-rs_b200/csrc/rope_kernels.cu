// Rotary positions of any layout: nd_rope. The forward's own rotation (half
// layout over the whole head, table built at load, v3/model.rs:378-413) stays
// inside qkv_post; this is the standalone form for projections a caller keeps,
// with the pair layouts, partial heads and context scalings other callers use.
#include <cmath>

#include "kernels.hpp"
#include "fastdiv.hpp"

namespace nb {

// Frequencies in turns per position, in 64 bits: pair i of a token at position
// p is rotated by frac(p * turns[i]) turns. The product and its reduction stay
// in 64 bits because a 32-bit angle p * w has an absolute error of p * w *
// 2^-24, 0.06 rad at position 2^20; the reduced fraction (at most half a turn)
// is then exact enough in 32.
struct RopeFreqs {
  double turns[ROPE_MAX_ROT / 2];
  float m;    // factor of cos and sin
  float sgn;  // -1: the transpose, by the negative angle and the same m
};

// One block: `tok` tokens. Its threads first form the tokens' cosines and sines
// in shared memory (once per token and pair, shared by all heads), then stream
// the rows, ROPE_FLIGHT items a thread loaded before the first is stored. An
// item is the piece of a head that one thread takes:
//   VEC, half layout: float4 at pairs 4j.. and the float4 half a rotation on;
//   VEC, interleaved: one float4 (two pairs);
//   scalar: one pair.
// Items past the rotated part copy (there are none when y is x).
// Bytes bound it: 8 per value; see launch_rope for the figures.
constexpr int ROPE_FLIGHT = 4;

template <bool VEC, bool INTER>
__global__ void __launch_bounds__(256) rope_kernel(const float* x, long ldx, float* y, long ldy,
                                                   const int* __restrict__ pos, int M, int dim, int rot, int tok,
                                                   FastDiv per_head, FastDiv per_tok,
                                                   const __grid_constant__ RopeFreqs F) {
  extern __shared__ __align__(16) float cs[];  // [tok][rot / 2] cosines, then sines; then the positions
  const int half = rot >> 1;
  float* sn = cs + tok * half;
  int* at = reinterpret_cast<int*>(sn + tok * half);
  const int t0 = blockIdx.x * tok, nt = min(tok, M - t0);
  for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
    const int t = i / half, j = i - t * half;
    const int p = pos[t0 + t];
    if (j == 0) at[t] = p;
    const double turn = (double)p * F.turns[j];
    float s, c;
    sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
    cs[i] = c * F.m;
    sn[i] = s * F.m * F.sgn;
  }
  __syncthreads();
  const int total = nt * (int)per_tok.d;
  // Pieces of a head: rotating ones first, then copies.
  const int nrot = VEC ? (INTER ? rot >> 2 : half >> 2) : half;
  for (int base = threadIdx.x; base < total; base += blockDim.x * ROPE_FLIGHT) {
    float4 a[ROPE_FLIGHT], b[ROPE_FLIGHT];
    float* to[ROPE_FLIGHT];
    int sc[ROPE_FLIGHT];  // where the piece's cosines lie, -1 for a copy
#pragma unroll
    for (int u = 0; u < ROPE_FLIGHT; ++u) {
      const int it = base + u * blockDim.x;
      to[u] = nullptr;
      if (it >= total) continue;
      const int t = per_tok.div(it), r = it - t * (int)per_tok.d;
      if (at[t] < 0) continue;  // padding row: left as it is
      const int h = per_head.div(r), j = r - h * (int)per_head.d;
      const size_t from = (size_t)(t0 + t) * ldx + (size_t)h * dim;
      to[u] = y + (size_t)(t0 + t) * ldy + (size_t)h * dim;
      const bool turn = j < nrot;
      // offset of the piece in the head
      const int e = VEC ? (turn ? 4 * j : rot + 4 * (j - nrot)) : (turn ? (INTER ? 2 * j : j) : rot + (j - nrot));
      sc[u] = turn ? t * half + (VEC ? (INTER ? 2 * j : 4 * j) : j) : -1;
      to[u] += e;
      if (VEC) {
        a[u] = *reinterpret_cast<const float4*>(x + from + e);
        if (!INTER && turn) b[u] = *reinterpret_cast<const float4*>(x + from + e + half);
      } else {
        a[u].x = x[from + e];
        if (turn) b[u].x = x[from + e + (INTER ? 1 : half)];
      }
    }
#pragma unroll
    for (int u = 0; u < ROPE_FLIGHT; ++u) {
      if (!to[u]) continue;
      if (sc[u] < 0) {
        if (VEC) *reinterpret_cast<float4*>(to[u]) = a[u];
        else *to[u] = a[u].x;
        continue;
      }
      const float *c = cs + sc[u], *s = sn + sc[u];
      if (VEC && !INTER) {
        const float4 cc = *reinterpret_cast<const float4*>(c), ss = *reinterpret_cast<const float4*>(s);
        *reinterpret_cast<float4*>(to[u]) = make_float4(a[u].x * cc.x - b[u].x * ss.x, a[u].y * cc.y - b[u].y * ss.y,
                                                        a[u].z * cc.z - b[u].z * ss.z, a[u].w * cc.w - b[u].w * ss.w);
        *reinterpret_cast<float4*>(to[u] + half) =
            make_float4(a[u].x * ss.x + b[u].x * cc.x, a[u].y * ss.y + b[u].y * cc.y, a[u].z * ss.z + b[u].z * cc.z,
                        a[u].w * ss.w + b[u].w * cc.w);
      } else if (VEC) {
        const float2 cc = *reinterpret_cast<const float2*>(c), ss = *reinterpret_cast<const float2*>(s);
        *reinterpret_cast<float4*>(to[u]) =
            make_float4(a[u].x * cc.x - a[u].y * ss.x, a[u].x * ss.x + a[u].y * cc.x, a[u].z * cc.y - a[u].w * ss.y,
                        a[u].z * ss.y + a[u].w * cc.y);
      } else {
        const float p = a[u].x, q = b[u].x;
        to[u][0] = p * c[0] - q * s[0];
        to[u][INTER ? 1 : half] = p * s[0] + q * c[0];
      }
    }
  }
}

cudaError_t launch_rope(const float* x, int ldx, float* y, int ldy, const int* pos, int M, int heads, int dim, int rot,
                        double theta, bool interleaved, int kind, double factor, double trained, double fast,
                        double slow, float mscale, bool inverse, cudaStream_t st) {
  if (M <= 0) return cudaSuccess;
  RopeFreqs F;
  const double two_pi = 6.283185307179586476925;
  for (int i = 0; i < rot / 2; ++i) {
    double f = std::pow(theta, -2.0 * i / rot) / two_pi;
    if (kind == 1) {
      f /= factor;
    } else if (kind == 2) {
      // Turns the pair makes over the trained context: above `fast` it keeps
      // its frequency, below `slow` it is stretched, in between a blend.
      const double r = trained * f;
      const double keep = std::fmin(1.0, std::fmax(0.0, (r - slow) / (fast - slow)));
      f = f * keep + f / factor * (1.0 - keep);
    }
    F.turns[i] = f;
  }
  F.m = mscale;
  F.sgn = inverse ? -1.0f : 1.0f;
  const int half = rot / 2;
  const bool vec = dim % 4 == 0 && rot % 4 == 0 && (interleaved || half % 4 == 0) && ldx % 4 == 0 && ldy % 4 == 0 &&
                   ((uintptr_t)x | (uintptr_t)y) % 16 == 0;
  const int copy = x == y ? 0 : 1;
  const int nrot = vec ? (interleaved ? rot / 4 : half / 4) : half;
  const int nhead = nrot + (copy ? (dim - rot) / (vec ? 4 : 1) : 0);
  const long items = (long)heads * nhead;
  // Tokens per block: one while that leaves SMs idle, else enough for about
  // 1024 items (four per thread) and at most 8, so that cosines and sines are
  // formed by most threads at once. 16384 rows of 18 heads of 64, 32 rotated: 1
  // token a block 44 us, 2: 31, 4: 29, 8: 29 (5.3 TB/s of 6.6 for a copy); 64 rows
  // of 14 heads of 48 take 3.3 us on the GPU and 5.2 with the call. The half layout
  // over whole heads: 30.9 us, in place as well (in place, half of each head: 20.6);
  // 16384 rows of 14 heads of 48 20.6, in place 22.3 (13.4 us of bytes).
  int tok = 1;
  while (tok < 8 && (long)M > 592L * tok && items * tok < 1024) tok *= 2;
  const size_t smem = (size_t)tok * (rot + 1) * sizeof(float);
  const dim3 grid((M - 1) / tok + 1);
  const FastDiv ph(nhead), pt((uint32_t)items);
#define NB_ROPE(V, I) \
  rope_kernel<V, I><<<grid, 256, smem, st>>>(x, ldx, y, ldy, pos, M, dim, rot, tok, ph, pt, F)
  if (vec && interleaved) NB_ROPE(true, true);
  else if (vec) NB_ROPE(true, false);
  else if (interleaved) NB_ROPE(false, true);
  else NB_ROPE(false, false);
#undef NB_ROPE
  return cudaGetLastError();
}

}  // namespace nb
