// Standalone writes to and reads from the KV rings of nd_attend_step's layout
// (k [sessions][slots][kv_heads][qk], v [..][vh], scales [..][kv_heads]):
// nd_kv_append quantises as it writes, nd_kv_read gives back the values. The
// quantiser is the engine's own rule (kv_quant_codes, common.cuh), so a ring
// filled here equals the engine's bit for bit.
#include <algorithm>

#include "fastdiv.hpp"
#include "kernels.hpp"

namespace nb {
namespace {

struct KvRing {
  void *k, *v;
  float *ks, *vs;
  int sessions, slots, kvh, qk, vh;
};

// Ring place (session * slots + slot) of a row, -1 for a row to skip: a
// negative position or a session out of range.
__device__ __forceinline__ long ring_place(const int* sess, const int* pos, int i, const KvRing& R) {
  const int p = pos[i], s = sess ? sess[i] : i;
  if (p < 0 || (unsigned)s >= (unsigned)R.sessions) return -1;
  return (long)s * R.slots + p % R.slots;
}

// A prompt longer than its ring: whether a later row of the same call takes
// row i's place (consecutive rows of a session, see needle.h).
__device__ __forceinline__ bool superseded(const int* sess, const int* pos, int i, int M, const KvRing& R) {
  if (i >= M - R.slots || !sess) return false;
  const int j = i + R.slots;
  return sess[j] == sess[i] && pos[j] == pos[i] + R.slots;
}

__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
  return (uint32_t)(uint8_t)(int8_t)a | (uint32_t)(uint8_t)(int8_t)b << 8 | (uint32_t)(uint8_t)(int8_t)c << 16 |
         (uint32_t)(uint8_t)(int8_t)d << 24;
}

// L lanes (16 or 32) hold one head vector, four values each per step: VEC, the
// values 4 * lane + 4 * L * s; else lane + L * i. Each group of lanes handles
// one vector (row, head, key or value); a row's vectors are neighbours, so a
// warp's loads cover whole cache lines of a projection row. Bytes bound it: 4
// read and 1 written per value.
template <bool VEC, int L, int S>
__global__ void __launch_bounds__(256) kv_append_i8_kernel(const float* __restrict__ k, long ldk,
                                                        const float* __restrict__ v, long ldv,
                                                        const int* __restrict__ sess, const int* __restrict__ pos,
                                                        int M, KvRing R, FastDiv per_row) {
  const long vec = ((long)blockIdx.x * 256 + threadIdx.x) / L;
  const int lane = threadIdx.x % L;
  const bool in = vec < (long)M * (int)per_row.d;
  const int i = in ? (int)(M > (1 << 20) ? vec / per_row.d : per_row.div((int)vec)) : 0;
  const int hv = in ? (int)(vec - (long)i * per_row.d) : 0;
  const bool val = hv >= R.kvh;
  const int h = val ? hv - R.kvh : hv, dim = val ? R.vh : R.qk;
  const float* src = (val ? v + (size_t)i * ldv : k + (size_t)i * ldk) + (size_t)h * dim;
  float x[S][4];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (VEC) {
      const int e = 4 * (lane + L * s);
      const float4 f = in && e < dim ? __ldg(reinterpret_cast<const float4*>(src + e)) : make_float4(0, 0, 0, 0);
      x[s][0] = f.x, x[s][1] = f.y, x[s][2] = f.z, x[s][3] = f.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = lane + L * (4 * s + j);
        x[s][j] = in && e < dim ? __ldg(src + e) : 0.f;
      }
    }
  }
  long at = in ? ring_place(sess, pos, i, R) : -1;
  if (at >= 0 && superseded(sess, pos, i, M, R)) at = -1;
  float scale = 1.f, am = 0.f;  // NaN counts as 0, as in kv_quant_absmax_warp
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) am = fmaxf(am, fabsf(x[s][j]));
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
#pragma unroll
  for (int s = 0; s < S; ++s) {
    scale = kv_quant_codes(am, x[s][0], x[s][1], &x[s][0], &x[s][1]);
    kv_quant_codes(am, x[s][2], x[s][3], &x[s][2], &x[s][3]);
  }
  if (at < 0) return;
  int8_t* dst = (int8_t*)(val ? R.v : R.k) + ((size_t)at * R.kvh + h) * dim;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (VEC) {
      const int e = 4 * (lane + L * s);
      if (e < dim) *reinterpret_cast<uint32_t*>(dst + e) = pack_codes(x[s][0], x[s][1], x[s][2], x[s][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = lane + L * (4 * s + j);
        if (e < dim) dst[e] = (int8_t)x[s][j];
      }
    }
  }
  if (lane == 0) (val ? R.vs : R.ks)[(size_t)at * R.kvh + h] = scale;
}

// The reverse, and the f32 append, move whole rows: a position's keys of all
// heads lie together in the ring and in the row, so a row is kvh * qk values,
// then kvh * vh. A block looks up the places of `rows` rows first (shared
// memory), then its threads move pieces of E values (4 where alignment allows,
// else 1), eight a thread in flight before the first is stored. Bytes bound it:
// per value 4 out and 1 in (int8) or 4.
constexpr int KV_THREADS = 256, KV_FLIGHT = 8, KV_ROWS = 64;

template <bool INT8, bool VEC, bool WRITE>
__global__ void __launch_bounds__(KV_THREADS) kv_rows_kernel(KvRing R, const int* __restrict__ sess,
                                                             const int* __restrict__ pos, int M, float* k, long ldk,
                                                             float* v, long ldv, int rows, FastDiv per_row,
                                                             FastDiv per_k, FastDiv per_v, int nk) {
  __shared__ long place[KV_ROWS];
  const int r0 = blockIdx.x * rows, n = min(rows, M - r0);
  for (int i = threadIdx.x; i < n; i += KV_THREADS) {
    long at = ring_place(sess, pos, r0 + i, R);
    if (WRITE && at >= 0) at = superseded(sess, pos, r0 + i, M, R) ? -1 : at;
    place[i] = at;
  }
  __syncthreads();
  constexpr int E = VEC ? 4 : 1;
  const int total = n * (int)per_row.d;
  for (int base = threadIdx.x; base < total; base += KV_THREADS * KV_FLIGHT) {
    float4 x[KV_FLIGHT];
    uint32_t c[KV_FLIGHT];
    float sc[KV_FLIGHT];
    float* row[KV_FLIGHT];
    size_t ring[KV_FLIGHT];
    bool val[KV_FLIGHT];
#pragma unroll
    for (int u = 0; u < KV_FLIGHT; ++u) {
      const int it = base + u * KV_THREADS;
      row[u] = nullptr;
      if (it >= total) continue;
      const int i = per_row.div(it);
      int e = it - i * (int)per_row.d;
      const long at = place[i];
      if (at < 0) continue;
      val[u] = e >= nk;
      if (val[u]) e -= nk;
      const int h = val[u] ? per_v.div(e) : per_k.div(e);
      row[u] = (val[u] ? v + (size_t)(r0 + i) * ldv : k + (size_t)(r0 + i) * ldk) + e * E;
      ring[u] = (size_t)at * R.kvh * (val[u] ? R.vh : R.qk) + e * E;
      if (WRITE) {
        if (VEC) x[u] = *reinterpret_cast<const float4*>(row[u]);
        else x[u].x = *row[u];
      } else if (INT8) {
        const int8_t* src = (const int8_t*)(val[u] ? R.v : R.k) + ring[u];
        sc[u] = __ldg((val[u] ? R.vs : R.ks) + (size_t)at * R.kvh + h);
        c[u] = VEC ? __ldg(reinterpret_cast<const uint32_t*>(src)) : (uint32_t)(uint8_t)__ldg(src);
      } else {
        const float* src = (const float*)(val[u] ? R.v : R.k) + ring[u];
        if (VEC) x[u] = __ldg(reinterpret_cast<const float4*>(src));
        else x[u].x = __ldg(src);
      }
    }
#pragma unroll
    for (int u = 0; u < KV_FLIGHT; ++u) {
      if (!row[u]) continue;
      if (!WRITE && INT8)
        x[u] = make_float4((float)(int8_t)c[u] * sc[u], (float)(int8_t)(c[u] >> 8) * sc[u],
                           (float)(int8_t)(c[u] >> 16) * sc[u], (float)(int8_t)(c[u] >> 24) * sc[u]);
      float* dst = WRITE ? (float*)(val[u] ? R.v : R.k) + ring[u] : row[u];
      if (VEC) *reinterpret_cast<float4*>(dst) = x[u];
      else *dst = x[u].x;
    }
  }
}

bool vec_ok(const void* p, int align) { return ((uintptr_t)p) % align == 0; }

}  // namespace

// Rows a block of kv_rows_kernel moves: eight pieces a thread, fewer where that
// would leave SMs without a block.
static int kv_block_rows(int M, int pieces) {
  int rows = std::max(1, std::min(KV_ROWS, KV_THREADS * KV_FLIGHT / std::max(1, pieces)));
  while (rows > 1 && (M + rows - 1) / rows < 148) rows /= 2;
  return rows;
}

template <bool INT8, bool VEC, bool WRITE>
static cudaError_t launch_kv_rows(const KvRing& R, const int* sess, const int* pos, int M, float* k, int ldk, float* v,
                                  int ldv, cudaStream_t st) {
  constexpr int E = VEC ? 4 : 1;
  const int nk = k ? R.kvh * R.qk / E : 0, nv = v ? R.kvh * R.vh / E : 0;
  const int rows = kv_block_rows(M, nk + nv);
  kv_rows_kernel<INT8, VEC, WRITE><<<(M + rows - 1) / rows, KV_THREADS, 0, st>>>(
      R, sess, pos, M, k, ldk, v, ldv, rows, FastDiv(nk + nv), FastDiv(std::max(1, R.qk / E)),
      FastDiv(std::max(1, R.vh / E)), nk);
  return cudaGetLastError();
}

cudaError_t launch_kv_append(const float* k, int ldk, const float* v, int ldv, const int* sess, const int* pos, int M,
                             int int8, int sessions, int slots, int kvh, int qk, int vh, void* kc, void* vc, float* ks,
                             float* vs, cudaStream_t st) {
  if (M <= 0) return cudaSuccess;
  const KvRing R{kc, vc, ks, vs, sessions, slots, kvh, qk, vh};
  const int al = int8 ? 4 : 16;
  const bool vec = qk % 4 == 0 && vh % 4 == 0 && ldk % 4 == 0 && ldv % 4 == 0 && vec_ok(k, 16) && vec_ok(v, 16) &&
                   vec_ok(kc, al) && vec_ok(vc, al);
  if (!int8) {  // the rows are only read
    float *kr = const_cast<float*>(k), *vr = const_cast<float*>(v);
    return vec ? launch_kv_rows<false, true, true>(R, sess, pos, M, kr, ldk, vr, ldv, st)
               : launch_kv_rows<false, false, true>(R, sess, pos, M, kr, ldk, vr, ldv, st);
  }
  const FastDiv per(2 * kvh);
  const long vecs = (long)M * 2 * kvh;
  const int big = std::max(qk, vh), L = big <= 64 ? 16 : 32;
  const long blocks = (vecs * L + 255) / 256;
  if (blocks > 0x7fffffffl) return cudaErrorInvalidValue;
#define NB_GO(V, L, S) \
  kv_append_i8_kernel<V, L, S><<<(unsigned)blocks, 256, 0, st>>>(k, ldk, v, ldv, sess, pos, M, R, per)
  if (big <= 64) {
    if (vec) NB_GO(true, 16, 1);
    else NB_GO(false, 16, 1);
  } else if (big <= 128) {
    if (vec) NB_GO(true, 32, 1);
    else NB_GO(false, 32, 1);
  } else {
    if (vec) NB_GO(true, 32, 2);
    else NB_GO(false, 32, 2);
  }
#undef NB_GO
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const void* kc, const void* vc, const float* ks, const float* vs, int int8, int sessions,
                           int slots, int kvh, int qk, int vh, const int* sess, const int* pos, int M, float* k,
                           int ldk, float* v, int ldv, cudaStream_t st) {
  if (M <= 0 || (!k && !v)) return cudaSuccess;
  const KvRing R{const_cast<void*>(kc), const_cast<void*>(vc), const_cast<float*>(ks), const_cast<float*>(vs),
                 sessions, slots, kvh, qk, vh};
  const int al = int8 ? 4 : 16;
  const bool vec = (!k || (qk % 4 == 0 && ldk % 4 == 0 && vec_ok(k, 16) && vec_ok(kc, al))) &&
                   (!v || (vh % 4 == 0 && ldv % 4 == 0 && vec_ok(v, 16) && vec_ok(vc, al)));
  if (int8)
    return vec ? launch_kv_rows<true, true, false>(R, sess, pos, M, k, ldk, v, ldv, st)
               : launch_kv_rows<true, false, false>(R, sess, pos, M, k, ldk, v, ldv, st);
  return vec ? launch_kv_rows<false, true, false>(R, sess, pos, M, k, ldk, v, ldv, st)
             : launch_kv_rows<false, false, false>(R, sess, pos, M, k, ldk, v, ldv, st);
}

}  // namespace nb
