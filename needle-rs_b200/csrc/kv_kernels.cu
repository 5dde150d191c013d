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

__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
  return (uint32_t)(uint8_t)(int8_t)a | (uint32_t)(uint8_t)(int8_t)b << 8 | (uint32_t)(uint8_t)(int8_t)c << 16 |
         (uint32_t)(uint8_t)(int8_t)d << 24;
}

// L lanes (16 or 32) hold one head vector, four values each per step: VEC, the
// values 4 * lane + 4 * L * s; else lane + L * i. Each group of lanes handles
// one vector (row, head, key or value); a row's vectors are neighbours, so a
// warp's loads cover whole cache lines of a projection row. Bytes bound it: 4
// read per value and 1 (int8) or 4 written.
template <bool INT8, bool VEC, int L, int S>
__global__ void __launch_bounds__(256) kv_append_kernel(const float* __restrict__ k, long ldk,
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
  // A prompt longer than its ring: the row whose place a later row of the same
  // call takes is not written (consecutive rows of a session, see needle.h).
  if (at >= 0 && i < M - R.slots) {
    const int j = i + R.slots;
    if ((sess ? sess[j] == sess[i] : false) && pos[j] == pos[i] + R.slots) at = -1;
  }
  float scale = 1.f;
  if (INT8) {
    float am = 0.f;  // NaN counts as 0, as in kv_quant_absmax_warp
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
  }
  if (at < 0) return;
  const size_t o = ((size_t)at * R.kvh + h) * dim;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (VEC) {
      const int e = 4 * (lane + L * s);
      if (e >= dim) continue;
      if (INT8)
        *reinterpret_cast<uint32_t*>((int8_t*)(val ? R.v : R.k) + o + e) =
            pack_codes(x[s][0], x[s][1], x[s][2], x[s][3]);
      else
        *reinterpret_cast<float4*>((float*)(val ? R.v : R.k) + o + e) =
            make_float4(x[s][0], x[s][1], x[s][2], x[s][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = lane + L * (4 * s + j);
        if (e >= dim) continue;
        if (INT8)
          ((int8_t*)(val ? R.v : R.k))[o + e] = (int8_t)x[s][j];
        else
          ((float*)(val ? R.v : R.k))[o + e] = x[s][j];
      }
    }
  }
  if (INT8 && lane == 0) (val ? R.vs : R.ks)[(size_t)at * R.kvh + h] = scale;
}

// The reverse: L lanes per vector. The places are looked up first, then the
// codes, then the rows go out; bytes bound it as above.
template <bool INT8, bool VEC, int L, int S>
__global__ void __launch_bounds__(256) kv_read_kernel(KvRing R, const int* __restrict__ sess,
                                                      const int* __restrict__ pos, int M, float* __restrict__ k,
                                                      long ldk, float* __restrict__ v, long ldv, FastDiv per_row) {
  const long vec = ((long)blockIdx.x * 256 + threadIdx.x) / L;
  const int lane = threadIdx.x % L;
  if (vec >= (long)M * (int)per_row.d) return;
  const int i = (int)(M > (1 << 20) ? vec / per_row.d : per_row.div((int)vec));
  const int hv = (int)(vec - (long)i * per_row.d);
  const bool val = !k || (v && hv >= R.kvh);
  const int h = k && val ? hv - R.kvh : hv, dim = val ? R.vh : R.qk;
  const long at = ring_place(sess, pos, i, R);
  if (at < 0) return;
  const size_t o = ((size_t)at * R.kvh + h) * dim;
  float* dst = (val ? v + (size_t)i * ldv : k + (size_t)i * ldk) + (size_t)h * dim;
  const float scale = INT8 ? __ldg((val ? R.vs : R.ks) + (size_t)at * R.kvh + h) : 1.f;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (VEC) {
      const int e = 4 * (lane + L * s);
      if (e >= dim) continue;
      if (INT8) {
        const char4 c = __ldg(reinterpret_cast<const char4*>((const int8_t*)(val ? R.v : R.k) + o + e));
        *reinterpret_cast<float4*>(dst + e) =
            make_float4((float)c.x * scale, (float)c.y * scale, (float)c.z * scale, (float)c.w * scale);
      } else {
        *reinterpret_cast<float4*>(dst + e) =
            __ldg(reinterpret_cast<const float4*>((const float*)(val ? R.v : R.k) + o + e));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = lane + L * (4 * s + j);
        if (e >= dim) continue;
        dst[e] = INT8 ? (float)__ldg((const signed char*)(val ? R.v : R.k) + o + e) * scale
                      : __ldg((const float*)(val ? R.v : R.k) + o + e);
      }
    }
  }
}

bool vec_ok(const void* p, int align) { return ((uintptr_t)p) % align == 0; }

}  // namespace

#define NB_KV_FORMS(GO)                               \
  do {                                                \
    const int big = std::max(k ? qk : 0, v ? vh : 0); \
    if (big <= 64) {                                  \
      if (vec) GO(true, 16, 1);                       \
      else GO(false, 16, 1);                          \
    } else if (big <= 128) {                          \
      if (vec) GO(true, 32, 1);                       \
      else GO(false, 32, 1);                          \
    } else {                                          \
      if (vec) GO(true, 32, 2);                       \
      else GO(false, 32, 2);                          \
    }                                                 \
  } while (0)

cudaError_t launch_kv_append(const float* k, int ldk, const float* v, int ldv, const int* sess, const int* pos, int M,
                             int int8, int sessions, int slots, int kvh, int qk, int vh, void* kc, void* vc, float* ks,
                             float* vs, cudaStream_t st) {
  if (M <= 0) return cudaSuccess;
  const KvRing R{kc, vc, ks, vs, sessions, slots, kvh, qk, vh};
  const int al = int8 ? 4 : 16;
  const bool vec = qk % 4 == 0 && vh % 4 == 0 && ldk % 4 == 0 && ldv % 4 == 0 && vec_ok(k, 16) && vec_ok(v, 16) &&
                   vec_ok(kc, al) && vec_ok(vc, al);
  const FastDiv per(2 * kvh);
  const long vecs = (long)M * 2 * kvh;
#define NB_GO(V, L, S)                                                                                           \
  do {                                                                                                           \
    const long blocks = (vecs * L + 255) / 256;                                                                  \
    if (blocks > 0x7fffffffl) return cudaErrorInvalidValue;                                                      \
    if (int8) kv_append_kernel<true, V, L, S><<<(unsigned)blocks, 256, 0, st>>>(k, ldk, v, ldv, sess, pos, M, R, per); \
    else kv_append_kernel<false, V, L, S><<<(unsigned)blocks, 256, 0, st>>>(k, ldk, v, ldv, sess, pos, M, R, per);     \
  } while (0)
  NB_KV_FORMS(NB_GO);
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
  const int n = (k ? kvh : 0) + (v ? kvh : 0);
  const FastDiv per(n);
  const long vecs = (long)M * n;
#define NB_GO(V, L, S)                                                                                          \
  do {                                                                                                          \
    const long blocks = (vecs * L + 255) / 256;                                                                 \
    if (blocks > 0x7fffffffl) return cudaErrorInvalidValue;                                                     \
    if (int8) kv_read_kernel<true, V, L, S><<<(unsigned)blocks, 256, 0, st>>>(R, sess, pos, M, k, ldk, v, ldv, per); \
    else kv_read_kernel<false, V, L, S><<<(unsigned)blocks, 256, 0, st>>>(R, sess, pos, M, k, ldk, v, ldv, per);     \
  } while (0)
  NB_KV_FORMS(NB_GO);
#undef NB_GO
  return cudaGetLastError();
}

}  // namespace nb
