// Standalone writes to and reads from KV rings of nd_attend_step's layout (k
// [sessions][slots][kv_heads][qk], v [..][vh], scales [..][kv_heads]):
// nd_kv_append quantises as it writes, nd_kv_read gives back the values. The
// quantiser is the engine's rule (kv_quant_codes, common.cuh), so codes and scales
// equal the engine's bit for bit; the rings do not, as a session's own are
// head-major and hold value codes offset by 128.
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
// row i's place. The session's rows stand one after another with positions that
// ascend by one (see needle.h), so that row holds position pos[i] + slots, and is
// row i + slots but for rows skipped in between: the walk goes ahead by what a
// position lacks (fewer rows cannot do) and over skipped rows eight at a time, to
// the session's end. Anything but the later position itself leaves row i alone.
__device__ __forceinline__ bool superseded(const int* sess, const int* pos, int i, int M, const KvRing& R) {
  if (i >= M - R.slots || !sess) return false;
  const int s = sess[i];
  const long want = (long)pos[i] + R.slots;
  for (long j = (long)i + R.slots; j < M && sess[j] == s;) {
    const int q = pos[j];
    if (q >= 0) {
      if (q >= want) return q == want;
      j += want - q;
      continue;
    }
    long hop = 8;  // to the next row of the eight that is not skipped
#pragma unroll
    for (int u = 7; u >= 1; --u)
      if (j + u < M && (sess[j + u] != s || pos[j + u] >= 0)) hop = u;
    j += hop;
  }
  return false;
}

__device__ __forceinline__ uint32_t pack_codes(int a, int b, int c, int d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

constexpr int KV_THREADS = 256, KV_ROWS = 64;

// The code of one value, kv_quant_codes' clamp(roundf(x * inv), -128, 127) in
// fewer instructions: half away from zero is truncation after adding half the
// sign with rounding toward zero (exact above a half, and just below it the
// truncated sum stays under one), the conversion to 8 bits clamps, and the max
// with -129 takes a NaN to -128 as the clamp does. The same bits on every input.
__device__ __forceinline__ int code_of(float x, float inv) {
  const float y = fmaxf(__fmul_rn(x, inv), -129.f);
  int c;
  asm("cvt.rzi.s8.f32 %0, %1;" : "=r"(c) : "f"(__fadd_rz(y, copysignf(0.5f, y))));
  return c;
}

// int8: L lanes (16 or 32) hold one head vector, four values each per step:
// VEC, the values 4 * lane + 4 * L * s; else lane + L * i. A block looks up the
// places of `rows` rows once (shared memory); its groups of lanes then take the
// rows' vectors (row, key or value, head), KV_VECS of them loaded before the
// first is quantised. A row's vectors are neighbours, so a warp reads whole
// cache lines of a projection row. 4 bytes read and 1 written per value: 16384 rows
// of 224 values are 2.8 us of bytes and take 10.4. A block makes one pass, and its
// warps wait at its one barrier for the places (4.2 barrier stalls per issue
// against 0.4 on memory, 63 % of the issue slots busy).
constexpr int KV_VECS = 4;

template <bool VEC, int L, int S>
__global__ void __launch_bounds__(KV_THREADS) kv_append_i8_kernel(const float* __restrict__ k, long ldk,
                                                                  const float* __restrict__ v, long ldv,
                                                                  const int* __restrict__ sess,
                                                                  const int* __restrict__ pos, int M, KvRing R,
                                                                  int rows, FastDiv per_row) {
  __shared__ long place[KV_ROWS];
  constexpr int U = S > 1 ? 2 : KV_VECS, GROUPS = KV_THREADS / L;
  const int r0 = blockIdx.x * rows, n = min(rows, M - r0);
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const int total = n * (int)per_row.d;
  float x[U][S][4];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int vec = base + u * GROUPS;
      const bool in = vec < total;
      const int i = in ? per_row.div(vec) : 0, hv = in ? vec - i * (int)per_row.d : 0;
      const bool val = hv >= R.kvh;
      const int h = val ? hv - R.kvh : hv, dim = val ? R.vh : R.qk;
      const float* src = (val ? v + (size_t)(r0 + i) * ldv : k + (size_t)(r0 + i) * ldk) + h * dim;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (VEC) {
          const int e = 4 * (lane + L * s);
          const float4 f = in && e < dim ? __ldg(reinterpret_cast<const float4*>(src + e)) : make_float4(0, 0, 0, 0);
          x[u][s][0] = f.x, x[u][s][1] = f.y, x[u][s][2] = f.z, x[u][s][3] = f.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int e = lane + L * (4 * s + j);
            x[u][s][j] = in && e < dim ? __ldg(src + e) : 0.f;
          }
        }
      }
    }
  };
  load(group);  // on its way while the places are looked up
  for (int i = threadIdx.x; i < n; i += KV_THREADS) {
    const long at = ring_place(sess, pos, r0 + i, R);
    place[i] = at >= 0 && superseded(sess, pos, r0 + i, M, R) ? -1 : at;
  }
  __syncthreads();
  for (int base = group; base < total + group; base += U * GROUPS) {  // the same count for the whole block
    if (base != group) load(base);
    float am[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      am[u] = 0.f;  // NaN counts as 0, as in kv_quant_absmax_warp
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) am[u] = fmaxf(am[u], fabsf(x[u][s][j]));
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) am[u] = fmaxf(am[u], __shfl_xor_sync(0xffffffffu, am[u], o));
    // The scale and its reciprocal of vector u by lane u of the group (IEEE
    // quotients are long), then handed round.
    float sc_own = 1.f, inv_own = 1.f;
    {
      float a = am[0];
#pragma unroll
      for (int u = 1; u < U; ++u) a = (lane & (U - 1)) == u ? am[u] : a;
      sc_own = a > 0.0f ? __fdiv_rn(a, 127.0f) : 1.0f;
      inv_own = __fdiv_rn(1.0f, sc_own);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float scale = __shfl_sync(0xffffffffu, sc_own, u, L), inv = __shfl_sync(0xffffffffu, inv_own, u, L);
      const int vec = base + u * GROUPS;
      if (vec >= total) continue;
      const int i = per_row.div(vec), hv = vec - i * (int)per_row.d;
      const long at = place[i];
      if (at < 0) continue;
      const bool val = hv >= R.kvh;
      const int h = val ? hv - R.kvh : hv, dim = val ? R.vh : R.qk;
      int8_t* dst = (int8_t*)(val ? R.v : R.k) + ((size_t)at * R.kvh + h) * dim;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        int c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = code_of(x[u][s][j], inv);
        if (VEC) {
          const int e = 4 * (lane + L * s);
          if (e < dim) *reinterpret_cast<uint32_t*>(dst + e) = pack_codes(c[0], c[1], c[2], c[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int e = lane + L * (4 * s + j);
            if (e < dim) dst[e] = (int8_t)c[j];
          }
        }
      }
      if (lane == 0) (val ? R.vs : R.ks)[(size_t)at * R.kvh + h] = scale;
    }
  }
}

// The reverse, and the f32 append, move whole rows: a position's keys of all
// heads lie together in the ring and in the row, so a row is kvh * qk values,
// then kvh * vh. A block looks up the places of `rows` rows first (shared
// memory), then its threads move pieces of E values, KV_FLIGHT of them loaded
// before the first is stored. E is 8 where the rows allow 32-byte accesses (a
// whole sector a thread, few instructions a value), 4 or 1 where they do not.
// Bytes bound it: per value 4 out and 1 in (int8) or 4.
constexpr int KV_FLIGHT = 4;

struct alignas(32) Float8 {
  float f[8];
};
__device__ __forceinline__ void store8(float* p, const Float8& x) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x.f[0]), "f"(x.f[1]), "f"(x.f[2]),
               "f"(x.f[3]), "f"(x.f[4]), "f"(x.f[5]), "f"(x.f[6]), "f"(x.f[7])
               : "memory");
}
__device__ __forceinline__ void load8(const float* p, Float8& x) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(x.f[0]), "=f"(x.f[1]), "=f"(x.f[2]), "=f"(x.f[3]), "=f"(x.f[4]), "=f"(x.f[5]), "=f"(x.f[6]),
                 "=f"(x.f[7])
               : "l"(p)
               : "memory");
}
// Byte j of a word of codes as a float: with its sign bit flipped it is the low
// mantissa byte of 2^23 + code + 128.
__device__ __forceinline__ float code_float(uint32_t flipped, int j) {
  return __uint_as_float(__byte_perm(flipped, 0x4b000000u, 0x7440 + j)) - 8388736.f;
}

template <bool INT8, int E, bool WRITE>
__global__ void __launch_bounds__(KV_THREADS) kv_rows_kernel(KvRing R, const int* __restrict__ sess,
                                                             const int* __restrict__ pos, int M, float* k, long ldk,
                                                             float* v, long ldv, int rows, FastDiv per_row,
                                                             FastDiv per_k, FastDiv per_v, int nk) {
  __shared__ long place[KV_ROWS];  // first vector of the row in the ring, -1: skip
  const int r0 = blockIdx.x * rows, n = min(rows, M - r0);
  for (int i = threadIdx.x; i < n; i += KV_THREADS) {
    long at = ring_place(sess, pos, r0 + i, R);
    if (WRITE && at >= 0) at = superseded(sess, pos, r0 + i, M, R) ? -1 : at;
    place[i] = at < 0 ? -1 : at * R.kvh;
  }
  __syncthreads();
  constexpr int CW = E == 8 ? 2 : 1;  // words of codes of a piece
  const int total = n * (int)per_row.d;
  for (int base = threadIdx.x; base < total; base += KV_THREADS * KV_FLIGHT) {
    float* dst[KV_FLIGHT];
    Float8 x[INT8 ? 1 : KV_FLIGHT];
    uint32_t c[INT8 ? KV_FLIGHT : 1][CW];
    float sc[INT8 ? KV_FLIGHT : 1];
#pragma unroll
    for (int u = 0; u < KV_FLIGHT; ++u) {
      const int it = base + u * KV_THREADS;
      dst[u] = nullptr;
      if (it >= total) continue;
      const int i = per_row.div(it);
      int e = it - i * (int)per_row.d;
      const long at = place[i];
      if (at < 0) continue;
      const bool val = e >= nk;
      if (val) e -= nk;
      float* row = (val ? v + (size_t)(r0 + i) * ldv : k + (size_t)(r0 + i) * ldk) + e * E;
      const size_t ring = (size_t)at * (val ? R.vh : R.qk) + e * E;
      const void* cache = val ? R.v : R.k;
      if (INT8) {
        const int iu = INT8 ? u : 0, h = val ? per_v.div(e) : per_k.div(e);
        const int8_t* src = (const int8_t*)cache + ring;
        dst[u] = row;
        sc[iu] = __ldg((val ? R.vs : R.ks) + at + h);
        if (E == 8) {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(src));
          c[iu][0] = w.x, c[iu][CW - 1] = w.y;
        } else {
          c[iu][0] = E == 4 ? __ldg(reinterpret_cast<const uint32_t*>(src)) : (uint32_t)(uint8_t)__ldg(src);
        }
      } else {
        const int xu = INT8 ? 0 : u;
        float* slot = const_cast<float*>((const float*)cache) + ring;
        dst[u] = WRITE ? slot : row;
        const float* src = WRITE ? row : slot;
        if (E == 8) {
          load8(src, x[xu]);
        } else if (E == 4) {
          const float4 f = *reinterpret_cast<const float4*>(src);
          x[xu].f[0] = f.x, x[xu].f[1] = f.y, x[xu].f[2] = f.z, x[xu].f[3] = f.w;
        } else {
          x[xu].f[0] = *src;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < KV_FLIGHT; ++u) {
      if (!dst[u]) continue;
      Float8 f = x[INT8 ? 0 : u];
      if (INT8) {
        const int iu = INT8 ? u : 0;
#pragma unroll
        for (int j = 0; j < E; ++j) f.f[j] = code_float(c[iu][j / 4 < CW ? j / 4 : 0] ^ 0x80808080u, j & 3) * sc[iu];
      }
      if (E == 8) store8(dst[u], f);
      else if (E == 4) *reinterpret_cast<float4*>(dst[u]) = make_float4(f.f[0], f.f[1], f.f[2], f.f[3]);
      else *dst[u] = f.f[0];
    }
  }
}

bool vec_ok(const void* p, int align) { return ((uintptr_t)p) % align == 0; }

}  // namespace

// Rows a block of kv_rows_kernel moves: KV_FLIGHT pieces a thread, fewer where that
// would leave SMs without a block. 133504 int8 rows read back (224 values): 4 rows
// a block 72 us, 8: 51, 16: 37, 32: 30.9, 36 (the rule): 30.8 (5.0 TB/s of 6.6 for a
// copy), 64: 30.9. f32 rows, 16384 written and read: 4: 31, 8: 21, 16: 18.4, 32: 16.1,
// 36 (the rule): 16.5, of which the write takes 8.3 (4.5 us of bytes), 64: 16.6.
static int kv_block_rows(int M, int pieces) {
  int rows = std::max(1, std::min(KV_ROWS, KV_THREADS * KV_FLIGHT / std::max(1, pieces)));
  while (rows > 1 && (M - 1) / rows + 1 < 148) rows /= 2;
  return rows;
}

template <bool INT8, int E, bool WRITE>
static cudaError_t launch_kv_rows(const KvRing& R, const int* sess, const int* pos, int M, float* k, int ldk, float* v,
                                  int ldv, cudaStream_t st) {
  const int nk = k ? R.kvh * R.qk / E : 0, nv = v ? R.kvh * R.vh / E : 0;
  const int rows = kv_block_rows(M, nk + nv);
  kv_rows_kernel<INT8, E, WRITE><<<(M - 1) / rows + 1, KV_THREADS, 0, st>>>(
      R, sess, pos, M, k, ldk, v, ldv, rows, FastDiv(nk + nv), FastDiv(std::max(1, R.qk / E)),
      FastDiv(std::max(1, R.vh / E)), nk);
  return cudaGetLastError();
}

// Widest piece that rows (f32, leading dimension ld) and ring of keys or values
// (es bytes a value) allow.
static int kv_piece(const float* row, int ld, const void* ring, int dim, int es) {
  for (int e = 8; e > 1; e /= 2)
    if (dim % e == 0 && ld % e == 0 && vec_ok(row, 4 * e) && vec_ok(ring, es * e)) return e;
  return 1;
}

template <bool INT8, bool WRITE>
static cudaError_t launch_kv_piece(const KvRing& R, const int* sess, const int* pos, int M, float* k, int ldk, float* v,
                                   int ldv, cudaStream_t st) {
  int e = 8;
  if (k) e = std::min(e, kv_piece(k, ldk, R.k, R.qk, INT8 ? 1 : 4));
  if (v) e = std::min(e, kv_piece(v, ldv, R.v, R.vh, INT8 ? 1 : 4));
  if (e == 8) return launch_kv_rows<INT8, 8, WRITE>(R, sess, pos, M, k, ldk, v, ldv, st);
  if (e == 4) return launch_kv_rows<INT8, 4, WRITE>(R, sess, pos, M, k, ldk, v, ldv, st);
  return launch_kv_rows<INT8, 1, WRITE>(R, sess, pos, M, k, ldk, v, ldv, st);
}

cudaError_t launch_kv_append(const float* k, int ldk, const float* v, int ldv, const int* sess, const int* pos, int M,
                             int int8, int sessions, int slots, int kvh, int qk, int vh, void* kc, void* vc, float* ks,
                             float* vs, cudaStream_t st) {
  if (M <= 0) return cudaSuccess;
  const KvRing R{kc, vc, ks, vs, sessions, slots, kvh, qk, vh};
  if (!int8) {  // the rows are only read
    float *kr = const_cast<float*>(k), *vr = const_cast<float*>(v);
    return launch_kv_piece<false, true>(R, sess, pos, M, kr, ldk, vr, ldv, st);
  }
  const bool vec = qk % 4 == 0 && vh % 4 == 0 && ldk % 4 == 0 && ldv % 4 == 0 && vec_ok(k, 16) && vec_ok(v, 16) &&
                   vec_ok(kc, 4) && vec_ok(vc, 4);
  // Rows a block: KV_VECS vectors a group, fewer where SMs would be without a
  // block. 16384 rows of 2 heads of 48 | 64: 2 rows 30.9 us, 4: 18.6, 8: 12.4, 16 (the
  // rule): 10.4, 32: 10.6, 64: 12.4.
  const int big = std::max(qk, vh), L = big <= 64 ? 16 : 32;
  int rows = std::max(1, std::min(KV_ROWS, (big > 128 ? 2 : KV_VECS) * (KV_THREADS / L) / (2 * kvh)));
  while (rows > 1 && (M - 1) / rows + 1 < 148) rows /= 2;
  const int blocks = (M - 1) / rows + 1;
#define NB_GO(V, L, S) \
  kv_append_i8_kernel<V, L, S>                \
      <<<blocks, KV_THREADS, 0, st>>>(k, ldk, v, ldv, sess, pos, M, R, rows, FastDiv(2 * kvh))
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
  return int8 ? launch_kv_piece<true, false>(R, sess, pos, M, k, ldk, v, ldv, st)
              : launch_kv_piece<false, false>(R, sess, pos, M, k, ldk, v, ldv, st);
}

}  // namespace nb
