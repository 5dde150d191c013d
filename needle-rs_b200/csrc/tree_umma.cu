// nd_attend_tree on the 5th-generation tensor cores, for trees whose T * rep
// rows of a KV head fill most of a 128-row MMA tile (tree_kernels.cu says when).
//
//   S = Q K^T,  P = 2^(S * scales - max),  O += P V
//
// per block of BN positions: S and O lie in tensor memory (TMEM), a softmax
// warpgroup holds one row a thread, P returns to TMEM in S's place as the A
// operand of the second product. f32 accuracy from f16 operands: the query and
// P are f16 high parts and remainders (22 bits; int8 codes are f16 values
// exactly; f32 keys and values are split the same way after a power-of-two
// scale per position, which is then treated like an int8 scale). The products
// with remainders go first: the tensor cores truncate when they accumulate,
// and truncation costs only what the sum already holds. For the same reason O
// is drained into f32 registers after every block.
//
// Warps: W softmax warpgroups (block i belongs to warpgroup i % W, each its
// own running max, sum and output, merged at the end) and four producer warps
// that read the ring and the draft, widen them to f16 and lay them down in the
// 128-byte swizzled form the MMA reads: keys as they lie, values transposed
// eight positions at a time in registers. With W = 1 two blocks share an SM, so one's
// softmax runs under the other's MMAs; 128-wide heads need the shared memory
// of a whole SM and W = 2. One thread of a softmax warpgroup issues its MMAs.
//
// Every wait is bounded as in umma_gemm.cu.
#include <algorithm>

#include "kernels.hpp"
#include "launch_util.hpp"
#include "tree.cuh"
#include "umma.cuh"

namespace nb {
namespace {

template <bool I8_, int QS_, int VP_, int W_, int BN_, int NST_>
struct TreeUmma {
  static constexpr bool I8 = I8_;
  static constexpr int QS = QS_;    // k16 steps of the key product
  static constexpr int VP = VP_;    // value width held (64 or 128)
  static constexpr int W = W_, BN = BN_, NST = NST_;
  static constexpr int KA = (QS * 16 + 63) / 64;  // 64-wide swizzle atoms of a key row
  static constexpr int PARTS = I8 ? 1 : 2;        // high part, remainder
  static constexpr int Q_TILE = KA * 128 * 128, K_TILE = KA * BN * 128, V_TILE = BN / 64 * VP * 128;
  static constexpr int STAGE = PARTS * (K_TILE + V_TILE);
  static constexpr int THREADS = W * 128 + 128, CTAS = W == 1 ? 2 : 1;
  // Registers a thread: the launch's, a softmax thread's, a producer's; the
  // warpgroups' shares add up to the launch's.
  static constexpr int REG_ALL = W == 1 ? 128 : 168, REG_SOFT = W == 1 ? 168 : 208, REG_PROD = 88;
  static_assert(W * REG_SOFT + REG_PROD == (W + 1) * REG_ALL, "register shares");
  static constexpr int S_COLS = BN, WG_COLS = BN + VP;  // TMEM columns of a warpgroup: S (then P), O
  static constexpr int TMEM = W * WG_COLS <= 128 ? 128 : W * WG_COLS <= 256 ? 256 : 512;
  static constexpr size_t META = NST * (size_t)(BN * 8 + BN / 8 + 16) + 128 * 4 + 512 + 2 * 4 * 64 * 4;
  static constexpr size_t SMEM = 1024 + 2 * (size_t)Q_TILE + NST * (size_t)STAGE + META;
};

__device__ __forceinline__ void tmem_st8(uint32_t t, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// kind::f16: f32 accumulate, f16 operands, both K-major, M = 128.
template <int N>
constexpr uint32_t tree_idesc() {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
template <int N>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(tree_idesc<N>()), "r"(accum));
}
// A operand from TMEM: lane = row, a column holds two K elements.
template <int N>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(tree_idesc<N>()), "r"(accum));
}

typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pk(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void up(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// (a, b) as an f16 pair, a in the low half.
__device__ __forceinline__ uint32_t cvt2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// x * 2^.. as high part and remainder halves of two values.
__device__ __forceinline__ void halves(float a, float b, uint32_t* hi, uint32_t* lo) {
  const uint32_t h = cvt2(a, b);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  *hi = h;
  *lo = cvt2(a - f.x, b - f.y);
}
// Four sign-flipped codes as f16 values, two a register (see codes_h2 of the
// mma.sync form): bytes 0, 1 and bytes 2, 3.
__device__ __forceinline__ void widen(uint32_t u, uint32_t* a, uint32_t* b) {
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  uint32_t p = __byte_perm(u, 0x64646464u, 0x4140), r = __byte_perm(u, 0x64646464u, 0x4342);
  __half2 x = __hsub2(*reinterpret_cast<__half2*>(&p), bias), y = __hsub2(*reinterpret_cast<__half2*>(&r), bias);
  *a = *reinterpret_cast<uint32_t*>(&x);
  *b = *reinterpret_cast<uint32_t*>(&y);
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
    if (start + cnt > A.slots) w |= bit_range(o, o + start + cnt - A.slots);
  }
  return w;
}

// One row over positions [v0, v1) by a warp, in f32 from the cache itself: the
// rows whose values or scales f16 operands cannot hold. Returns log2 max, sum,
// and dims lane + 32 j of the output.
template <bool I8>
__device__ __noinline__ void tree_slow_row(const TreeArgs& A, const TreePlace& P, size_t node_at, int node, int head,
                                           int start, int cnt, int n_ring, int v0, int v1, float* m_out, float* l_out,
                                           float (&o)[4]) {
  const int lane = threadIdx.x & 31;
  const float* q = A.q + node_at * A.ldq + (size_t)head * A.qk;
  float m = -INFINITY, l = 0.f;
  o[0] = o[1] = o[2] = o[3] = 0.f;
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
        for (int i = 0; i < A.qk; ++i) s = fmaf(q[i], (float)k[i] * sc, s);
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
  *m_out = m;
  *l_out = l;
}

// Grid (tiles of 128 rows * kvh * nsplit, sessions).
template <class C>
__global__ void __launch_bounds__(C::THREADS, C::CTAS) tree_umma_kernel(const __grid_constant__ TreeArgs A, int* werr) {
  constexpr bool I8 = C::I8;
  constexpr int BN = C::BN, VP = C::VP, QS = C::QS, W = C::W, NST = C::NST, NC = BN / 32;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  unsigned char *qhi = sm, *qlo = sm + C::Q_TILE, *stages = sm + 2 * C::Q_TILE;
  float* col_k = reinterpret_cast<float*>(stages + (size_t)NST * C::STAGE);  // [NST][BN] key scales
  float* col_v = col_k + NST * BN;                                          // [NST][BN] value scales times 2^(140 - e)
  uint32_t* odd = reinterpret_cast<uint32_t*>(col_v + NST * BN);            // [NST][NC] columns to keep out
  int* expo = reinterpret_cast<int*>(odd + NST * NC);                       // [NST][2] e, least exponent so far
  float* row_q = reinterpret_cast<float*>(expo + 2 * NST);                  // [128] score scale of a row
  float* wmax = row_q + 128;                                                // [2][4][64] producers' maxima
  uint64_t* full = reinterpret_cast<uint64_t*>(wmax + 2 * 4 * 64);
  uint64_t* empty = full + NST;
  uint64_t* s_full = empty + NST;   // [W] S of the warpgroup's block
  uint64_t* o_full = s_full + W;    // [W] O of the warpgroup's block
  uint64_t* drain = o_full + W;     // [W] every MMA of the warpgroup
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + W);
  volatile uint32_t* abort = tmem_slot + 1;
  int* range = reinterpret_cast<int*>(tmem_slot + 2);    // [2]
  uint32_t* slow = reinterpret_cast<uint32_t*>(range + 2);  // [4] rows for tree_slow_row

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.y;
  int bx = blockIdx.x;
  const int z = bx % A.nsplit;
  bx /= A.nsplit;
  const int kh = bx % A.kvh, tile = bx / A.kvh;
  const int R = A.T * A.rep, r0 = tile * 128, rows = min(128, R - r0);
  const int n0 = A.by_rep.div(r0), n1 = A.by_rep.div(r0 + rows - 1);

  if (tid == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(&full[s], 128);  // the producers
      mbar_init(&empty[s], 1);   // one tcgen05.commit
    }
    for (int w = 0; w < W; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&o_full[w], 1);
      mbar_init(&drain[w], 1);
    }
    *abort = 0;
    range[0] = 0x7fffffff, range[1] = -1;
    slow[0] = slow[1] = slow[2] = slow[3] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)),
                 "r"((uint32_t)C::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // Zeros where the copies never write: dims past the heads' widths, rows past the tile's.
  for (int i = tid * 16; i < 2 * C::Q_TILE + NST * C::STAGE; i += C::THREADS * 16)
    *reinterpret_cast<uint4*>(sm + i) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  for (int n = n0 + tid; n <= n1; n += C::THREADS) {
    const int h = A.hi[(size_t)b * A.T + n];
    int l = max(A.lo[(size_t)b * A.T + n], 0);
    if (h >= 0) l = max(l, h - A.slots + 1);
    if (l <= h) {
      atomicMin(&range[0], l);
      atomicMax(&range[1], h);
    }
  }
  // Queries: two threads a row, each half of its dims; scaled by the power of
  // two that brings the row's max into [2^13, 2^14).
  if (tid < 256) {
    const int r = tid >> 1, half = tid & 1;
    const bool in = r < rows;
    const int rr = r0 + (in ? r : 0), n = A.by_rep.div(rr), h = kh * A.rep + rr - n * A.rep;
    const float* q = A.q + ((size_t)b * A.T + n) * A.ldq + (size_t)h * A.qk;
    constexpr int HC = QS;  // 8-dim chunks of a half row
    float mx = 0.f;
    for (int c = 0; c < HC; ++c)
      for (int i = 0; i < 8; ++i) {
        const int d = (half * HC + c) * 8 + i;
        if (in && d < A.qk) mx = fmaxf(mx, fabsf(__ldg(q + d)));
      }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    const int ef = (int)(__float_as_uint(mx) >> 23);
    const int ex = ef == 0 || ef >= 255 ? 0 : min(140 - ef, 126);
    const float by = __uint_as_float((uint32_t)(127 + ex) << 23);
    for (int c = 0; c < HC; ++c) {
      const int ch = half * HC + c;  // 16-byte chunk of the row: atom ch / 8
      uint32_t hh[4], ll[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = ch * 8 + 2 * i;
        const float x = in && d < A.qk ? __ldg(q + d) * by : 0.f, y = in && d + 1 < A.qk ? __ldg(q + d + 1) * by : 0.f;
        halves(x, y, &hh[i], &ll[i]);
      }
      const int at = (ch >> 3) * 128 * 128 + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
      *reinterpret_cast<uint4*>(qhi + at) = make_uint4(hh[0], hh[1], hh[2], hh[3]);
      *reinterpret_cast<uint4*>(qlo + at) = make_uint4(ll[0], ll[1], ll[2], ll[3]);
    }
    if (half == 0) row_q[r] = A.scale * __uint_as_float((uint32_t)(127 - ex) << 23);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int base = range[1] >= 0 ? range[0] : 0;
  const int n_ring = range[1] >= 0 ? (int)min((long)range[1] - base + 1, (long)A.slots) : 0;
  TreePlace P;
  P.ring = (size_t)b * A.slots * A.kvh + kh;
  P.draft = (size_t)b * A.T * A.kvh + kh;
  P.drafted = A.drafted, P.slot0 = base % A.slots, P.slots = A.slots, P.kvh = A.kvh, P.total = A.drafted + n_ring;
  const int blocks = (P.total + BN - 1) / BN;
  const int blk0 = (int)((long)blocks * z / A.nsplit), nblk = (int)((long)blocks * (z + 1) / A.nsplit) - blk0;

  // The row of a softmax thread (for the others: of thread tid % 128).
  const int r = tid & 127;
  const bool mine = r < rows;
  const int rr = r0 + min(r, rows - 1), node = A.by_rep.div(rr), head = kh * A.rep + rr - node * A.rep;
  const size_t node_at = (size_t)b * A.T + node;
  int start, cnt;
  {
    const int h = A.hi[node_at];
    int l = max(A.lo[node_at], 0);
    if (h >= 0) l = max(l, h - A.slots + 1);
    cnt = l <= h ? h - l + 1 : 0;
    start = cnt ? (int)((long)(l - base) % A.slots) : 0;
  }

  const int wg = warp >> 2;
  if (wg < W) {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_SOFT));
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + wg * C::WG_COLS, o_at = s_at + C::S_COLS;
    const float qs = row_q[r];
    // Positions every row of the warp sees without a look at the mask.
    int full0 = A.drafted + start, full1 = A.drafted + min(start + cnt, n_ring);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      full0 = max(full0, __shfl_xor_sync(0xffffffffu, full0, d));
      full1 = min(full1, __shfl_xor_sync(0xffffffffu, full1, d));
    }
    f32x2 o[VP / 2];  // dims 2 d, 2 d + 1
    float m = -INFINITY, l = 0.f;
    bool is_slow = false, ok = true;
#pragma unroll
    for (int d = 0; d < VP / 2; ++d) o[d] = pk(0.f, 0.f);
    const bool issuer = (tid & 127) == 0;

    auto issue_qk = [&](int i) {  // S of block i
      const int st = i % NST;
      if (!mbar_wait(&full[st], (uint32_t)(i / NST) & 1u, abort, werr)) return;
      tc_fence_after();
      unsigned char* kt = stages + (size_t)st * C::STAGE;
      const uint64_t dqh = sw128_desc(qhi), dql = sw128_desc(qlo), dk = sw128_desc(kt);
      uint32_t acc = 0;
      auto steps = [&](uint64_t dq, uint64_t dkk) {
#pragma unroll
        for (int k = 0; k < QS; ++k) {
          mma_ss<BN>(s_at, dq + (uint64_t)((k >> 2) * (128 * 128 >> 4) + (k & 3) * 2),
                     dkk + (uint64_t)((k >> 2) * (BN * 128 >> 4) + (k & 3) * 2), acc);
          acc = 1;
        }
      };
      steps(dql, dk);
      if (!I8) steps(dqh, dk + (uint64_t)(C::K_TILE >> 4));
      steps(dqh, dk);
      umma_commit(&s_full[wg]);
    };
    auto issue_pv = [&](int i) {  // O of block i
      const int st = i % NST;
      unsigned char* vt = stages + (size_t)st * C::STAGE + C::PARTS * C::K_TILE;
      const uint64_t dv = sw128_desc(vt);
      uint32_t acc = 0;
      auto steps = [&](uint32_t a, uint64_t dvv) {
#pragma unroll
        for (int k = 0; k < BN / 16; ++k) {
          mma_ts<VP>(o_at, a + k * 16, dvv + (uint64_t)((k >> 2) * (VP * 128 >> 4) + (k & 3) * 2),
                     acc);
          acc = 1;
        }
      };
      steps(s_at + 8, dv);
      if (!I8) steps(s_at, dv + (uint64_t)(C::V_TILE >> 4));
      steps(s_at, dv);
      umma_commit(&o_full[wg]);
      umma_commit(&empty[st]);
    };
    if (issuer && wg < nblk) issue_qk(wg);
    __syncwarp();

    int e_old = 14, it = 0;
    int low = 255;
    for (int i = wg; i < nblk; i += W, ++it) {
      const int st = i % NST;
      if (ok && !mbar_wait(&s_full[wg], (uint32_t)it & 1u, abort, werr)) ok = false;
      if (ok && !mbar_wait(&full[st], (uint32_t)(i / NST) & 1u, abort, werr)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        const int v0 = (blk0 + i) * BN;
        const float4* k4 = reinterpret_cast<const float4*>(col_k + st * BN);
        const float4* v4 = reinterpret_cast<const float4*>(col_v + st * BN);
        // ---- the block's max
        float mx = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < NC; ++c) {
          uint32_t x[2][16];
          tmem_ld16(s_at + lanes + c * 32, x[0]);
          tmem_ld16(s_at + lanes + c * 32 + 16, x[1]);
          const int v = v0 + c * 32;
          const bool all = v >= full0 && v + 32 <= full1;  // the same for the warp
          uint32_t sees = 0xffffffffu;
          if (!all) sees = mine ? tree_sees(A, node_at, node, start, cnt, n_ring, v) : 0u;
          is_slow |= (sees & odd[st * NC + c]) != 0;
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 k = k4[c * 8 + j];
            float a, d, e, f;
            const uint32_t* y = x[j >> 2] + 4 * (j & 3);
            up(mul2(pk(__uint_as_float(y[0]), __uint_as_float(y[1])), pk(k.x, k.y)), a, d);
            up(mul2(pk(__uint_as_float(y[2]), __uint_as_float(y[3])), pk(k.z, k.w)), e, f);
            if (!all) {
              const uint32_t w = sees >> (4 * j);
              a = w & 1 ? a : -INFINITY, d = w & 2 ? d : -INFINITY;
              e = w & 4 ? e : -INFINITY, f = w & 8 ? f : -INFINITY;
            }
            mx = fmaxf(mx, fmaxf(fmaxf(a, d), fmaxf(e, f)));
          }
        }
        const float mn = fmaxf(m, mx * qs), mz = mn == -INFINITY ? 0.f : mn;
        const float corr = ex2(m - mz);
        m = mn;
        // ---- the last block's output, then the new scale
        const int e = expo[2 * st];
        low = expo[2 * st + 1];
        if (it > 0) {
          if (!mbar_wait(&o_full[wg], (uint32_t)(it - 1) & 1u, abort, werr)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < VP; c += 16) {
            uint32_t x[16];
            tmem_ld16(o_at + lanes + c, x);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              o[(c + j) / 2] = add2(o[(c + j) / 2], pk(__uint_as_float(x[j]), __uint_as_float(x[j + 1])));
            }
          }
          const float by = corr * (e - e_old > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (e - e_old)) << 23));
          if (__any_sync(0xffffffffu, by != 1.f)) {
#pragma unroll
            for (int d = 0; d < VP / 2; ++d) o[d] = mul2(o[d], pk(by, by));
          }
        }
        e_old = e;
        // ---- weights: sum, and times the value scale as f16 parts into S's place
        // (16 positions at a time: their 16 columns take 8 of high parts, 8 of remainders)
        f32x2 add = pk(0.f, 0.f);
        const f32x2 qs2 = pk(qs, qs), mz2 = pk(-mz, -mz);
#pragma unroll 1
        for (int c = 0; c < 2 * NC; ++c) {
          uint32_t x[16];
          tmem_ld16(s_at + lanes + c * 16, x);
          const int v = v0 + (c >> 1) * 32;
          const bool all = v >= full0 && v + 32 <= full1;
          uint32_t seen = 0xffffffffu;
          if (!all) seen = mine ? tree_sees(A, node_at, node, start, cnt, n_ring, v) >> ((c & 1) * 16) : 0u;
          tmem_wait_ld();
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 k = k4[c * 4 + j], vv = v4[c * 4 + j];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float a, d;
              up(fma2(mul2(pk(__uint_as_float(x[4 * j + 2 * h]), __uint_as_float(x[4 * j + 2 * h + 1])),
                           h ? pk(k.z, k.w) : pk(k.x, k.y)),
                      qs2, mz2),
                 a, d);
              if (!all) {
                const uint32_t w = seen >> (4 * j + 2 * h);
                a = w & 1 ? a : -INFINITY, d = w & 2 ? d : -INFINITY;
              }
              const f32x2 p = pk(ex2(a), ex2(d));
              add = add2(add, p);
              float wa, wd;
              up(mul2(p, h ? pk(vv.z, vv.w) : pk(vv.x, vv.y)), wa, wd);
              const float ta = __uint_as_float(__float_as_uint(wa) & 0xffffe000u),
                          td = __uint_as_float(__float_as_uint(wd) & 0xffffe000u);
              hi[2 * j + h] = cvt2(ta, td);
              lo[2 * j + h] = cvt2(wa - ta, wd - td);
            }
          }
          tmem_st8(s_at + lanes + c * 16, hi);
          tmem_st8(s_at + lanes + c * 16 + 8, lo);
        }
        float a, d;
        up(add, a, d);
        l = l * corr + (a + d);
        tmem_wait_st();
        tc_fence_before();
      }
      if (W == 1 || wg == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
      else asm volatile("bar.sync 2, 128;" ::: "memory");
      if (issuer && ok) {
        tc_fence_after();
        issue_pv(i);
        // The next S takes the place of this P: only once the product is done.
        if (i + W < nblk && mbar_wait(&o_full[wg], (uint32_t)it & 1u, abort, werr)) issue_qk(i + W);
      }
      __syncwarp();
    }
    if (it > 0) {
      if (ok && !mbar_wait(&o_full[wg], (uint32_t)(it - 1) & 1u, abort, werr)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        // Outputs to their own scale. A row whose output came out infinite or
        // NaN, or far below what the block's largest value scale holds bits
        // for, is done again.
        const float by = __uint_as_float((uint32_t)(e_old - 13) << 23);
        float top = 0.f;
        bool bad = false;
#pragma unroll
        for (int c = 0; c < VP; c += 16) {
          uint32_t x[16];
          tmem_ld16(o_at + lanes + c, x);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const f32x2 t = add2(o[(c + j) / 2], pk(__uint_as_float(x[j]), __uint_as_float(x[j + 1])));
            float t0, t1;
            up(t, t0, t1);
            top = fmaxf(top, fmaxf(fabsf(t0), fabsf(t1)));
            bad |= !(fabsf(t0) <= 3.4028234e38f) || !(fabsf(t1) <= 3.4028234e38f);
            o[(c + j) / 2] = mul2(t, pk(by, by));
          }
        }
        is_slow |= bad || (e_old - low > 12 && l > 0.f && top < (I8 ? 2.f : 16384.f) * l);
      } else {  // a wait gave up: the flag is up, and the rows say so
#pragma unroll
        for (int d = 0; d < VP / 2; ++d) o[d] = pk(__uint_as_float(0x7fc00000u), __uint_as_float(0x7fc00000u));
        l = 1.f, m = 0.f;
        is_slow = false;
      }
    }
    if (issuer) {  // every issued MMA completes before TMEM is freed
      umma_commit(&drain[wg]);
      mbar_drain(&drain[wg], 0);
    }
    __syncwarp();
    if (mine && is_slow) atomicOr(&slow[r >> 5], 1u << (r & 31));
    // ---- merge the warpgroups (every block is consumed: the stages' memory is
    // free) and write
    if (W == 2) {
      // [VP / 2][128] pairs, then [2][128] max and sum
      f32x2* xch = reinterpret_cast<f32x2*>(stages);
      float* xml = reinterpret_cast<float*>(xch + VP / 2 * 128);
      asm volatile("bar.sync 3, 256;" ::: "memory");
      if (wg == 1) {
#pragma unroll
        for (int d = 0; d < VP / 2; ++d) xch[d * 128 + r] = o[d];
        xml[r] = m, xml[128 + r] = l;
      }
      asm volatile("bar.sync 3, 256;" ::: "memory");
      is_slow = (slow[r >> 5] >> (r & 31)) & 1;
      if (wg == 0) {
        const float m1 = xml[r], l1 = xml[128 + r], M = fmaxf(m, m1);
        // a sum without a max is NaN, and stays
        const float f0 = l == 0.f ? 0.f : m == -INFINITY ? 1.f : ex2(m - M);
        const float f1 = l1 == 0.f ? 0.f : m1 == -INFINITY ? 1.f : ex2(m1 - M);
#pragma unroll
        for (int d = 0; d < VP / 2; ++d) {
          const f32x2 c = f1 == 0.f ? pk(0.f, 0.f) : mul2(xch[d * 128 + r], pk(f1, f1));
          o[d] = add2(f0 == 0.f ? pk(0.f, 0.f) : mul2(o[d], pk(f0, f0)), c);
        }
        l = (f0 == 0.f ? 0.f : f0 * l) + (f1 == 0.f ? 0.f : f1 * l1);
        m = M;
      }
    }
    if (wg == 0 && mine && !is_slow) {
      if (A.nsplit > 1) {
        float* dst = A.part + ((((size_t)b * A.kvh + kh) * A.nsplit + z) * R + rr) * (A.vh + 2);
#pragma unroll
        for (int d = 0; d < VP; d += 2)
          if (d < A.vh) *reinterpret_cast<f32x2*>(dst + d) = o[d / 2];
        *reinterpret_cast<float2*>(dst + A.vh) = make_float2(m, l);
      } else {
        float* dst = A.out + (node_at * A.heads + head) * A.vh;
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int d = 0; d < VP; d += 2)  // vh and the start of out are multiples of two floats
          if (d < A.vh) *reinterpret_cast<f32x2*>(dst + d) = mul2(o[d / 2], pk(inv, inv));
      }
    }
  } else {
    // ------------------------------------------------------------ producers
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_PROD));
    const int p = tid - W * 128, pw = p >> 5;
    bool ok = true;
    int e = 14, low = 255;
    for (int i = 0; i < nblk; ++i) {
      const int st = i % NST, v0 = (blk0 + i) * BN;
      unsigned char* kt = stages + (size_t)st * C::STAGE;
      unsigned char* vt = kt + C::PARTS * C::K_TILE;
      const bool wait_empty = ok;
      if (I8) {
        // Keys: a position a thread. Values: eight positions (octet) by VP / 8
        // dims a thread; a warp reads whole sectors and writes one 16-byte
        // chunk of eight positions per dim, lanes in different chunks.
        constexpr int DV = VP / 8;  // dims of a thread
        const int v = v0 + p, pr = (pw & 1) * 8 + (lane & 7), d0 = ((pw >> 1) * 4 + (lane >> 3)) * DV;
        uint4 k[QS];
        uint32_t x[8][DV / 4];
        float ksc = 0.f, vsc = 0.f;
        {
          const bool in = v < P.total;
          const bool d = P.in_draft(v);
          const size_t row = in ? P.row(v) : 0;
          if (in) ksc = (d ? A.tks : A.ks)[row], vsc = (d ? A.tvs : A.vs)[row];
          const char* src = (d ? A.tk : A.k) + row * A.qk;
#pragma unroll
          for (int c = 0; c < QS; ++c)
            k[c] = in && c * 16 < A.qk ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int vj = v0 + pr * 8 + j;
          const bool in = vj < P.total && d0 < A.vh;
          const char* src = (P.in_draft(vj) ? A.tv : A.v) + (in ? P.row(vj) : 0) * A.vh + d0;
          if (DV == 8) {
            const uint2 t = in ? __ldg(reinterpret_cast<const uint2*>(src)) : make_uint2(0, 0);
            x[j][0] = t.x, x[j][1] = t.y;
          } else {
            const uint4 t = in ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
            x[j][0] = t.x, x[j][1] = t.y, x[j][DV / 4 - 2] = t.z, x[j][DV / 4 - 1] = t.w;
          }
        }
        if (wait_empty && !mbar_wait(&empty[st], ((uint32_t)(i / NST) & 1u) ^ 1u, abort, werr)) ok = false;
        // scales
        const bool sane = fabsf(ksc) <= 3.4028234e38f && fabsf(vsc) <= 3.4028234e38f;
        const uint32_t oddw = __ballot_sync(0xffffffffu, !sane);
        if (!sane) vsc = 0.f;
        const uint32_t vb = __float_as_uint(fabsf(vsc));
        const uint32_t hi = __reduce_max_sync(0xffffffffu, vb),
                       lo = __reduce_min_sync(0xffffffffu, vb ? vb : 0x7f800000u);
        uint32_t* wm = reinterpret_cast<uint32_t*>(wmax) + (i & 1) * 8;
        if (lane == 0) wm[pw] = hi, wm[4 + pw] = lo;
        if (lane == 0) odd[st * NC + pw] = oddw;
        asm volatile("bar.sync 4, 128;" ::: "memory");
        e = min(max(e, (int)(max(max(wm[0], wm[1]), max(wm[2], wm[3])) >> 23)), 253);
        low = min(low, (int)(min(min(wm[4], wm[5]), min(wm[6], wm[7])) >> 23));
        col_k[st * BN + p] = ksc;
        col_v[st * BN + p] = vsc * __uint_as_float((uint32_t)(267 - e) << 23);
        if (p == 0) expo[2 * st] = e, expo[2 * st + 1] = low;
        // keys
#pragma unroll
        for (int c = 0; c < QS; ++c) {
          uint32_t w[8];
          widen(k[c].x ^ 0x80808080u, &w[0], &w[1]);
          widen(k[c].y ^ 0x80808080u, &w[2], &w[3]);
          widen(k[c].z ^ 0x80808080u, &w[4], &w[5]);
          widen(k[c].w ^ 0x80808080u, &w[6], &w[7]);
          unsigned char* row = kt + (c >> 2) * (BN * 128) + p * 128;
          *reinterpret_cast<uint4*>(row + ((((c & 3) * 2) ^ (p & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(row + ((((c & 3) * 2 + 1) ^ (p & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
        }
        // values, transposed: dims 2g, 2g + 1 of two positions in one permute
        if (d0 < A.vh) {
#pragma unroll
          for (int q = 0; q < DV / 4; ++q) {
            uint32_t w[4][4];  // [dim][position pair]
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t a = x[2 * j][q] ^ 0x80808080u, c = x[2 * j + 1][q] ^ 0x80808080u;
              widen(__byte_perm(a, c, 0x5140), &w[0][j], &w[1][j]);
              widen(__byte_perm(a, c, 0x7362), &w[2][j], &w[3][j]);
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const int d = d0 + 4 * q + t;
              *reinterpret_cast<uint4*>(vt + (pr >> 3) * (VP * 128) + d * 128 + (((pr & 7) ^ (d & 7)) << 4)) =
                  make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]);
            }
          }
        }
      } else {
        // f32, BN = 64. Keys: two threads a position. Values: eight positions
        // by four dims a thread.
        constexpr int HC = QS;  // 8-dim chunks of half a key row
        const int kp = p >> 1, half = p & 1, v = v0 + kp;
        const int pr = lane & 7, d0 = (pw * 4 + (lane >> 3)) * 4;
        float4 x[8];
        bool sane = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int vj = v0 + pr * 8 + j;
          const bool in = vj < P.total && d0 < A.vh;
          const float* src =
              reinterpret_cast<const float*>(P.in_draft(vj) ? A.tv : A.v) + (in ? P.row(vj) : 0) * A.vh + d0;
          x[j] = in ? __ldg(reinterpret_cast<const float4*>(src)) : make_float4(0, 0, 0, 0);
        }
        if (wait_empty && !mbar_wait(&empty[st], ((uint32_t)(i / NST) & 1u) ^ 1u, abort, werr)) ok = false;
        float ksc;
        {
          const bool in = v < P.total;
          const float* src = reinterpret_cast<const float*>(P.in_draft(v) ? A.tk : A.k) + (in ? P.row(v) : 0) * A.qk;
          float4 k[HC][2];
          float mx = 0.f;
#pragma unroll
          for (int c = 0; c < HC; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int d = (half * HC + c) * 8 + 4 * h;
              k[c][h] = in && d < A.qk ? __ldg(reinterpret_cast<const float4*>(src + d)) : make_float4(0, 0, 0, 0);
              mx = fmaxf(mx, fmaxf(fmaxf(fabsf(k[c][h].x), fabsf(k[c][h].y)), fmaxf(fabsf(k[c][h].z), fabsf(k[c][h].w))));
              sane &= fabsf(k[c][h].x) <= 3.4028234e38f && fabsf(k[c][h].y) <= 3.4028234e38f &&
                      fabsf(k[c][h].z) <= 3.4028234e38f && fabsf(k[c][h].w) <= 3.4028234e38f;
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          const int ef = min(max((int)(__float_as_uint(mx) >> 23), 14), 253);
          const float by = __uint_as_float((uint32_t)(267 - ef) << 23);  // max into [2^13, 2^14)
          ksc = __uint_as_float((uint32_t)(ef - 13) << 23);
#pragma unroll
          for (int c = 0; c < HC; ++c) {
            uint32_t hh[4], ll[4];
            halves(k[c][0].x * by, k[c][0].y * by, &hh[0], &ll[0]);
            halves(k[c][0].z * by, k[c][0].w * by, &hh[1], &ll[1]);
            halves(k[c][1].x * by, k[c][1].y * by, &hh[2], &ll[2]);
            halves(k[c][1].z * by, k[c][1].w * by, &hh[3], &ll[3]);
            const int ch = half * HC + c;
            unsigned char* at = kt + (ch >> 3) * (BN * 128) + kp * 128 + (((ch & 7) ^ (kp & 7)) << 4);
            *reinterpret_cast<uint4*>(at) = make_uint4(hh[0], hh[1], hh[2], hh[3]);
            *reinterpret_cast<uint4*>(at + C::K_TILE) = make_uint4(ll[0], ll[1], ll[2], ll[3]);
          }
        }
        uint32_t oddk = __ballot_sync(0xffffffffu, !sane);  // two lanes a position: positions 16 pw ..
        // largest value of each position: over the warp's dims, then the warps'
        float* wm = wmax + (i & 1) * 256;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float a = fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w)));
          // NaN and infinity both read as infinity
          const float s = fabsf(x[j].x) + fabsf(x[j].y) + fabsf(x[j].z) + fabsf(x[j].w);
          if (!(a <= 3.4028234e38f) || s != s) a = INFINITY;
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 8));
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 16));
          if (lane < 8) wm[pw * 64 + pr * 8 + j] = a;
        }
        uint32_t* om = odd + st * NC;
        if (p < NC) om[p] = 0;
        asm volatile("bar.sync 4, 128;" ::: "memory");
        float mxs[8];
        int top = 0, least = 255;
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at = pr * 8 + j;
          const float a = fmaxf(fmaxf(wm[at], wm[64 + at]), fmaxf(wm[128 + at], wm[192 + at]));
          mxs[j] = a;
          if (a == INFINITY) {
            bad |= 1u << j;
          } else if (a > 0.f) {
            const int f = min(max((int)(__float_as_uint(a) >> 23), 14), 253) - 13;
            top = max(top, f), least = min(least, f);
          }
        }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) {
          top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
          least = min(least, __shfl_xor_sync(0xffffffffu, least, d));
        }
        e = max(e, top), low = min(low, least);
        // odd columns: bits 8 (pr % 4) + j of word pr / 4 for values, spread pairs for keys
        if (pw == 0 && lane < 8 && bad) atomicOr(&om[pr >> 2], bad << ((pr & 3) * 8));
        if (lane == 0 && oddk) {
          uint32_t w = 0;
          for (int j = 0; j < 16; ++j)
            if ((oddk >> (2 * j)) & 3u) w |= 1u << j;
          atomicOr(&om[pw >> 1], w << ((pw & 1) * 16));
        }
        if (half == 0) col_k[st * BN + kp] = v < P.total ? ksc : 0.f;
        if (p == 0) expo[2 * st] = e, expo[2 * st + 1] = low;
        uint32_t hh[4][4], ll[4][4];  // [dim][position pair]
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float by[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float a = mxs[2 * j + h];
            const int ef = min(max((int)(__float_as_uint(a) >> 23), 14), 253);
            const bool use = a > 0.f && a != INFINITY;
            by[h] = use ? __uint_as_float((uint32_t)(267 - ef) << 23) : 0.f;
            // value scale 2^(ef - 140) times 2^(140 - e): exponent ef - 13 below e
            const int f = 127 + 13 + ef - 13 - e;
            if (pw == 0 && lane < 8)
              col_v[st * BN + pr * 8 + 2 * j + h] = use && f > 0 ? __uint_as_float((uint32_t)f << 23) : 0.f;
          }
          const float4 a = x[2 * j], c = x[2 * j + 1];
          const bool ua = by[0] != 0.f, uc = by[1] != 0.f;
          halves(ua ? a.x * by[0] : 0.f, uc ? c.x * by[1] : 0.f, &hh[0][j], &ll[0][j]);
          halves(ua ? a.y * by[0] : 0.f, uc ? c.y * by[1] : 0.f, &hh[1][j], &ll[1][j]);
          halves(ua ? a.z * by[0] : 0.f, uc ? c.z * by[1] : 0.f, &hh[2][j], &ll[2][j]);
          halves(ua ? a.w * by[0] : 0.f, uc ? c.w * by[1] : 0.f, &hh[3][j], &ll[3][j]);
        }
        if (d0 < A.vh) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int d = d0 + t;
            unsigned char* at = vt + d * 128 + ((pr ^ (d & 7)) << 4);
            *reinterpret_cast<uint4*>(at) = make_uint4(hh[t][0], hh[t][1], hh[t][2], hh[t][3]);
            *reinterpret_cast<uint4*>(at + C::V_TILE) = make_uint4(ll[t][0], ll[t][1], ll[t][2], ll[t][3]);
          }
        }
        asm volatile("bar.sync 4, 128;" ::: "memory");  // the odd words are whole
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&full[st]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TMEM));
  }
  // ---- rows to do again, a warp each
  for (int wd = 0; wd < 4; ++wd) {
    uint32_t todo = slow[wd];
    int turn = 0;
    while (todo) {
      const int r2 = wd * 32 + __ffs(todo) - 1;
      todo &= todo - 1;
      if (turn++ % (C::THREADS / 32) != warp) continue;
      const int q2 = r0 + r2, n2 = A.by_rep.div(q2), h2 = kh * A.rep + q2 - n2 * A.rep;
      const size_t at2 = (size_t)b * A.T + n2;
      const int hh = A.hi[at2];
      int ll = max(A.lo[at2], 0);
      if (hh >= 0) ll = max(ll, hh - A.slots + 1);
      const int c2 = ll <= hh ? hh - ll + 1 : 0, s2 = c2 ? (int)((long)(ll - base) % A.slots) : 0;
      float m2, l2, o2[4];
      tree_slow_row<I8>(A, P, at2, n2, h2, s2, c2, n_ring, blk0 * BN, min((blk0 + nblk) * BN, P.total), &m2, &l2, o2);
      float* dst = A.nsplit > 1 ? A.part + ((((size_t)b * A.kvh + kh) * A.nsplit + z) * R + q2) * (A.vh + 2)
                                : A.out + (at2 * A.heads + h2) * A.vh;
      for (int j = 0; j < 4; ++j)
        if (lane + 32 * j < A.vh) dst[lane + 32 * j] = A.nsplit > 1 ? o2[j] : l2 == 0.f ? 0.f : o2[j] / l2;
      if (A.nsplit > 1 && lane == 0) dst[A.vh] = m2, dst[A.vh + 1] = l2;
    }
  }
}

template <class C>
cudaError_t launch_umma_form(const TreeArgs& A, int B, cudaStream_t st) {
  auto kern = tree_umma_kernel<C>;
  cudaError_t e = allow_smem((const void*)kern, C::SMEM);
  if (e != cudaSuccess) return e;
  // The warpgroups' register shares assume the launch's: another count would
  // leave setmaxnreg waiting.
  static const int regs = [kern] {
    cudaFuncAttributes fa;
    return cudaFuncGetAttributes(&fa, (const void*)kern) == cudaSuccess ? fa.numRegs : -1;
  }();
  if (regs != C::REG_ALL) return cudaErrorNotSupported;
  int* werr = nullptr;
  e = umma_error_ptr(&werr);
  if (e != cudaSuccess) return e;
  const int R = A.T * A.rep, tiles = (R + 127) / 128;
  for (int b0 = 0; b0 < B; b0 += 65535) {
    const int n = std::min(65535, B - b0);
    const TreeArgs S = tree_sessions(A, b0, C::I8 ? 1 : 4);
    kern<<<dim3((unsigned)tiles * A.kvh * A.nsplit, n), C::THREADS, C::SMEM, st>>>(S, werr);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

typedef TreeUmma<true, 3, 64, 1, 128, 2> UmmaI8x48;
typedef TreeUmma<true, 4, 64, 1, 128, 2> UmmaI8x64;
typedef TreeUmma<true, 8, 128, 2, 128, 2> UmmaI8x128;
typedef TreeUmma<false, 3, 64, 1, 64, 2> UmmaF32x48;
typedef TreeUmma<false, 4, 64, 1, 64, 2> UmmaF32x64;

}  // namespace

bool tree_umma_takes(int int8, int rows, int qk, int vh, int piece) {
  if (piece != 16 || qk % 16 || vh % 16 || rows < 48) return false;
  return int8 || (qk <= 64 && vh <= 64);
}

// Splits that need the fewest rounds of blocks: a block of positions costs
// about 1, a CTA's start and end about 4.
int tree_umma_nsplit(int int8, int B, int rows, int kvh, int qk, int vh, int span) {
  const bool wide = qk > 64 || vh > 64;
  const long work = (long)B * kvh * ((rows + 127) / 128), room = 148 * (wide ? 1 : 2);
  const int bn = int8 ? 128 : 64, blocks = (span + bn - 1) / bn;
  int best = 1;
  double cost = 1e300;
  for (int ns = 1; ns <= 128 && ns <= blocks; ++ns) {
    const double c = (double)((work * ns + room - 1) / room) * ((blocks + ns - 1) / ns + 4) + (ns > 1 ? 4.0 : 0.0);
    if (c < cost * 0.97) cost = c, best = ns;
  }
  return best;
}

cudaError_t launch_tree_umma(const TreeArgs& A, int int8, int B, cudaStream_t st) {
  if (int8) {
    if (A.qk > 64 || A.vh > 64) return launch_umma_form<UmmaI8x128>(A, B, st);
    if (A.qk > 48) return launch_umma_form<UmmaI8x64>(A, B, st);
    return launch_umma_form<UmmaI8x48>(A, B, st);
  }
  if (A.qk > 48) return launch_umma_form<UmmaF32x64>(A, B, st);
  return launch_umma_form<UmmaF32x48>(A, B, st);
}

}  // namespace nb
