// nd_attend_tree on the 5th-generation tensor cores, for trees with more than 16
// rows (T * rep) of a KV head.
//
//   S = Q K^T,  P = 2^(S * scales - max),  O += P V
//
// per step of 64 positions: S and O lie in tensor memory (TMEM), a softmax
// warpgroup holds one row a thread, P returns to TMEM in S's place as the A
// operand of the second product. f32 accuracy from f16 operands: the query and
// P are f16 high parts and remainders (22 bits; int8 codes are f16 values
// exactly; f32 keys and values are split the same way after a power-of-two
// scale per position, which is then treated like an int8 scale; an element far
// below its vector's largest is held to 2^-38 of that, where f16 ends). The products
// with remainders go first: the tensor cores truncate when they accumulate,
// and truncation costs only what the sum already holds. For the same reason O
// is drained into f32 registers after every block.
//
// Warps: one softmax warpgroup with a thread a row, or, for 128-wide heads,
// whose outputs would fill a thread's registers, and for f32, two with half of a
// row's positions and half of its outputs each (they tell each other their
// maxima), and one warpgroup (f32: two) of
//   a key warp and two value warps (f32: two and four, whose conversion is what
//   bounds a step: a chain of 3300 cycles of 64 positions, 5400 with the maxima
//   of eight positions reduced one after another), which read the ring and the
//   draft, turn them to f16 and lay them down in the 128-byte swizzled form the
//   MMA reads (keys as they lie, values transposed eight positions at a time in
//   registers; of int8 the key warp also forms the steps' scales), and
//   an MMA warp, which issues every product as soon as its operands stand: a
//   warp that issues MMAs is held for as long as they run.
// int8 heads of up to 64 leave room for two blocks on an SM, which hide each
// other's latencies; the others take a whole SM.
//
// Measured: 256 sessions x 96 rows x 1043 int8 positions (48/64) 77 us (0.9 TB/s,
// 20 % of the tensor pipe); 16 x 288 rows x 2051 f32 positions 65 us; 4 x 8 heads x
// 128 rows x 32771 int8 positions (128 wide) 220 to 228 us (1.1 TB/s, 28 %). The chain of a
// softmax step bounds the int8 forms: about 2900 cycles alone, 4300 with two blocks
// on the SM, no pipe above 40 %.
//
// Every wait is bounded as in umma_gemm.cu.
#include <algorithm>

#include "kernels.hpp"
#include "launch_util.hpp"
#include "tree.cuh"
#include "umma.cuh"

namespace nb {
namespace {

template <bool I8_, int QS_, int VP_, int TPR_, int NST_>
struct TreeUmma {
  static constexpr bool I8 = I8_;
  static constexpr int QS = QS_;        // k16 steps of the key product
  static constexpr int VP = VP_;        // value width held (64 or 128)
  static constexpr int TPR = TPR_;      // softmax threads a row
  static constexpr int OW = VP / TPR;   // outputs of a softmax thread
  static constexpr int NST = NST_;
  static constexpr int BN = 64;         // positions of a stage, and of a step of the softmax
  static constexpr int CW = BN / TPR;   // positions of a softmax thread's step
  static constexpr int KA = (QS * 16 + 63) / 64;  // 64-wide swizzle atoms of a key row
  static constexpr int PARTS = I8 ? 1 : 2;        // high part, remainder
  static constexpr int Q_TILE = KA * 128 * 128, K_TILE = KA * BN * 128, V_TILE = VP * 128;
  static constexpr int STAGE = PARTS * (K_TILE + V_TILE);
  static constexpr int PWG = I8 ? 1 : 2;        // warpgroups that read keys and values and issue MMAs
  static constexpr int KW = I8 ? 1 : 2, VW = I8 ? 2 : 4;  // key and value warps among them
  static constexpr int THREADS = (TPR + PWG) * 128, CTAS = I8 && TPR == 1 ? 2 : 1;
  // Registers a thread: the launch's, a softmax thread's, the other warpgroups';
  // the warpgroups' shares add up to the launch's.
  static constexpr int REG_ALL = I8 && TPR == 2 ? 168 : 128,
                       REG_SOFT = I8 ? (TPR == 1 ? 184 : 176) : VP == 64 ? 144 : 160,
                       REG_PROD = ((TPR + PWG) * REG_ALL - TPR * REG_SOFT) / PWG;
  static_assert(TPR * REG_SOFT + PWG * REG_PROD == (TPR + PWG) * REG_ALL && REG_PROD % 8 == 0 &&
                    THREADS * CTAS * REG_ALL <= 65536 && REG_SOFT >= REG_ALL,
                "register shares");
  static constexpr int TMEM = 2 * BN + VP <= 128 ? 128 : 256;  // columns: two of S (then P), O
  static constexpr size_t META = NST * (size_t)(BN * 8 + 16 + 16) + 128 * 4 + 512 + 2 * 2 * 128 * 4;
  static constexpr size_t SMEM = 1024 + 2 * (size_t)Q_TILE + NST * (size_t)STAGE + META;
};

__device__ __forceinline__ void tmem_st8(uint32_t t, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]));
}
// As tmem_wait_ld, but ordinary loads may move across it.
__device__ __forceinline__ void tmem_landed() { asm volatile("tcgen05.wait::ld.sync.aligned;"); }
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

// One lane of a converged warp, in a form the compiler knows to be uniform.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
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
// tree_slow_row out of line: inlined, it cost the roles registers (48 nodes f32 65.8
// -> 72 us). A row of 2051 positions takes a warp 1.6 ms: with an infinite value in
// every head's sight 48 nodes take 27 ms.
template <bool I8>
__device__ __noinline__ void tree_slow_call(const TreeArgs& A, const TreePlace& P, size_t node_at, int node, int head,
                                            int start, int cnt, int n_ring, int v0, int v1, float* m, float* l,
                                            float (&o)[4]) {
  const float* q = A.q + node_at * A.ldq + (size_t)head * A.qk;
  bool none = false;
  for (int i = threadIdx.x & 31; i < A.qk; i += 32) none |= q[i] != q[i];
  if (__any_sync(0xffffffffu, none)) {  // a NaN in the query (a padding node's, say): so is all it sees
    *l = __uint_as_float(0x7fc00000u);
    return;
  }
  tree_slow_row<I8>(A, P, node_at, node, head, start, cnt, n_ring, v0, v1, m, l, o);
}

// Grid (tiles of 128 rows * kvh * nsplit, sessions).
template <class C>
__global__ void __launch_bounds__(C::THREADS, C::CTAS) tree_umma_kernel(const __grid_constant__ TreeArgs A, int* werr) {
  constexpr bool I8 = C::I8;
  constexpr int BN = C::BN, VP = C::VP, QS = C::QS, TPR = C::TPR, OW = C::OW, CW = C::CW, NST = C::NST, NC = BN / 32;
  extern __shared__ unsigned char raw[];
  // An offset, not a rounded integer: the compiler keeps track of the address space.
  unsigned char* sm = raw + ((0u - su32(raw)) & 1023u);
  unsigned char *qhi = sm, *qlo = sm + C::Q_TILE, *stages = sm + 2 * C::Q_TILE;
  float* col_k = reinterpret_cast<float*>(stages + (size_t)NST * C::STAGE);  // [NST][BN] key scales
  float* col_v = col_k + NST * BN;                                          // [NST][BN] value scales times 2^(140 - e)
  uint32_t* odd = reinterpret_cast<uint32_t*>(col_v + NST * BN);            // [NST][NC] columns to keep out (f32: of keys, of values)
  int* expo = reinterpret_cast<int*>(odd + NST * 4);                       // [NST][2] e, least exponent so far
  float* row_q = reinterpret_cast<float*>(expo + 2 * NST);                  // [128] score scale of a row
  uint64_t* full = reinterpret_cast<uint64_t*>(row_q + 128);
  uint64_t* empty = full + NST;
  uint64_t* s_full = empty + NST;  // [2] S of a step
  uint64_t* o_full = s_full + 2;   // O of a step
  uint64_t* p_full = o_full + 1;   // P of a step, one arrival a softmax warp with rows
  uint64_t* q_full = p_full + 1;   // the queries
  uint64_t* drain = q_full + 1;    // every MMA
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile uint32_t* abort = tmem_slot + 1;
  int* range = reinterpret_cast<int*>(tmem_slot + 2);    // [2]
  uint32_t* slow = reinterpret_cast<uint32_t*>(range + 2);  // [4] rows for tree_slow_row
  int* vmax = reinterpret_cast<int*>(slow + 4);             // [2][8] the value warps' exponents
  float* both = reinterpret_cast<float*>(full) + 128;       // [2][2][128] what two threads of a row tell each other

  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int b = blockIdx.y;
  int bx = blockIdx.x;
  const int z = bx % A.nsplit;
  bx /= A.nsplit;
  const int kh = bx % A.kvh, tile = bx / A.kvh;
  const int R = A.T * A.rep, r0 = tile * 128, rows = min(128, R - r0);
  const int n0 = A.by_rep.div(r0), n1 = A.by_rep.div(r0 + rows - 1);

  if (tid == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(&full[s], 32 * (C::KW + C::VW));  // the key and value warps
      mbar_init(&empty[s], 1);   // one tcgen05.commit
    }
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(o_full, 1);
    mbar_init(p_full, TPR * ((rows + 31) / 32));
    mbar_init(q_full, 128);
    mbar_init(drain, 1);
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
  // Zeros where nothing is ever written: dims past the heads' widths.
  if (A.qk != QS * 16 || A.vh != VP)
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
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
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
  if (wg < TPR) {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_SOFT));
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + wg * CW, o_at = tmem + 2 * BN + wg * OW;  // the thread's columns of S and O
    // ---- queries: a row a thread of the first warpgroup, scaled by the power
    // of two that brings the row's max into [2^13, 2^14)
    if (wg == 0) {
      const float* q = A.q + node_at * A.ldq + (size_t)head * A.qk;
      float x[QS * 16];
      if (mine && (reinterpret_cast<uintptr_t>(q) & 15) == 0) {
#pragma unroll
        for (int c = 0; c < QS * 4; ++c) {
          const float4 f = c * 4 < A.qk ? __ldg(reinterpret_cast<const float4*>(q) + c) : make_float4(0, 0, 0, 0);
          x[4 * c] = f.x, x[4 * c + 1] = f.y, x[4 * c + 2] = f.z, x[4 * c + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < QS * 16; ++i) x[i] = mine && i < A.qk ? __ldg(q + i) : 0.f;
      }
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < QS * 16; ++i) mx = fmaxf(mx, fabsf(x[i]));
      const int ef = (int)(__float_as_uint(mx) >> 23);
      const int ex = ef == 0 || ef >= 255 ? 0 : min(140 - ef, 126);
      const float by = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
      for (int c = 0; c < 2 * QS; ++c) {
        uint32_t hh[4], ll[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) halves(x[8 * c + 2 * i] * by, x[8 * c + 2 * i + 1] * by, &hh[i], &ll[i]);
        const int at = (c >> 3) * 128 * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(qhi + at) = make_uint4(hh[0], hh[1], hh[2], hh[3]);
        *reinterpret_cast<uint4*>(qlo + at) = make_uint4(ll[0], ll[1], ll[2], ll[3]);
      }
      row_q[r] = A.scale * __uint_as_float((uint32_t)(127 - ex) << 23);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(q_full);
    }
    if (TPR == 2) asm volatile("bar.sync 5, 256;" ::: "memory");
    const float qs = row_q[r];
    // Positions every row of the warp sees without a look at the mask.
    int full0 = A.drafted + start, full1 = A.drafted + min(start + cnt, n_ring);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      full0 = max(full0, __shfl_xor_sync(0xffffffffu, full0, d));
      full1 = min(full1, __shfl_xor_sync(0xffffffffu, full1, d));
    }
    f32x2 o[OW / 2];  // dims 2 d, 2 d + 1 of the thread's
    float m = -INFINITY, l = 0.f;
    bool is_slow = false, ok = true;
#pragma unroll
    for (int d = 0; d < OW / 2; ++d) o[d] = pk(0.f, 0.f);
    // Warps whose rows are all padding take no part.
    const int nj = (warp & 3) * 32 < rows ? nblk : 0;
    // What a thread has for the other of its row, and has from it; `turn`
    // alternates between two places, so one meeting a turn is enough.
    auto meet = [&](int turn, float mine_) {
      both[turn * 256 + wg * 128 + r] = mine_;
      if ((warp & 3) == 0) asm volatile("bar.sync 1, 64;" ::: "memory");
      else if ((warp & 3) == 1) asm volatile("bar.sync 2, 64;" ::: "memory");
      else if ((warp & 3) == 2) asm volatile("bar.sync 3, 64;" ::: "memory");
      else asm volatile("bar.sync 6, 64;" ::: "memory");
      return both[turn * 256 + (1 - wg) * 128 + r];
    };

    int e_old = 14;
    int low = 255;
    for (int i = 0; i < nj; ++i) {
      const int st = i % NST;
      if (ok && !mbar_wait_spin(&s_full[i & 1], (uint32_t)(i >> 1) & 1u, abort, werr)) ok = false;
      if (ok && !mbar_wait_spin(&full[st], (uint32_t)(i / NST) & 1u, abort, werr)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      float mx = -INFINITY;
      f32x2 s[CW / 2];
      const uint32_t s_now = s_at + lanes + (i & 1) * BN;
      const float4* v4 = reinterpret_cast<const float4*>(col_v + st * BN + wg * CW);
      if (ok) {
        tc_fence_after();
        const int v0 = (blk0 + i) * BN + wg * CW;
        const float4* k4 = reinterpret_cast<const float4*>(col_k + st * BN + wg * CW);
        const bool all = v0 >= full0 && v0 + CW <= full1;  // the same for the warp
        uint32_t sees[CW / 32];
#pragma unroll
        for (int c = 0; c < CW / 32; ++c) {
          sees[c] = 0xffffffffu;
          if (!all) sees[c] = mine ? tree_sees(A, node_at, node, start, cnt, n_ring, v0 + 32 * c) : 0u;
          const int w = wg * (CW / 32) + c;
          is_slow |= (sees[c] & (I8 ? odd[st * NC + w] : odd[st * 2 * NC + w] | odd[st * 2 * NC + NC + w])) != 0;
        }
        // ---- scores times the key scales, and their max
        uint32_t x[CW / 16][16];
#pragma unroll
        for (int c = 0; c < CW / 16; ++c) tmem_ld16(s_now + 16 * c, x[c]);
        tmem_landed();
#pragma unroll
        for (int c = 0; c < CW / 16; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 k = k4[c * 4 + j];
            s[8 * c + 2 * j] = mul2(pk(__uint_as_float(x[c][4 * j]), __uint_as_float(x[c][4 * j + 1])), pk(k.x, k.y));
            s[8 * c + 2 * j + 1] =
                mul2(pk(__uint_as_float(x[c][4 * j + 2]), __uint_as_float(x[c][4 * j + 3])), pk(k.z, k.w));
          }
        if (!all) {
#pragma unroll
          for (int j = 0; j < CW / 2; ++j) {
            const uint32_t w = sees[j >> 4] >> (2 * (j & 15));
            float f0, f1;
            up(s[j], f0, f1);
            s[j] = pk(w & 1 ? f0 : -INFINITY, w & 2 ? f1 : -INFINITY);
          }
        }
#pragma unroll
        for (int j = 0; j < CW / 2; ++j) {
          float f0, f1;
          up(s[j], f0, f1);
          mx = fmaxf(fmaxf(mx, f0), f1);
        }
      }
      if (TPR == 2) mx = fmaxf(mx, meet(i & 1, mx));
      if (ok) {
        const float mn = fmaxf(m, mx * qs), mz = mn == -INFINITY ? 0.f : mn;
        const float corr = ex2(m - mz);
        m = mn;
        // ---- weights: sum, and times the value scale as f16 parts into S's place
        // (16 positions' columns take 8 of high parts, then 8 of remainders)
        f32x2 add = pk(0.f, 0.f);
        const f32x2 qs2 = pk(qs, qs), mz2 = pk(-mz, -mz), minus = pk(-1.f, -1.f);
#pragma unroll
        for (int c = 0; c < CW / 16; ++c) {
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 vv = v4[c * 4 + j];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              float f0, f1, w0, w1;
              up(fma2(s[8 * c + 2 * j + g], qs2, mz2), f0, f1);
              const f32x2 p = pk(ex2(f0), ex2(f1));
              add = add2(add, p);
              const f32x2 w = mul2(p, g ? pk(vv.z, vv.w) : pk(vv.x, vv.y));
              const f32x2 t = w & 0xffffe000ffffe000ull;
              up(t, w0, w1);
              hi[2 * j + g] = cvt2(w0, w1);
              up(fma2(t, minus, w), w0, w1);
              lo[2 * j + g] = cvt2(w0, w1);
            }
          }
          tmem_st8(s_now + c * 16, hi);
          tmem_st8(s_now + c * 16 + 8, lo);
        }
        float a, d;
        up(add, a, d);
        l = l * corr + (a + d);
        // ---- the last step's output (its product ran under the weights), then the new scale
        const int e = expo[2 * st];
        low = expo[2 * st + 1];
        if (i > 0) {
          if (!mbar_wait_spin(o_full, (uint32_t)(i - 1) & 1u, abort, werr)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < OW; c += 32) {
            uint32_t x[2][16];
            tmem_ld16(o_at + lanes + c, x[0]);
            tmem_ld16(o_at + lanes + c + 16, x[1]);
            tmem_landed();
#pragma unroll
            for (int j = 0; j < 32; j += 2)
              o[(c + j) / 2] = add2(o[(c + j) / 2], pk(__uint_as_float(x[j >> 4][j & 15]), __uint_as_float(x[j >> 4][(j & 15) + 1])));
          }
          const float by = corr * (e - e_old > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (e - e_old)) << 23));
          if (__any_sync(0xffffffffu, by != 1.f)) {
#pragma unroll
            for (int d2 = 0; d2 < OW / 2; ++d2) o[d2] = mul2(o[d2], pk(by, by));
          }
        }
        e_old = e;
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(p_full);
    }
    if (nj > 0) {
      float top = 0.f;
      bool faint = false;
      if (ok && !mbar_wait_spin(o_full, (uint32_t)(nj - 1) & 1u, abort, werr)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        // Outputs to their own scale. A row whose output came out infinite or
        // NaN, or far below what the largest value scale holds bits for, is done
        // again.
        const float by = __uint_as_float((uint32_t)(e_old - 13) << 23);
        bool bad = false;
#pragma unroll
        for (int c = 0; c < OW; c += 16) {
          uint32_t x[16];
          tmem_ld16(o_at + lanes + c, x);
          tmem_landed();
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
        is_slow |= bad;
        faint = e_old - low > 12;
      } else {  // a wait gave up: the flag is up, and the rows say so
#pragma unroll
        for (int d = 0; d < OW / 2; ++d) o[d] = pk(__uint_as_float(0x7fc00000u), __uint_as_float(0x7fc00000u));
        l = 1.f, m = 0.f;
        is_slow = false;
      }
      if (TPR == 2) l += meet(nj & 1, l);
      is_slow |= faint && l > 0.f && top < (I8 ? 2.f : 16384.f) * l;
      if (mine && is_slow) atomicOr(&slow[r >> 5], 1u << (r & 31));
      if (TPR == 2) is_slow |= meet(~nj & 1, is_slow ? 1.f : 0.f) != 0.f;
    }
    if (mine && !is_slow) {
      const int d0 = wg * OW;
      if (A.nsplit > 1) {
        float* dst = A.part + ((((size_t)b * A.kvh + kh) * A.nsplit + z) * R + rr) * (A.vh + 2);
#pragma unroll
        for (int d = 0; d < OW; d += 2)
          if (d0 + d < A.vh) *reinterpret_cast<f32x2*>(dst + d0 + d) = o[d / 2];
        if (wg == 0) *reinterpret_cast<float2*>(dst + A.vh) = make_float2(m, l);
      } else {
        float* dst = A.out + (node_at * A.heads + head) * A.vh;
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int d = 0; d < OW; d += 4)  // vh and the start of out are multiples of four floats
          if (d0 + d < A.vh)
            *reinterpret_cast<ulonglong2*>(dst + d0 + d) =
                make_ulonglong2(mul2(o[d / 2], pk(inv, inv)), mul2(o[d / 2 + 1], pk(inv, inv)));
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_PROD));
    const int pw = warp - TPR * 4;
    if (pw == 3) {
      // ---------------------------------------------------------- MMA issue
      const uint64_t dq_hi = sw128_desc(qhi), dq_lo = sw128_desc(qlo), d_stage = sw128_desc(stages);
      auto issue_qk = [&](int i) {  // S of step i
        const int st = i % NST;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t dk = d_stage + (uint64_t)(st * (C::STAGE >> 4));
          const uint32_t d = tmem + (i & 1) * BN;
          uint32_t acc = 0;
          auto steps = [&](uint64_t dq, uint64_t dkk) {
#pragma unroll
            for (int k = 0; k < QS; ++k) {
              mma_ss<BN>(d, dq + (uint64_t)((k >> 2) * (128 * 128 >> 4) + (k & 3) * 2),
                         dkk + (uint64_t)((k >> 2) * (BN * 128 >> 4) + (k & 3) * 2), acc);
              acc = 1;
            }
          };
          steps(dq_lo, dk);
          if (!I8) steps(dq_hi, dk + (uint64_t)(C::K_TILE >> 4));
          steps(dq_hi, dk);
          umma_commit(&s_full[i & 1]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int i) {  // O of step i
        const int st = i % NST;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t dv = d_stage + (uint64_t)((st * C::STAGE + C::PARTS * C::K_TILE) >> 4);
          const uint32_t p = tmem + (i & 1) * BN;
          uint32_t acc = 0;
          auto steps = [&](uint32_t a, uint64_t dvv) {
#pragma unroll
            for (int k = 0; k < BN / 16; ++k) {
              mma_ts<VP>(tmem + 2 * BN, a + k * 16, dvv + (uint64_t)(k * 2), acc);
              acc = 1;
            }
          };
          steps(p + 8, dv);
          if (!I8) steps(p, dv + (uint64_t)(C::V_TILE >> 4));
          steps(p, dv);
          umma_commit(o_full);
          umma_commit(&empty[st]);
        }
        __syncwarp();
      };
      // The scores of the first two steps, then after each second product scores
      // again: they take the place of that step's weights, so the product must be
      // done.
      auto scores = [&](int q) {
        bool ready = mbar_wait_spin(&full[q % NST], (uint32_t)(q / NST) & 1u, abort, werr);
        if (ready && q >= 2) ready = mbar_wait_spin(o_full, (uint32_t)q & 1u, abort, werr);
        ready = __all_sync(0xffffffffu, ready);
        if (ready) issue_qk(q);
        return ready;
      };
      bool ok = nblk == 0 || mbar_wait_spin(q_full, 0, abort, werr);
      ok = __all_sync(0xffffffffu, ok);
      for (int q = 0; q < 2 && q < nblk && ok; ++q) ok = scores(q);
      for (int i = 0; i < nblk && ok; ++i) {
        ok = mbar_wait_spin(p_full, (uint32_t)i & 1u, abort, werr);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) issue_pv(i);
        if (ok && i + 2 < nblk) ok = scores(i + 2);
      }
      // Every issued MMA completes before TMEM is freed.
      if (elect_one()) umma_commit(drain);
      __syncwarp();
      mbar_drain(drain, 0);
    } else if (pw == 0 || (!I8 && pw == 5)) {
      // ---------------------------------------------------------- keys and scales
      bool ok = true;
      int e = 14, low = 255;
      // int8: positions lane and lane + 32 of a step and their scales; the next
      // step's are on their way while one is widened.
      uint4 kn[2][QS];
      float ksn[2], vsn[2];
      auto load = [&](int i) {
        const int v0 = (blk0 + i) * BN;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int v = v0 + h * 32 + lane;
          const bool in = v < P.total, d = P.in_draft(v);
          const size_t row = in ? P.row(v) : 0;
          ksn[h] = in ? __ldg((d ? A.tks : A.ks) + row) : 0.f;
          vsn[h] = in ? __ldg((d ? A.tvs : A.vs) + row) : 0.f;
          const uint4* src = reinterpret_cast<const uint4*>((d ? A.tk : A.k) + row * A.qk);
#pragma unroll
          for (int c = 0; c < QS; ++c) kn[h][c] = in && c * 16 < A.qk ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
        }
      };
      // f32: LK lanes a key, 32 / LK keys at a time.
      constexpr int LK = 2 * C::KA, DL = QS * 16 / LK;
      const int kw = pw == 0 ? 0 : 1;
      float4 fn[DL / 4];
      auto fetch = [&](int i, int u) {
        const int v = (blk0 + i) * BN + kw * 32 + u * (32 / LK) + lane / LK, d0 = lane % LK * DL;
        const bool in = v < P.total;
        const float4* src = reinterpret_cast<const float4*>(
            reinterpret_cast<const float*>(P.in_draft(v) ? A.tk : A.k) + (in ? P.row(v) : 0) * A.qk);
#pragma unroll
        for (int c = 0; c < DL / 4; ++c)
          fn[c] = in && d0 + c * 4 < A.qk ? __ldg(src + d0 / 4 + c) : make_float4(0, 0, 0, 0);
      };
      if (nblk > 0) {
        if (I8) load(0);
        else fetch(0, 0);
      }
      for (int i = 0; i < nblk; ++i) {
        const int st = i % NST, v0 = (blk0 + i) * BN;
        unsigned char* kt = stages + (size_t)st * C::STAGE;
        float ksc[2], vsc[2];
        bool sane[2];
        if (I8) {
          if (ok && !mbar_wait_spin(&empty[st], ((uint32_t)(i / NST) & 1u) ^ 1u, abort, werr)) ok = false;
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int kp = h * 32 + lane;
            ksc[h] = ksn[h], vsc[h] = vsn[h];
            uint4 kk[QS];
#pragma unroll
            for (int c = 0; c < QS; ++c) kk[c] = kn[h][c];
            if (h == 1 && i + 1 < nblk) load(i + 1);
#pragma unroll
            for (int c = 0; c < QS; ++c) {
              uint32_t w[8];
              widen(kk[c].x ^ 0x80808080u, &w[0], &w[1]);
              widen(kk[c].y ^ 0x80808080u, &w[2], &w[3]);
              widen(kk[c].z ^ 0x80808080u, &w[4], &w[5]);
              widen(kk[c].w ^ 0x80808080u, &w[6], &w[7]);
              unsigned char* row = kt + (c >> 2) * (BN * 128) + kp * 128;
              *reinterpret_cast<uint4*>(row + ((((c & 3) * 2) ^ (kp & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(row + ((((c & 3) * 2 + 1) ^ (kp & 7)) << 4)) =
                  make_uint4(w[4], w[5], w[6], w[7]);
            }
            sane[h] = fabsf(ksc[h]) <= KEY_SCALE_FAR && fabsf(vsc[h]) <= 3.4028234e38f;
          }
          // Value scales, held so that the largest so far is in [2^13, 2^14).
          uint32_t top = 0, least = 0x7f800000u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!sane[h]) vsc[h] = 0.f;
            const uint32_t a = __float_as_uint(fabsf(vsc[h]));
            top = max(top, a), least = min(least, a ? a : 0x7f800000u);
          }
          e = min(max(e, (int)(__reduce_max_sync(0xffffffffu, top) >> 23)), 253);
          low = min(low, (int)(__reduce_min_sync(0xffffffffu, least) >> 23));
          const float f = __uint_as_float((uint32_t)(267 - e) << 23);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            col_k[st * BN + h * 32 + lane] = ksc[h];
            col_v[st * BN + h * 32 + lane] = vsc[h] * f;
            const uint32_t w = __ballot_sync(0xffffffffu, !sane[h]);
            if (lane == 0) odd[st * NC + h] = w;
          }
          if (lane == 0) expo[2 * st] = e, expo[2 * st + 1] = low;
        } else {
          // f32: each key scaled by the power of two that brings its largest
          // element into [2^13, 2^14); the values' scales are the value warps'
          // matter. A warp has 32 positions, DL elements a lane; the next keys are
          // on their way while some are converted.
          uint32_t outs = 0;
#pragma unroll
          for (int u = 0; u < LK; ++u) {
            const int kp = kw * 32 + u * (32 / LK) + lane / LK;
            float4 x[DL / 4];
#pragma unroll
            for (int c = 0; c < DL / 4; ++c) x[c] = fn[c];
            if (u + 1 < LK) fetch(i, u + 1);
            else if (i + 1 < nblk) fetch(i + 1, 0);
            float mx = 0.f, t = 0.f;  // t: NaN where one is
#pragma unroll
            for (int c = 0; c < DL / 4; ++c) {
              mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[c].x), fabsf(x[c].y)), fmaxf(fabsf(x[c].z), fabsf(x[c].w))));
              t += fabsf(x[c].x) + fabsf(x[c].y) + fabsf(x[c].z) + fabsf(x[c].w);
            }
            if (t != t) mx = INFINITY;
#pragma unroll
            for (int d = 1; d < LK; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const int ef = min(max((int)(__float_as_uint(mx) >> 23), 14), 253);
            const float by = __uint_as_float((uint32_t)(267 - ef) << 23);
            if (u == 0) {
              if (ok && !mbar_wait_spin(&empty[st], ((uint32_t)(i / NST) & 1u) ^ 1u, abort, werr)) ok = false;
              __syncwarp();
            }
#pragma unroll
            for (int c = 0; c < DL / 8; ++c) {
              uint32_t hh[4], ll[4];
              halves(x[2 * c].x * by, x[2 * c].y * by, &hh[0], &ll[0]);
              halves(x[2 * c].z * by, x[2 * c].w * by, &hh[1], &ll[1]);
              halves(x[2 * c + 1].x * by, x[2 * c + 1].y * by, &hh[2], &ll[2]);
              halves(x[2 * c + 1].z * by, x[2 * c + 1].w * by, &hh[3], &ll[3]);
              const int ch = lane % LK * (DL / 8) + c;
              unsigned char* at = kt + (ch >> 3) * (BN * 128) + kp * 128 + (((ch & 7) ^ (kp & 7)) << 4);
              *reinterpret_cast<uint4*>(at) = make_uint4(hh[0], hh[1], hh[2], hh[3]);
              *reinterpret_cast<uint4*>(at + C::K_TILE) = make_uint4(ll[0], ll[1], ll[2], ll[3]);
            }
            if (lane % LK == 0) col_k[st * BN + kp] = v0 + kp < P.total ? __uint_as_float((uint32_t)(ef - 13) << 23) : 0.f;
            if (!(mx <= KEY_SCALE_FAR)) outs |= 1u << (kp & 31);  // the scale is 2^13 to 2^14 times less, a product up to 2^35
          }
          outs = __reduce_or_sync(0xffffffffu, outs);
          if (lane == 0) odd[st * 2 * NC + kw] = outs;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&full[st]);
      }
    } else if (pw != 4) {
      // ---------------------------------------------------------- values
      const int vw = pw < 3 ? pw - 1 : pw - 4;
      bool ok = true;
      int e = 14, low = 255;
      // int8: eight positions (an octet) by VP / 8 dims a thread: a warp reads
      // whole sectors and writes one 16-byte chunk of eight positions per dim, its
      // lanes in different chunks. The next step's values are on their way while
      // one is widened.
      constexpr int DV = VP / 8;
      const int d0 = (vw * 4 + (lane >> 3)) * DV;
      uint32_t xn[8][DV / 4];
      auto get = [&](const char* src, bool in, uint32_t (&x)[DV / 4]) {
        if (DV == 8) {
          const uint2 t = in ? __ldg(reinterpret_cast<const uint2*>(src)) : make_uint2(0, 0);
          x[0] = t.x, x[1] = t.y;
        } else {
          const uint4 t = in ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
          x[0] = t.x, x[1] = t.y, x[DV / 4 - 2] = t.z, x[DV / 4 - 1] = t.w;
        }
      };
      auto load = [&](int i) {
        const int v = (blk0 + i) * BN + (lane & 7) * 8;
        if (P.plain((blk0 + i) * BN, BN)) {  // the same for the warp
          const char* src = A.v + P.row(v) * A.vh + d0;
          const size_t step = (size_t)A.kvh * A.vh;
#pragma unroll
          for (int j = 0; j < 8; ++j) get(src + j * step, d0 < A.vh, xn[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool in = v + j < P.total && d0 < A.vh;
            get((P.in_draft(v + j) ? A.tv : A.v) + (in ? P.row(v + j) : 0) * A.vh + (in ? d0 : 0), in, xn[j]);
          }
        }
      };
      // f32: VP / 4 lanes an octet, OCT octets at a time.
      constexpr int OCT = 128 / VP, PASS = 2 / OCT;
      float4 fn[8];
      auto fetch = [&](int i, int p) {
        const int v = (blk0 + i) * BN + (vw * 2 + p * OCT + lane % OCT) * 8, d = lane / OCT * 4;
        if (P.plain((blk0 + i) * BN, BN)) {  // the same for the warp
          const float* src = reinterpret_cast<const float*>(A.v) + P.row(v) * A.vh + d;
          const size_t step = (size_t)A.kvh * A.vh;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            fn[j] = d < A.vh ? __ldg(reinterpret_cast<const float4*>(src + j * step)) : make_float4(0, 0, 0, 0);
          return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = v + j < P.total && d < A.vh;
          const float* row =
              reinterpret_cast<const float*>(P.in_draft(v + j) ? A.tv : A.v) + (in ? P.row(v + j) : 0) * A.vh + (in ? d : 0);
          fn[j] = in ? __ldg(reinterpret_cast<const float4*>(row)) : make_float4(0, 0, 0, 0);
        }
      };
      if (nblk > 0) {
        if (I8) load(0);
        else if (PASS == 1) fetch(0, 0);
      }
      for (int i = 0; i < nblk; ++i) {
        const int st = i % NST;
        unsigned char* vt = stages + (size_t)st * C::STAGE + C::PARTS * C::K_TILE;
        if (I8) {
          const int pr = lane & 7;
          uint32_t x[8][DV / 4];
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int q = 0; q < DV / 4; ++q) x[j][q] = xn[j][q];
          if (i + 1 < nblk) load(i + 1);
          if (ok && !mbar_wait_spin(&empty[st], ((uint32_t)(i / NST) & 1u) ^ 1u, abort, werr)) ok = false;
          __syncwarp();
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
                *reinterpret_cast<uint4*>(vt + d * 128 + ((pr ^ (d & 7)) << 4)) =
                    make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]);
              }
            }
          }
        } else {
          // f32: a warp holds 16 positions (two octets; of 128-wide values one at a
          // time) whole, four dims a lane, so a position's largest value is the
          // warp's own matter. A value is scaled like a key; 2^(140 - e) is a step's
          // share of the scale, by the largest exponent of the warps so far. Lanes
          // take their four dims in an order that keeps their writes in different
          // banks.
          const int da = lane / OCT * 4, turn = OCT == 2 ? lane >> 1 & 2 : lane >> 1 & 3;
          int top = 0, least = 255, own[2] = {0, 0};
          uint32_t bad = 0;
          int* seen = vmax + (i & 1) * 8;
#pragma unroll
          for (int p = 0; p < PASS; ++p) {
            const int pr = vw * 2 + p * OCT + lane % OCT;
            float4 x[8];
            if (PASS == 2) fetch(i, p);  // without registers to hold two
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = fn[j];
            if (PASS == 1 && i + 1 < nblk) fetch(i + 1, 0);
            // The octet's eight maxima, one left a lane: position lane / 4.
            float a[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float t = fabsf(x[j].x) + fabsf(x[j].y) + fabsf(x[j].z) + fabsf(x[j].w);  // NaN where one is
              a[j] = fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w)));
              a[j] = t == t ? a[j] : INFINITY;
            }
#pragma unroll
            for (int h = 4; h >= 1; h >>= 1) {
              const bool up = lane & 4 * h;
#pragma unroll
              for (int j = 0; j < h; ++j) {
                const float send = up ? a[j] : a[j + h], keep = up ? a[j + h] : a[j];
                a[j] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, 4 * h));
              }
            }
#pragma unroll
            for (int d = OCT; d < 4; d <<= 1) a[0] = fmaxf(a[0], __shfl_xor_sync(0xffffffffu, a[0], d));
            // Its exponent field: 0 none, 255 not finite.
            const int eb = (int)(__float_as_uint(a[0]) >> 23);
            const int y = a[0] == 0.f ? 0 : eb == 255 ? 255 : min(max(eb, 14), 253);
            if (p == 0) own[0] = y;
            else own[1] = y;
            if (y == 255) bad |= 1u << (8 * (pr & 1) + (lane >> 2));
            if (y != 0 && y != 255) top = max(top, y - 13), least = min(least, y - 13);
            if (p + 1 == PASS) {
              top = __reduce_max_sync(0xffffffffu, top), least = __reduce_min_sync(0xffffffffu, least);
              if (lane == 0) seen[vw] = top, seen[4 + vw] = least;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int yj = __shfl_sync(0xffffffffu, y, 4 * j + lane % OCT);
              const bool use = yj != 0 && yj != 255;  // nothing of one that is not finite
              const float by = __uint_as_float((uint32_t)(267 - yj) << 23);
              x[j] = use ? make_float4(x[j].x * by, x[j].y * by, x[j].z * by, x[j].w * by) : make_float4(0, 0, 0, 0);
              if (OCT == 1 && turn & 1) x[j] = make_float4(x[j].y, x[j].z, x[j].w, x[j].x);
              if (turn & 2) x[j] = make_float4(x[j].z, x[j].w, x[j].x, x[j].y);
            }
            if (p == 0) {
              if (ok && !mbar_wait_spin(&empty[st], ((uint32_t)(i / NST) & 1u) ^ 1u, abort, werr)) ok = false;
              __syncwarp();
            }
            if (da < A.vh) {
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                uint32_t hh[4], ll[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float4 a = x[2 * j], c = x[2 * j + 1];
                  halves(t == 0 ? a.x : t == 1 ? a.y : t == 2 ? a.z : a.w, t == 0 ? c.x : t == 1 ? c.y : t == 2 ? c.z : c.w,
                         &hh[j], &ll[j]);
                }
                const int d = da + ((t + turn) & 3);
                unsigned char* to = vt + d * 128 + ((pr ^ (d & 7)) << 4);
                *reinterpret_cast<uint4*>(to) = make_uint4(hh[0], hh[1], hh[2], hh[3]);
                *reinterpret_cast<uint4*>(to + C::V_TILE) = make_uint4(ll[0], ll[1], ll[2], ll[3]);
              }
            }
          }
          bad = __reduce_or_sync(0xffffffffu, bad);
          asm volatile("bar.sync 4, 128;" ::: "memory");
          e = max(max(e, max(seen[0], seen[1])), max(seen[2], seen[3]));
          low = min(min(low, min(seen[4], seen[5])), min(seen[6], seen[7]));
          if (lane == 0) reinterpret_cast<uint16_t*>(odd + st * 2 * NC + NC)[vw] = (uint16_t)bad;
          if (vw == 0 && lane == 0) expo[2 * st] = e, expo[2 * st + 1] = low;
          if ((lane & 3) < OCT) {
#pragma unroll
            for (int p = 0; p < PASS; ++p) {
              const int y = own[p], f = 127 + y - e;  // 2^(y - 140) 2^(140 - e)
              col_v[st * BN + (vw * 2 + p * OCT + lane % OCT) * 8 + (lane >> 2)] =
                  y != 0 && y != 255 && f > 0 ? __uint_as_float((uint32_t)f << 23) : 0.f;
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&full[st]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TMEM));
  }
  // ---- rows to do again, a warp each: the softmax warps, whose register share is
  // no smaller than the launch's (the others gave theirs up, and code past the
  // roles need not keep to what they have left)
  for (int wd = 0; wd < 4; ++wd) {
    uint32_t todo = slow[wd];
    int turn = 0;
    while (todo) {
      const int r2 = wd * 32 + __ffs(todo) - 1;
      todo &= todo - 1;
      if (turn++ % (TPR * 4) != warp) continue;
      const int q2 = r0 + r2, n2 = A.by_rep.div(q2), h2 = kh * A.rep + q2 - n2 * A.rep;
      const size_t at2 = (size_t)b * A.T + n2;
      const int hh = A.hi[at2];
      int ll = max(A.lo[at2], 0);
      if (hh >= 0) ll = max(ll, hh - A.slots + 1);
      const int c2 = ll <= hh ? hh - ll + 1 : 0, s2 = c2 ? (int)((long)(ll - base) % A.slots) : 0;
      float m2 = -INFINITY, l2 = 0.f, o2[4] = {0.f, 0.f, 0.f, 0.f};
      tree_slow_call<I8>(A, P, at2, n2, h2, s2, c2, n_ring, blk0 * BN, min((blk0 + nblk) * BN, P.total), &m2, &l2, o2);
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
  cudaError_t e = allow_smem((const void*)kern, C::SMEM, true);
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

typedef TreeUmma<true, 3, 64, 1, 4> UmmaI8x48;
typedef TreeUmma<true, 4, 64, 1, 4> UmmaI8x64;
typedef TreeUmma<true, 8, 128, 2, 4> UmmaI8x128;
typedef TreeUmma<false, 3, 64, 2, 5> UmmaF32x48;
typedef TreeUmma<false, 4, 64, 2, 5> UmmaF32x64;
typedef TreeUmma<false, 8, 128, 2, 2> UmmaF32x128;

}  // namespace

// More than 16 rows, whole 16-byte pieces and MMA steps. A step costs nearly the
// same for 17 rows as for 128; mma.sync pays per 16 rows. Measured, mma.sync -> here:
//   rows   48/64 int8, 256 x 1043   48/64 f32, 128 x 1043   128 int8, 4 x 16000   128 f32, 32 x 1043
//     6        49 ->  62 us              64 ->  68 us            83 -> 114 us         225 -> 186 us
//    12        53 ->  62                 66 ->  69               88 -> 115            231 -> 186
//    24        72 ->  63                 84 ->  69              155 -> 116            438 -> 187
//    48       136 ->  74                156 ->  72              270 -> 119            646 -> 190
//    96       205 ->  78                228 ->  76              527 -> 124           1193 -> 194
// and at eight sessions of 1043 (48/64 int8) 6 rows 12.6 -> 16.8, 12: 15.4 -> 16.7, 24:
// 22.1 -> 17.1. One bound for all forms: of 128-wide f32 heads it lies too high, and up
// to 16 rows there take the slower form.
bool tree_umma_takes(int int8, int rows, int qk, int vh, int piece) {
  return piece == 16 && qk % 16 == 0 && vh % 16 == 0 && rows > 16;
}

// The cheapest number of position splits, in us: what a step of 64 positions
// costs a block that has its SM to itself, or (int8 heads up to 64 wide) shares
// it with another; a block's start and end, more where it leaves partial results;
// their join. Measured (splits: us):
//   int8 48/64: 256 x 96 rows x 1043    1: 78    2: 132   4: 160
//               1 x 384 rows x 6000     1: 118   8: 30   16: 25   24: 24  32: 29  48: 31
//   int8 128:   4 x 128 rows x 32771    1: 812   4: 230   9: 223  16: 268
//               20 x 64 rows x 1043     1: 69    2: 83    4: 100
//   f32 48/64:  16 x 288 rows x 2051    1: 66    2: 77    3: 67    6: 84
//   f32 128:    2 x 128 rows x 8000     1: 511   4: 158   8: 105   9: 105  16: 119
int tree_umma_nsplit(int int8, int B, int rows, int kvh, int qk, int vh, int span) {
  const bool wide = qk > 64 || vh > 64, two = int8 && !wide;
  const double one = int8 ? (wide ? 1.6 : 1.2) : (wide ? 3.8 : 1.9), both = two ? 2.1 : one;
  const long work = (long)B * kvh * ((rows + 127) / 128), room = 148 * (two ? 2 : 1);
  const int blocks = (span + 63) / 64;
  int best = 1;
  double cost = 1e300;
  for (int ns = 1; ns <= 128 && ns <= blocks; ++ns) {
    const long rest = work * ns % room;
    const double step = (blocks + ns - 1) / ns, ends = ns > 1 ? 13 : 6;
    const double c = (double)(work * ns / room) * (both * step + ends) +
                     (rest == 0 ? 0.0 : (rest <= 148 ? one : both) * step + ends) +
                     (ns > 1 ? 3 + 1.9 * ((ns + 7) / 8) : 0.0);
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
  if (A.qk > 64 || A.vh > 64) return launch_umma_form<UmmaF32x128>(A, B, st);
  if (A.qk > 48) return launch_umma_form<UmmaF32x64>(A, B, st);
  return launch_umma_form<UmmaF32x48>(A, B, st);
}

}  // namespace nb
