// Attention of drafted nodes over a KV ring and their own ancestors:
// nd_attend_tree. T nodes of a session (a tree, a chain, or one token) are the
// queries; node t sees the ring positions lo..hi of its own and the drafted
// nodes its mask names, whose keys and values lie in a second buffer of the
// ring's form. nd_attend_step is the case of one query and no draft.
//
//   s_j = (q . k_j) / sqrt(qk),  m = max s,  out = sum exp(s_j - m) v_j / sum exp(s_j - m)
//
// over the seen positions j, in one pass with a running max and sum; a node
// that sees nothing gets zeros.
//
// The rows of one KV head are its T * rep (node, query head) pairs. Products
// run on mma.sync with rows as the 16 and positions as the 8: int8 codes are
// f16 values exactly, the query and the softmax weights go in as an f16 high
// part and remainder (22 bits); f32 rings as three TF32 products of high parts
// and remainders. Sums, max and the outputs are f32. The tensor cores truncate as
// they accumulate, always towards zero: so a block's products start from zero,
// remainders first, and are added to the running outputs (and long dot products
// chunk by chunk) in f32. Left in the accumulators over 5651 positions the bias
// was 8e-7 to 1.5e-6 of the result against 3.4e-7 of the plain 32-bit form. Eight
// sessions' single token over 512 positions take 10.4 us (f32 14.5; nd_attend_step 20.5
// and 22.7), with a draft of one node 12.3: latency, 64 blocks of a short chain. 256
// sessions over 1043 positions take 47 (f32 121; nd_attend_step 66 and 206).
#include <cooperative_groups.h>

#include <algorithm>

#include "kernels.hpp"
#include "launch_util.hpp"
#include "tree.cuh"

namespace nb {
namespace {

// Value dimension of column `col` (0..7) of output tile n: int8 tiles come in
// pairs holding the even and odd dimensions of 16 (the order ldmatrix.trans
// gives byte pairs in), f32 tiles are 8 dimensions in order.
template <bool I8>
__device__ __forceinline__ int tree_dim(int n, int col) {
  return I8 ? (n >> 1) * 16 + 2 * col + (n & 1) : n * 8 + col;
}

constexpr int TREE_CLUSTER = 8;  // blocks of a portable cluster
constexpr int TREE_WARPS = 4;
constexpr int TREE_THREADS = TREE_WARPS * 32;

__device__ __forceinline__ void mma_h(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_t(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void add4(float (&d)[4], const float (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] += x[i];
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"((unsigned)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"((unsigned)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// (x, y) as f16 pairs of high parts and remainders.
__device__ __forceinline__ void split2(float x, float y, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  *lo = h2(x - f.x, y - f.y);
}
// x as a TF32 high part (rounded) and its remainder.
__device__ __forceinline__ void split_t(float x, uint32_t* hi, uint32_t* lo) {
  uint32_t h;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(h) : "f"(x));
  *hi = h;
  *lo = __float_as_uint(x - __uint_as_float(h));
}
// Four codes (one register of ring bytes) as f16 pairs (0, 1) and (2, 3), or
// with SEL two positions' pairs (0, 2) and (1, 3): the byte with its sign bit
// flipped is the low mantissa of 1024 + byte, less 1152.
template <uint32_t S0, uint32_t S1>
__device__ __forceinline__ void codes_h2(uint32_t u, uint32_t* a, uint32_t* b) {
  u ^= 0x80808080u;
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  uint32_t p = __byte_perm(u, 0x64646464u, S0), r = __byte_perm(u, 0x64646464u, S1);
  __half2 x = __hsub2(*reinterpret_cast<__half2*>(&p), bias), y = __hsub2(*reinterpret_cast<__half2*>(&r), bias);
  *a = *reinterpret_cast<uint32_t*>(&x);
  *b = *reinterpret_cast<uint32_t*>(&y);
}

// Shared memory of one warp: NB buffers of PB positions. Row strides keep the
// fragment loads free of bank conflicts: int8 rows an odd number of 16-byte
// pieces apart; f32 key rows 16 words past a multiple of 32, value rows 4 past
// a multiple of 16.
template <bool I8, int QKP, int VHP>
struct TreeTile {
  static constexpr int ES = I8 ? 1 : 4;
  static constexpr int PB = I8 ? 32 : 16;
  static constexpr int NB = 2;
  static constexpr int KS = QKP == 48 ? 48 : QKP + 16;  // elements
  static constexpr int VS = I8 ? VHP + 16 : VHP + 4;
  static constexpr int K_BYTES = PB * KS * ES, V_BYTES = PB * VS * ES;
  static constexpr int BUF = K_BYTES + V_BYTES + (I8 ? PB * 8 : 0);
  static constexpr int WARP_BYTES = NB * BUF;
};

// One warp's copy of PB positions into a buffer: offsets o0.. of the ring
// (`count` of them in use; ring slot = first slot + offset, wrapped) or nodes
// o0.. of the draft. Positions past the end are filled with zeros, so that
// whatever lies there never reaches a product.
template <class TT, bool I8, int PIECE>
__device__ __forceinline__ void tree_copy(char* buf, const char* k, const char* v, const float* ks, const float* vs,
                                          int kvh, int kh, int qk, int vh, int o0, int count, int slot0, int slots,
                                          int lane) {
  constexpr int ES = TT::ES;
  const int kp = qk * ES / PIECE, vp = vh * ES / PIECE;
  auto slot_of = [&](int i) {  // o0 + i < count <= slots: wraps at most once
    const int s = slot0 + o0 + i;
    return s >= slots ? s - slots : s;
  };
  auto rows = [&](char* dst, const char* src, int pieces, int dim, int stride) {
    for (int j = lane; j < TT::PB * pieces; j += 32) {
      const int i = j / pieces, pc = j - i * pieces;
      const bool ok = o0 + i < count;
      const char* g = src + ((size_t)(ok ? slot_of(i) : 0) * kvh + kh) * dim * ES + pc * PIECE;
      char* s = dst + i * stride * ES + pc * PIECE;
      if (PIECE == 16) cp_async16(s, g, ok);
      else cp_async4(s, g, ok);
    }
  };
  rows(buf, k, kp, qk, TT::KS);
  rows(buf + TT::K_BYTES, v, vp, vh, TT::VS);
  if (I8) {
    float* sc = reinterpret_cast<float*>(buf + TT::K_BYTES + TT::V_BYTES);
    for (int i = lane; i < TT::PB; i += 32) {
      const bool ok = o0 + i < count;
      const size_t at = (size_t)(ok ? slot_of(i) : 0) * kvh + kh;
      cp_async4(sc + i, ks + at, ok);
      cp_async4(sc + TT::PB + i, vs + at, ok);
    }
  }
}

// A warp's rows again, over its own blocks of PB positions and in plain f32: those
// of the TILE rows of `mine` (row stride PW: outputs, then max and sum at AT) whose
// sum is no number or, with `far`, that see a key scale above KEY_SCALE_FAR.
// Everything is worked out afresh, so that the kernel keeps no register for it
// (with the ranges handed over the 128-wide forms were 5 to 7 % slower than without
// this call; as it is, f32 ones are 3 %: 32 x 1043 with 6 rows 218 -> 225 us, int8
// 50.1 -> 49.9).
template <bool I8, int TILE, int PB, int PW, int AT>
__device__ __noinline__ void tree_again(const TreeArgs& A, float* mine, bool far) {
  const int b = blockIdx.y, wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int z = blockIdx.x % A.nsplit, kh = blockIdx.x / A.nsplit % A.kvh, tile = blockIdx.x / A.nsplit / A.kvh;
  const int R = A.T * A.rep, r0 = tile * TILE, rows = min(TILE, R - r0);
  int first = 0x7fffffff, last = -1;
  for (int n = A.by_rep.div(r0) + lane; n <= A.by_rep.div(r0 + rows - 1); n += 32) {
    const int h = A.hi[(size_t)b * A.T + n];
    int l = max(A.lo[(size_t)b * A.T + n], 0);
    if (h >= 0) l = max(l, h - A.slots + 1);
    if (l <= h) first = min(first, l), last = max(last, h);
  }
  first = __reduce_min_sync(0xffffffffu, first), last = __reduce_max_sync(0xffffffffu, last);
  const int base = last >= 0 ? first : 0, n_ring = last >= 0 ? (int)min((long)last - base + 1, (long)A.slots) : 0;
  const int ring_blocks = (n_ring + PB - 1) / PB, blocks = ring_blocks + (A.drafted + PB - 1) / PB;
  const int blk0 = (int)((long)blocks * z / A.nsplit) + wid, blk1 = (int)((long)blocks * (z + 1) / A.nsplit);
  TreePlace P;
  P.ring = (size_t)b * A.slots * A.kvh + kh, P.draft = (size_t)b * A.T * A.kvh + kh;
  P.drafted = A.drafted, P.slot0 = base % A.slots, P.slots = A.slots, P.kvh = A.kvh, P.total = A.drafted + n_ring;
  for (int r = 0; r < rows; ++r) {
    float* row = mine + (size_t)r * PW;
    const bool number = row[AT + 1] <= 3.4028234e38f;
    if (!far && number) continue;
    const int rr = r0 + r, node = A.by_rep.div(rr), head = kh * A.rep + rr - node * A.rep;
    const size_t node_at = (size_t)b * A.T + node;
    const float* q = A.q + node_at * A.ldq + (size_t)head * A.qk;
    bool none = false;
    for (int i = lane; i < A.qk; i += 32) none |= q[i] != q[i];
    if (__any_sync(0xffffffffu, none)) continue;  // a NaN in the query: NaN it stays
    const int h = A.hi[node_at];
    int l = max(A.lo[node_at], 0);
    if (h >= 0) l = max(l, h - A.slots + 1);
    const int cnt = l <= h ? h - l + 1 : 0, start = cnt ? (int)((long)(l - base) % A.slots) : 0;
    if (number) {  // whether the row sees one of the scales at all
      bool sees = false;
      for (int blk = blk0; blk < blk1; blk += TREE_WARPS) {
        const int v0 = blk < ring_blocks ? P.drafted + blk * PB : (blk - ring_blocks) * PB;
        const int v1 = min(v0 + PB, blk < ring_blocks ? P.total : P.drafted);
        for (int at = v0 & ~31; at < v1; at += 32) {
          const int v = at + lane;
          if (v >= v0 && v < v1 && ((tree_sees(A, node_at, node, start, cnt, n_ring, at) >> lane) & 1))
            sees |= fabsf((P.in_draft(v) ? A.tks : A.ks)[P.row(v)]) > KEY_SCALE_FAR;
        }
      }
      if (!__any_sync(0xffffffffu, sees)) continue;
    }
    float m = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int blk = blk0; blk < blk1; blk += TREE_WARPS) {
      const int v0 = blk < ring_blocks ? P.drafted + blk * PB : (blk - ring_blocks) * PB;
      tree_slow_row<I8>(A, P, node_at, node, head, start, cnt, n_ring, v0,
                        min(v0 + PB, blk < ring_blocks ? P.total : P.drafted), &m, &sum, o);
    }
    __syncwarp();  // the row's sum has been read
    for (int j = 0; j < 4; ++j)
      if (lane + 32 * j < A.vh) row[lane + 32 * j] = o[j];
    if (lane == 0) row[AT] = m, row[AT + 1] = sum;
  }
}

// Grid (row tiles * kvh * nsplit, B), four warps: each holds the same MT * 16
// rows (queries in registers) and takes every fourth block of PB positions of
// its split through its own double-buffered copies, so the loop has no block
// barrier; the warps' maxima, sums and outputs meet at the end. Positions are
// the ring's (offsets 0 .. n_ring - 1 from the tile's lowest position) and
// then the draft's nodes.
template <bool I8, int QKP, int VHP, int MT>
__global__ void __launch_bounds__(TREE_THREADS) attend_tree_kernel(const __grid_constant__ TreeArgs A, int piece,
                                                                   int cluster) {
  using TT = TreeTile<I8, QKP, VHP>;
  constexpr int PB = TT::PB, NT = PB / 8;        // 8-position score tiles of a block
  constexpr int KC = QKP / 16, VN = VHP / 8;     // 16-dim chunks of a key, 8-dim tiles of an output
  extern __shared__ __align__(16) char smem[];
  __shared__ int range[3];  // lowest and highest seen position; int8: whether a score may have passed the range
  const int b = blockIdx.y;
  int bx = blockIdx.x;
  const int z = bx % A.nsplit;
  bx /= A.nsplit;
  const int kh = bx % A.kvh, tile = bx / A.kvh;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
  const int R = A.T * A.rep, r0 = tile * MT * 16, rows = min(MT * 16, R - r0);
  const int n0 = A.by_rep.div(r0), n1 = A.by_rep.div(r0 + rows - 1);  // first and last node of the tile

  // Ring range of the tile. Each node's lo is held within one turn of the ring.
  if (tid == 0) range[0] = 0x7fffffff, range[1] = -1, range[2] = 0;
  __syncthreads();
  for (int n = n0 + tid; n <= n1; n += TREE_THREADS) {
    const int h = A.hi[(size_t)b * A.T + n];
    int l = max(A.lo[(size_t)b * A.T + n], 0);
    if (h >= 0) l = max(l, h - A.slots + 1);
    if (l <= h) {
      atomicMin(&range[0], l);
      atomicMax(&range[1], h);
    }
  }
  __syncthreads();
  const int base = range[1] >= 0 ? range[0] : 0;
  const int n_ring = range[1] >= 0 ? (int)min((long)range[1] - base + 1, (long)A.slots) : 0;
  const int slot0 = base % A.slots;

  // This lane's rows g and g + 8 of every 16: the node's visible offsets
  // [start, start + cnt) modulo the ring, its index, and the full span common
  // to all of this warp's rows.
  int start[2 * MT], cnt[2 * MT], node[2 * MT];
  int full0 = 0, full1 = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    const int r = (i >> 1) * 16 + (i & 1) * 8 + g;
    node[i] = A.by_rep.div(r0 + min(r, rows - 1));
    const int h = A.hi[(size_t)b * A.T + node[i]];
    int l = max(A.lo[(size_t)b * A.T + node[i]], 0);
    if (h >= 0) l = max(l, h - A.slots + 1);
    cnt[i] = l <= h ? h - l + 1 : 0;
    start[i] = cnt[i] ? (int)((long)(l - base) % A.slots) : 0;
    full0 = max(full0, start[i]);
    full1 = min(full1, start[i] + cnt[i]);
  }
  full1 = min(full1, n_ring);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    full0 = max(full0, __shfl_xor_sync(0xffffffffu, full0, o));
    full1 = min(full1, __shfl_xor_sync(0xffffffffu, full1, o));
  }

  // Queries: lane (g, t) holds dims 16c + 4t .. + 3 of its rows, which the
  // chunk's contraction takes in the order the key bytes come in.
  uint32_t qh[MT][KC][4], ql[MT][KC][4];  // f16: one k16 step a chunk
  uint32_t th[MT][I8 ? 1 : KC][2][4], tl[MT][I8 ? 1 : KC][2][4];  // TF32: two k8 steps a chunk
  float qs[2 * MT];                        // scale of a score: log2(e) / sqrt(qk) / query scale
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    float4 f[2][KC];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = m * 16 + e * 8 + g;
      const bool in = r < rows;
      const int rr = r0 + (in ? r : 0), n = A.by_rep.div(rr), h = kh * A.rep + rr - n * A.rep;
      const float* src = A.q + ((size_t)b * A.T + n) * A.ldq + (size_t)h * A.qk;
      float mx = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = c * 16 + 4 * t + i;
          x[i] = in && d < A.qk ? __ldg(src + d) : 0.f;
          mx = fmaxf(mx, fabsf(x[i]));
        }
        f[e][c] = make_float4(x[0], x[1], x[2], x[3]);
      }
      float s = A.scale;
      if (I8) {
        // Power of two that brings the row's max into [2^13, 2^14): the f16
        // remainders of all but vanishing elements stay normal numbers.
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int ef = (int)(__float_as_uint(mx) >> 23);
        const int ex = ef == 0 || ef >= 255 ? 0 : min(140 - ef, 126);
        const float up = __uint_as_float((uint32_t)(127 + ex) << 23);
        s *= __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          f[e][c].x *= up, f[e][c].y *= up, f[e][c].z *= up, f[e][c].w *= up;
        }
      }
      qs[2 * m + e] = s;
    }
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      if (I8) {
        split2(f[0][c].x, f[0][c].y, &qh[m][c][0], &ql[m][c][0]);
        split2(f[1][c].x, f[1][c].y, &qh[m][c][1], &ql[m][c][1]);
        split2(f[0][c].z, f[0][c].w, &qh[m][c][2], &ql[m][c][2]);
        split2(f[1][c].z, f[1][c].w, &qh[m][c][3], &ql[m][c][3]);
      } else {
        const int cc = I8 ? 0 : c;
        split_t(f[0][c].x, &th[m][cc][0][0], &tl[m][cc][0][0]);
        split_t(f[1][c].x, &th[m][cc][0][1], &tl[m][cc][0][1]);
        split_t(f[0][c].y, &th[m][cc][0][2], &tl[m][cc][0][2]);
        split_t(f[1][c].y, &th[m][cc][0][3], &tl[m][cc][0][3]);
        split_t(f[0][c].z, &th[m][cc][1][0], &tl[m][cc][1][0]);
        split_t(f[1][c].z, &th[m][cc][1][1], &tl[m][cc][1][1]);
        split_t(f[0][c].w, &th[m][cc][1][2], &tl[m][cc][1][2]);
        split_t(f[1][c].w, &th[m][cc][1][3], &tl[m][cc][1][3]);
      }
    }
  }

  char* mine = smem + wid * TT::WARP_BYTES;
  // Columns past the head's width are zero for good (the copies never write
  // them); the first block's copies start after.
  for (int i = lane * 16; i < TT::WARP_BYTES; i += 512)
    *reinterpret_cast<uint4*>(mine + i) = make_uint4(0, 0, 0, 0);
  __syncwarp();

  const size_t ring_at = (size_t)b * A.slots * A.kvh, draft_at = (size_t)b * A.T * A.kvh;
  const char *rk = A.k + ring_at * A.qk * TT::ES, *rv = A.v + ring_at * A.vh * TT::ES;
  const char *dk = A.drafted ? A.tk + draft_at * A.qk * TT::ES : nullptr,
             *dv = A.drafted ? A.tv + draft_at * A.vh * TT::ES : nullptr;
  const int ring_blocks = (n_ring + PB - 1) / PB, blocks = ring_blocks + (A.drafted + PB - 1) / PB;
  const int blk0 = (int)((long)blocks * z / A.nsplit) + wid, blk1 = (int)((long)blocks * (z + 1) / A.nsplit);

  auto issue = [&](int blk, int buf) {
    if (blk < blk1) {
      char* dst = mine + buf * TT::BUF;
      if (blk < ring_blocks) {
        if (piece == 16)
          tree_copy<TT, I8, 16>(dst, rk, rv, I8 ? A.ks + ring_at : nullptr, I8 ? A.vs + ring_at : nullptr,
                                          A.kvh, kh, A.qk, A.vh, blk * PB, n_ring, slot0, A.slots, lane);
        else
          tree_copy<TT, I8, 4>(dst, rk, rv, I8 ? A.ks + ring_at : nullptr, I8 ? A.vs + ring_at : nullptr,
                                         A.kvh, kh, A.qk, A.vh, blk * PB, n_ring, slot0, A.slots, lane);
      } else {
        const int o = (blk - ring_blocks) * PB;
        if (piece == 16)
          tree_copy<TT, I8, 16>(dst, dk, dv, I8 ? A.tks + draft_at : nullptr,
                                          I8 ? A.tvs + draft_at : nullptr, A.kvh, kh, A.qk, A.vh, o, A.drafted, 0,
                                          A.T, lane);
        else
          tree_copy<TT, I8, 4>(dst, dk, dv, I8 ? A.tks + draft_at : nullptr,
                                         I8 ? A.tvs + draft_at : nullptr, A.kvh, kh, A.qk, A.vh, o, A.drafted, 0, A.T,
                                         lane);
      }
    }
    cp_commit();
  };

  float o[MT][VN][4], mx[2 * MT], sum[2 * MT];
  int vexp, vlow;         // int8: outputs are held times 2^(140 - vexp); least exponent of a value scale
  bool careful = false;   // a second run over the blocks, see below
again:
  vexp = 14, vlow = 255;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < VN; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) mx[i] = -INFINITY, sum[i] = 0.f;

  issue(blk0, 0);
  int buf = 0;
  for (int blk = blk0; blk < blk1; blk += TREE_WARPS, buf ^= 1) {
    issue(blk + TREE_WARPS, buf ^ 1);
    cp_wait<1>();
    __syncwarp();
    const char* kb = mine + buf * TT::BUF;
    const char* vb = kb + TT::K_BYTES;
    const float* sc = reinterpret_cast<const float*>(vb + TT::V_BYTES);
    const bool ring = blk < ring_blocks;
    const int o0 = (ring ? blk : blk - ring_blocks) * PB;

    // ---- scores of PB positions
    float s[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.f;
    if (I8) {
      // ldmatrix: (positions 0-7, chunk c), (8-15, c), (0-7, c + 1), (8-15, c + 1)
      const char* kr = kb + (((lane >> 3) & 1) * 8 + (lane & 7)) * TT::KS + (lane >> 4) * 16;
#pragma unroll
      for (int p = 0; p < PB / 16; ++p)
#pragma unroll
        for (int c = 0; c < KC; c += 2) {
          uint32_t u[4];
          // The last odd chunk's second half reads its own first half again.
          ldm4(u, kr + p * 16 * TT::KS + c * 16 - (c + 1 < KC ? 0 : (lane >> 4) * 16));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (c + (e >> 1) >= KC) continue;
            const int cc = c + (e >> 1) < KC ? c + (e >> 1) : 0;
            uint32_t b0, b1;
            codes_h2<0x4140, 0x4342>(u[e], &b0, &b1);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              if (KC > 4) {
                float x[4] = {0.f, 0.f, 0.f, 0.f};
                mma_h(x, ql[m][cc], b0, b1);
                mma_h(x, qh[m][cc], b0, b1);
                add4(s[m][2 * p + (e & 1)], x);
              } else {
                mma_h(s[m][2 * p + (e & 1)], ql[m][cc], b0, b1);
                mma_h(s[m][2 * p + (e & 1)], qh[m][cc], b0, b1);
              }
            }
          }
        }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const float4 f = *reinterpret_cast<const float4*>(kb + ((n * 8 + g) * TT::KS + c * 16 + 4 * t) * 4);
          uint32_t h[4], l[4];
          split_t(f.x, &h[0], &l[0]);
          split_t(f.y, &h[1], &l[1]);
          split_t(f.z, &h[2], &l[2]);
          split_t(f.w, &h[3], &l[3]);
          const int cc = I8 ? 0 : c;
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              mma_t(x, tl[m][cc][w], h[2 * w], h[2 * w + 1]);
              mma_t(x, th[m][cc][w], l[2 * w], l[2 * w + 1]);
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) mma_t(x, th[m][cc][w], h[2 * w], h[2 * w + 1]);
            add4(s[m][n], x);
          }
        }
    }
    if (I8) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 k2 = *reinterpret_cast<const float2*>(sc + n * 8 + 2 * t);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          s[m][n][0] *= k2.x, s[m][n][1] *= k2.y;
          s[m][n][2] *= k2.x, s[m][n][3] *= k2.y;
        }
      }
    }
    // ---- what the rows see
    if (!ring) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) {
        uint32_t w;
        if (A.mask) {
          w = __ldg(A.mask + ((size_t)b * A.T + node[i]) * A.words + (o0 >> 5)) >> (o0 & 31);
        } else {
          const int up = node[i] - o0 + 1;  // a chain: nodes 0 .. its own
          w = up >= 32 ? 0xffffffffu : up <= 0 ? 0u : (1u << up) - 1u;
        }
        const int left = A.drafted - o0;
        if (left < 32) w &= (1u << left) - 1u;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!((w >> (n * 8 + 2 * t + e)) & 1)) s[i >> 1][n][(i & 1) * 2 + e] = -INFINITY;
      }
    } else if (o0 < full0 || o0 + PB > full1) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int off = o0 + n * 8 + 2 * t + e;
            int d = off - start[i];
            if (d < 0) d += A.slots;
            if (off >= n_ring || d >= cnt[i]) s[i >> 1][n][(i & 1) * 2 + e] = -INFINITY;
          }
    }
    // ---- running max and sum per row
    float mz[2 * MT], corr[2 * MT];
    bool moved = false;
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
      float m = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n) m = fmaxf(m, fmaxf(s[i >> 1][n][(i & 1) * 2], s[i >> 1][n][(i & 1) * 2 + 1]));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      m = fmaxf(m * qs[i], mx[i]);  // in base-2 units
      moved |= m != mx[i];
      mz[i] = m == -INFINITY ? 0.f : m;
      corr[i] = ex2(mx[i] - mz[i]);
      mx[i] = m;
    }
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
      float add = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[i >> 1][n][(i & 1) * 2 + e];
          x = ex2(fmaf(x, qs[i], -mz[i]));
          add += x;
        }
      sum[i] = sum[i] * corr[i] + add;
    }
    // ---- value scales: held so that the largest so far is in [2^13, 2^14),
    // where the weights' f16 remainders stay normal numbers
    float grow = 1.f;
    float2 v2[NT];
    if (I8) {
      if (fabsf(sc[lane]) > KEY_SCALE_FAR) range[2] = 1;
      const uint32_t a = __float_as_uint(fabsf(sc[PB + lane]));
      const uint32_t top = __reduce_max_sync(0xffffffffu, a);
      vlow = min(vlow, (int)(__reduce_min_sync(0xffffffffu, a ? a : 0x7f800000u) >> 23));
      const int e = min(max((int)(top >> 23), vexp), 253);
      if (!careful && e != vexp) {
        grow = e - vexp > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (e - vexp)) << 23);
        vexp = e;
        moved = true;
      }
      const float f = __uint_as_float((uint32_t)(267 - vexp) << 23);  // 2^(140 - vexp)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        v2[n] = *reinterpret_cast<const float2*>(sc + PB + n * 8 + 2 * t);
        if (!careful) v2[n].x *= f, v2[n].y *= f;
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < VN; ++n) {
          o[m][n][0] *= corr[2 * m] * grow, o[m][n][1] *= corr[2 * m] * grow;
          o[m][n][2] *= corr[2 * m + 1] * grow, o[m][n][3] *= corr[2 * m + 1] * grow;
        }
    }
    // ---- outputs
    if (careful) {
      // One position at a time, leaving out those of weight zero.
#pragma unroll 1
      for (int p = 0; p < PB; ++p) {
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
          float w = 0.f;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (p == n * 8 + 2 * t + e) w = s[i >> 1][n][(i & 1) * 2 + e];
          w = __shfl_sync(0xffffffffu, w, (lane & ~3) + ((p & 7) >> 1));
          if (w == 0.f) continue;
#pragma unroll
          for (int n = 0; n < VN; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = tree_dim<I8>(n, 2 * t + e);
              const float x = I8 ? (float)*(const int8_t*)(vb + p * TT::VS + d) * sc[PB + p]
                                 : *reinterpret_cast<const float*>(vb + (p * TT::VS + d) * 4);
              o[i >> 1][n][(i & 1) * 2 + e] += w * x;
            }
        }
      }
    } else if (I8) {
      constexpr int PS = PB / 16;
      uint32_t ah[PS][MT][4], al[PS][MT][4];
#pragma unroll
      for (int p = 0; p < PS; ++p)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const float* x = s[m][2 * p + w];
            const float2 vv = v2[2 * p + w];
            split2(x[0] * vv.x, x[1] * vv.y, &ah[p][m][2 * w], &al[p][m][2 * w]);
            split2(x[2] * vv.x, x[3] * vv.y, &ah[p][m][2 * w + 1], &al[p][m][2 * w + 1]);
          }
      // ldmatrix.trans: (positions 0-7, dims 16c ..), (8-15, same), then chunk c + 1
      const char* vr = vb + (((lane >> 3) & 1) * 8 + (lane & 7)) * TT::VS + (lane >> 4) * 16;
#pragma unroll
      for (int c = 0; c < VHP / 16; c += 2) {
        uint32_t u[PS][4];
#pragma unroll
        for (int p = 0; p < PS; ++p) ldm4t(u[p], vr + p * 16 * TT::VS + c * 16);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t ev[PS][2], od[PS][2];  // even and odd dims of positions 0-7 and 8-15
#pragma unroll
          for (int p = 0; p < PS; ++p)
#pragma unroll
            for (int h = 0; h < 2; ++h) codes_h2<0x4240, 0x4341>(u[p][2 * w + h], &ev[p][h], &od[p][h]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = 0; p < PS; ++p) mma_h(x, al[p][m], ev[p][0], ev[p][1]), mma_h(y, al[p][m], od[p][0], od[p][1]);
#pragma unroll
            for (int p = 0; p < PS; ++p) mma_h(x, ah[p][m], ev[p][0], ev[p][1]), mma_h(y, ah[p][m], od[p][0], od[p][1]);
            add4(o[m][2 * (c + w)], x);
            add4(o[m][2 * (c + w) + 1], y);
          }
        }
      }
    } else {
      uint32_t ah[NT][MT][4], al[NT][MT][4];  // k index t is position 2t, t + 4 position 2t + 1
#pragma unroll
      for (int p = 0; p < NT; ++p)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          split_t(s[m][p][0], &ah[p][m][0], &al[p][m][0]);
          split_t(s[m][p][2], &ah[p][m][1], &al[p][m][1]);
          split_t(s[m][p][1], &ah[p][m][2], &al[p][m][2]);
          split_t(s[m][p][3], &ah[p][m][3], &al[p][m][3]);
        }
      const float* vr = reinterpret_cast<const float*>(vb) + 2 * t * TT::VS + g;
#pragma unroll
      for (int n = 0; n < VN; ++n) {
        uint32_t vh2[NT][2], vl2[NT][2];
#pragma unroll
        for (int p = 0; p < NT; ++p)
#pragma unroll
          for (int h = 0; h < 2; ++h) split_t(vr[(p * 8 + h) * TT::VS + n * 8], &vh2[p][h], &vl2[p][h]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = 0; p < NT; ++p) {
            mma_t(x, al[p][m], vh2[p][0], vh2[p][1]);
            mma_t(x, ah[p][m], vl2[p][0], vl2[p][1]);
          }
#pragma unroll
          for (int p = 0; p < NT; ++p) mma_t(x, ah[p][m], vh2[p][0], vh2[p][1]);
          add4(o[m][n], x);
        }
      }
    }
    __syncwarp();  // this buffer is refilled next
  }
  cp_wait<0>();
  bool lost = false;  // a row whose sum is no number
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
    lost |= !(sum[i] <= 3.4028234e38f);
  }
  // A weight of zero times a value that is no number must not count (a node
  // masked for some rows only may hold anything), and neither may a scale that a
  // row does not see cost it bits: where an output came out infinite or NaN (of a
  // row whose sum is a number; the others see to themselves below), or the value
  // scales lie more than 2^12 apart, the warp takes its blocks again, position by
  // position in f32: 256 sessions over 1043 int8 positions 49 -> 190 us with one such
  // value scale in each.
  if (!careful) {
    bool odd = I8 && vexp - vlow > 12;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < VN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          odd |= !(fabsf(o[m][n][e]) <= 3.4028234e38f) && sum[2 * m + (e >> 1)] <= 3.4028234e38f;
    if (__any_sync(0xffffffffu, odd)) {
      careful = true;
      __syncwarp();
      goto again;
    }
  }
  // Outputs to their own scale.
  if (I8 && !careful) {
    const float f = __uint_as_float((uint32_t)(vexp - 13) << 23);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < VN; ++n) o[m][n][0] *= f, o[m][n][1] *= f, o[m][n][2] *= f, o[m][n][3] *= f;
  }
  // ---- the four warps' results meet (shared memory reused)
  __syncthreads();
  constexpr int PW = VHP + 4;
  float* P = reinterpret_cast<float*>(smem);  // [warp][MT * 16][PW]: outputs, max, sum
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    float* row = P + ((size_t)wid * MT * 16 + (i >> 1) * 16 + (i & 1) * 8 + g) * PW;
#pragma unroll
    for (int n = 0; n < VN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) row[tree_dim<I8>(n, 2 * t + e)] = o[i >> 1][n][(i & 1) * 2 + e];
    if (t == 0) row[VHP] = mx[i], row[VHP + 1] = sum[i];
  }
  // Rows whose sum is no number (an infinite key has no finite parts: its
  // remainder is NaN, but its score may be -inf and weigh nothing) are done again,
  // and so are rows of which a score may have passed the range before the query's
  // power of two is taken back.
  const bool far = I8 && *(volatile int*)(range + 2);
  if (__builtin_expect(__any_sync(0xffffffffu, lost || far), 0)) {
    __syncwarp();
    tree_again<I8, MT * 16, PB, PW, VHP>(A, P + (size_t)wid * MT * 16 * PW, far);
  }
  __syncthreads();
  // Splits of a cluster: each block leaves its rows (outputs, max, sum) in warp
  // 0's place, then the blocks share the rows out and read one another's.
  const bool split = A.nsplit > 1;
  const int width = split ? A.vh + 2 : A.vh;
  const size_t ws = (size_t)MT * 16 * PW;
  for (int i = tid; i < rows * width; i += TREE_THREADS) {
    const int r = i / width, d = i - r * width;
    const float* p = P + (size_t)r * PW;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < TREE_WARPS; ++w) M = fmaxf(M, p[w * ws + VHP]);
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < TREE_WARPS; ++w) {
      const float m = p[w * ws + VHP], l = p[w * ws + VHP + 1];
      if (l == 0.f) continue;
      const float f = m == -INFINITY ? 1.f : ex2(m - M);  // a sum without a max is NaN, and stays
      L += f * l;
      if (d < A.vh) acc += f * p[w * ws + d];
    }
    const int rr = r0 + r;
    if (split) {
      const float x = d < A.vh ? acc : d == A.vh ? M : L;
      if (cluster)
        P[TREE_WARPS * ws + (size_t)r * PW + d] = x;
      else
        A.part[((((size_t)b * A.kvh + kh) * A.nsplit + z) * R + rr) * (A.vh + 2) + d] = x;
    } else {
      const int n = A.by_rep.div(rr), h = kh * A.rep + rr - n * A.rep;
      A.out[(((size_t)b * A.T + n) * A.heads + h) * A.vh + d] = L == 0.f ? 0.f : acc / L;
    }
  }
  if (!cluster) return;
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  const float* own = P + TREE_WARPS * ws;
  for (int i = tid; i < rows * A.vh; i += TREE_THREADS) {
    const int r = i / A.vh, d = i - r * A.vh;
    if (r % A.nsplit != z) continue;
    float M = -INFINITY;
    for (int s = 0; s < A.nsplit; ++s) M = fmaxf(M, cl.map_shared_rank(own, s)[(size_t)r * PW + A.vh]);
    float L = 0.f, acc = 0.f;
    for (int s = 0; s < A.nsplit; ++s) {
      const float* p = cl.map_shared_rank(own, s) + (size_t)r * PW;
      const float m = p[A.vh], l = p[A.vh + 1];
      if (l == 0.f) continue;
      const float f = m == -INFINITY ? 1.f : ex2(m - M);
      L += f * l;
      acc += f * p[d];
    }
    const int rr = r0 + r, n = A.by_rep.div(rr), h = kh * A.rep + rr - n * A.rep;
    A.out[(((size_t)b * A.T + n) * A.heads + h) * A.vh + d] = L == 0.f ? 0.f : acc / L;
  }
  cl.sync();  // no block leaves while it may be read
}

// Joins the splits, a warp a row: the weights 2^(m_z - M) in lanes, then two
// neighbouring dims a lane, eight splits on their way at a time, in split order.
__global__ void __launch_bounds__(256) tree_join_kernel(const float* __restrict__ part, int rows_all, int R, int T,
                                                        int heads, int kvh, int rep, int vh, int ns,
                                                        float* __restrict__ out) {
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (w >= rows_all) return;
  const int bk = w / R, r = w - bk * R, b = bk / kvh, kh = bk - b * kvh;
  const size_t pw = vh + 2, step = (size_t)R * pw;
  const float* p = part + ((size_t)bk * ns * R + r) * pw;
  float M = -INFINITY;
  for (int z = lane; z < ns; z += 32) M = fmaxf(M, p[z * step + vh]);
  M = warp_max(M);
  float L = 0.f;
  float2 acc[2] = {{0.f, 0.f}, {0.f, 0.f}};
  for (int z0 = 0; z0 < ns; z0 += 32) {
    const int z = z0 + lane;
    float f = 0.f, l = 0.f;
    if (z < ns) {
      const float2 ml = *reinterpret_cast<const float2*>(p + z * step + vh);
      l = ml.y;
      f = l == 0.f ? 0.f : ml.x == -INFINITY ? 1.f : ex2(ml.x - M);  // a sum without a max is NaN, and stays
      l = l == 0.f ? 0.f : f * l;
    }
    L += warp_sum(l);
    const int n = min(32, ns - z0);
    for (int i0 = 0; i0 < n; i0 += 8) {
      float2 x[8][2];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = 2 * lane + 64 * j;
          x[i][j] = i0 + i < n && d < vh ? *reinterpret_cast<const float2*>(p + (z0 + i0 + i) * step + d) : make_float2(0.f, 0.f);
        }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float g = i0 + i < n ? __shfl_sync(0xffffffffu, f, i0 + i) : 0.f;
        if (g == 0.f) continue;  // an empty split's row may hold anything
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[j].x += g * x[i][j].x, acc[j].y += g * x[i][j].y;
      }
    }
  }
  const int t = r / rep, h = kh * rep + r - t * rep;
  float* dst = out + (((size_t)b * T + t) * heads + h) * vh;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int d = 2 * lane + 64 * j;
    if (d < vh) dst[d] = L == 0.f ? 0.f : acc[j].x / L, dst[d + 1] = L == 0.f ? 0.f : acc[j].y / L;
  }
}

template <bool I8, int QKP, int VHP, int MT>
constexpr size_t tree_smem() {
  return std::max((size_t)TREE_WARPS * TreeTile<I8, QKP, VHP>::WARP_BYTES,
                  (size_t)(TREE_WARPS + 1) * MT * 16 * (VHP + 4) * 4);
}

// Blocks an SM holds.
template <bool I8, int QKP, int VHP, int MT>
int tree_resident() {
  static const int n = [] {
    auto kern = attend_tree_kernel<I8, QKP, VHP, MT>;
    int r = 0;
    if (allow_smem((const void*)kern, tree_smem<I8, QKP, VHP, MT>(), true) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&r, kern, TREE_THREADS, tree_smem<I8, QKP, VHP, MT>()) != cudaSuccess)
      r = 1;
    return std::max(r, 1);
  }();
  return n;
}

template <bool I8, int QKP, int VHP, int MT>
cudaError_t launch_tree(TreeArgs A, int B, int piece, cudaStream_t st) {
  using TT = TreeTile<I8, QKP, VHP>;
  const size_t smem = tree_smem<I8, QKP, VHP, MT>();
  auto kern = attend_tree_kernel<I8, QKP, VHP, MT>;
  cudaError_t e = allow_smem((const void*)kern, smem, true);
  if (e != cudaSuccess) return e;
  const int R = A.T * A.rep, tiles = (R + MT * 16 - 1) / (MT * 16);
  const int cluster = A.nsplit > 1 && !A.part;
  for (int b0 = 0; b0 < B; b0 += 65535) {
    const int n = std::min(65535, B - b0);
    const TreeArgs C = tree_sessions(A, b0, TT::ES);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tiles * A.kvh * A.nsplit, n);
    cfg.blockDim = dim3(TREE_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster ? A.nsplit : 1;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kern, C, piece, cluster);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

int tree_tile_rows(int R, int qk, int vh) { return R <= 16 || qk > 64 || vh > 64 ? 16 : 32; }

// F<I8, QKP, VHP, MT> of the mma.sync form that heads of these widths and R rows take.
#define NB_TREE_FORM(CALL)                                       \
  do {                                                           \
    const bool one = tree_tile_rows(R, qk, vh) == 16;            \
    if (qk > 64 || vh > 64) CALL(128, 128, 1);                   \
    else if (qk > 48 && one) CALL(64, 64, 1);                    \
    else if (qk > 48) CALL(64, 64, 2);                           \
    else if (one) CALL(48, 64, 1);                               \
    else CALL(48, 64, 2);                                        \
  } while (0)

}  // namespace

// How a call runs: on tcgen05 or mma.sync, and over how many position splits.
// mma.sync: as many as keep the grid in one wave (clusters leave a few places
// empty), each of at least 8 blocks of 32 positions; 9 to 16 are 8, which join
// inside their cluster. Measured at one token, 6 rows of 48/64 int8 (splits: us):
//   16 x 1000   2: 17.4  4: 14.3  8: 13.0      32 x 1000   2: 18.1  6: 15.4  8: 22.9
//   64 x 1000   1: 22.1  2: 20.3  3: 18.8  4: 28.2
//   256 x 1000  1: 45.2  2: 58.1               16 x 4000   8: 18.8  9: 22.9  16: 27.2
//   1 x 6000    4: 29.0  8: 20.8  16: 18.8  24: 16.7
// and with eight splits left to a join kernel 16 x 1000 takes 15.3, 16 x 4000 20.8.
// Both forms plan from `slots`, as the ranges lie on the device: a ring much larger
// than what is seen of it is split as if full. Eight sessions that see 512
// positions take 17.9 us in rings of 33000 places against 14.5 in rings of 544 (12 rows
// of a KV head; 96 rows, tcgen05: 23.5 against 20.5).
TreePlan tree_plan(const void* k, const void* v, const void* tk, const void* tv, const float* out, int int8, int B,
                   int T, int heads, int kvh, int qk, int vh, int slots) {
  const int es = int8 ? 1 : 4, R = T * (heads / kvh);
  auto al16 = [](const void* p) { return (uintptr_t)p % 16 == 0; };
  TreePlan P;
  P.piece = qk * es % 16 == 0 && vh * es % 16 == 0 && al16(k) && al16(v) && al16(tk) && al16(tv) ? 16 : 4;
  P.umma = al16(out) && tree_umma_takes(int8, R, qk, vh, P.piece);
  if (P.umma) {
    P.nsplit = tree_umma_nsplit(int8, B, R, kvh, qk, vh, slots + (tk ? T : 0));
    P.part = P.nsplit > 1;
    return P;
  }
  const int tr = tree_tile_rows(R, qk, vh);
  const long ctas = (long)B * kvh * ((R + tr - 1) / tr);
  int res = 1;
#define NB_RES(Q, V, M) res = int8 ? tree_resident<true, Q, V, M>() : tree_resident<false, Q, V, M>()
  NB_TREE_FORM(NB_RES);
#undef NB_RES
  const long want = 148l * res * 12 / 13 / ctas, most = std::max(1, (slots + 255) / 256);
  P.nsplit = (int)std::max(1l, std::min(std::min(want, most), 256l));
  if (P.nsplit > TREE_CLUSTER && P.nsplit <= 2 * TREE_CLUSTER) P.nsplit = TREE_CLUSTER;
  // Up to eight splits are a cluster that joins itself; more leave partial
  // results for a second kernel.
  P.part = P.nsplit > TREE_CLUSTER;
  return P;
}

size_t tree_part_floats(int B, int T, int heads, int vh, int nsplit) {
  return nsplit > 1 ? (size_t)B * T * heads * nsplit * (vh + 2) : 0;
}

cudaError_t launch_attend_tree(const float* q, int ldq, const void* k, const void* v, const float* ks, const float* vs,
                               int int8, int slots, const int* lo, const int* hi, const void* tk, const void* tv,
                               const float* tks, const float* tvs, const uint32_t* mask, int B, int T, int heads,
                               int kvh, int qk, int vh, const TreePlan& plan, float* part, float* out,
                               cudaStream_t st) {
  if (B <= 0 || T <= 0) return cudaSuccess;
  TreeArgs A;
  A.q = q, A.ldq = ldq;
  A.k = (const char*)k, A.v = (const char*)v, A.ks = ks, A.vs = vs;
  A.tk = (const char*)tk, A.tv = (const char*)tv, A.tks = tks, A.tvs = tvs;
  A.lo = lo, A.hi = hi, A.mask = mask;
  A.slots = slots, A.T = T, A.heads = heads, A.kvh = kvh, A.rep = heads / kvh, A.qk = qk, A.vh = vh;
  A.words = (T + 31) / 32, A.drafted = tk ? T : 0, A.nsplit = plan.nsplit;
  A.scale = (float)(1.4426950408889634 / sqrt((double)qk));
  A.by_rep = FastDiv(A.rep);
  A.out = out, A.part = part;
  const int piece = plan.piece;
  const int R = T * A.rep;
  cudaError_t e;
#define NB_TREE(Q, V, M) e = int8 ? launch_tree<true, Q, V, M>(A, B, piece, st) : launch_tree<false, Q, V, M>(A, B, piece, st)
  if (plan.umma) e = launch_tree_umma(A, int8, B, st);
  else NB_TREE_FORM(NB_TREE);
#undef NB_TREE
  if (e != cudaSuccess || !plan.part) return e;
  const long rows = (long)B * T * heads;
  tree_join_kernel<<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(part, (int)rows, R, T, heads, kvh, A.rep, vh, plan.nsplit,
                                                               out);
  return cudaGetLastError();
}

}  // namespace nb
