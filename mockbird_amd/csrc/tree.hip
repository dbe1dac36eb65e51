// Attention of drafted trees over the KV rings, and the commit of an accepted
// path into them.
//
// A tree of n <= 64 drafted rows hangs below the last cached position pos0 - 1
// of a sequence: node i has a parent before it (or none), stands at position
// p_i = pos0 + depth(i) and sees
//   - the ring slots whose stored position p satisfies 0 <= p < pos0 and
//     p_i - p < C: what the window would hold had its ancestors been appended
//     (their appends evict exactly the positions p <= p_i - C), and nothing of
//     an earlier draft that was not kept (p >= pos0);
//   - the drafted rows of its ancestors in its window (p_i - p < C) and its own, K
//     roped at their own positions and K and V rounded as the ring stores them.
// So out_i is what appending i's ancestors and i one after another and then
// attending would give, for all nodes in one pass over the window.
#include <algorithm>
#include <type_traits>

#include "kv_types.h"
#include "mb_internal.h"
#include "planes.h"
#include "rope.h"

namespace mb {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

constexpr int kTreeWaves = 4;  // waves per workgroup

struct TreeIn {
  const void* qkv;  // [B][rows] fused rows, row_stride elements apart
  int64_t row_stride;
  int qkv_bf16, rows;
  const int32_t *parent, *pos0, *n_nodes;  // [B][rows], [B], [B] or null (all rows)
  const char *k, *v;
  const int32_t* sp;
  int64_t seq_stride;
  int C;
  const float2* rope;
  float* out;
  int64_t out_stride;
  int B, pieces;  // pieces 0: a workgroup per (sequence, head, group)
  int cus;        // then, if not 0: those in the order of their work, this many at a time
  int32_t* plan;  // kPlanWords: the sequences' places on the line, and a piece's length
  float* part;    // two states per workgroup and row
};

// Nodes of sequence b that are attended (0: none), and the first position.
__device__ __forceinline__ int tree_size(const int32_t* pos0, const int32_t* n_nodes, int rows,
                                         int b, int& p0) {
  p0 = pos0[b];
  const int n = n_nodes ? min(n_nodes[b], rows) : rows;
  return p0 < 0 || p0 > INT32_MAX - kTreeMaxNodes ? 0 : n;
}

// The work as a line.  A sequence's drafted rows are one quantum and every QS
// slots of its window (a batch for each wave of a workgroup) another; the
// sequences' quanta follow one another, and the line is cut into `pieces` equal
// ones, one for each workgroup of a head (and group of nodes).  So all
// workgroups have the same work whatever the windows' lengths are, and all fit
// the chip at once.  (More and smaller workgroups than fit at once start under
// load, where each of their three trips to memory takes several us.)
// A state of a sequence that was cut goes to place 0 of its workgroup where the
// sequence began before the piece, else to place 1.
constexpr int kLineSeqs = 64, kPlanWords = 192;  // sequences on a line; words of TreeIn::plan
// The line's places in LDS: where sequence i begins (starts[kLineSeqs]: the end),
// its position and its nodes.
struct Line {
  int32_t starts[kLineSeqs + 1], p0[kLineSeqs], n[kLineSeqs];
};
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
// Lane i = sequence i; wave 0 (`write`) writes the line.  Returns the line's length,
// that of a piece, and the sequence that the piece begins in.
template <int QS>
__device__ __forceinline__ int lay_line(const TreeIn& a, int piece, int lane, bool write, Line& line,
                                        int& length, int& first) {
  int p0 = 0, n = 0;
  if (lane < a.B) n = tree_size(a.pos0, a.n_nodes, a.rows, lane, p0);
  const int q = n > 0 ? 1 + (min(p0, a.C) + QS - 1) / QS : 0;
  int upto = dpp_add<0x111, 0xF>(q);    // row_shr:1, :2, :4, :8
  upto = dpp_add<0x112, 0xF>(upto);
  upto = dpp_add<0x114, 0xF>(upto);
  upto = dpp_add<0x118, 0xF>(upto);
  upto = dpp_add<0x142, 0xA>(upto);     // row_bcast:15 and :31
  upto = dpp_add<0x143, 0xC>(upto);
  const int total = __builtin_amdgcn_readlane(upto, 63);
  if (write) {
    line.starts[lane] = upto - q;
    line.p0[lane] = p0;
    line.n[lane] = n;
    if (lane == 63) line.starts[kLineSeqs] = total;
  }
  length = max(1, (total + a.pieces - 1) / a.pieces);
  const int at = piece * length;
  const uint64_t who = __ballot(at >= upto - q && at < upto);
  first = who ? __ffsll((unsigned long long)who) - 1 : 0;
  return total;
}
// Workgroups for each (sequence, head, group) in the order of their work.  Such a
// launch fits the chip at once, its workgroups i, i + cus, i + 2 cus .. on one CU, so
// the time is that of the CU with the most work (24 voices of 17 to 61 nodes over up
// to 1001 fp32 slots: 57.5 us in the sequences' order, 46.5 in this).  The longest come first and every
// second round of cus runs backwards, which puts short ones to the longest.
// Returns the sequence of this workgroup (-1: none), and its head and group; all
// waves count ranks, 16 sequences each.
template <int QS, int NT, int G>
__device__ __forceinline__ int by_work(const TreeIn& a, int lane, int wave, int32_t* ranks,
                                       int& head, int& group, int& p0_of, int& n_of) {
  int p0 = 0, n = 0;
  if (lane < a.B) n = tree_size(a.pos0, a.n_nodes, a.rows, lane, p0);
  uint32_t key[G];  // the work, and the lower sequence of the first group first
#pragma unroll
  for (int g = 0; g < G; g++) {
    const int tiles = min(NT, (n - g * 16 * NT + 15) >> 4);
    key[g] = tiles > 0 ? (uint32_t)(tiles * (1 + (min(p0, a.C) + QS - 1) / QS)) << 7 | (127 - 64 * g - lane) : 0u;
  }
  int above[G] = {};
  const int j0 = wave * (kLineSeqs / kTreeWaves), j1 = min(a.B, j0 + kLineSeqs / kTreeWaves);
  for (int j = j0; j < j1; j++)
#pragma unroll
    for (int h = 0; h < G; h++) {
      const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)key[h], j);
#pragma unroll
      for (int g = 0; g < G; g++) above[g] += other > key[g];
    }
#pragma unroll
  for (int g = 0; g < G; g++) ranks[(wave * G + g) * 64 + lane] = above[g];
  __syncthreads();
  const int round = blockIdx.x / a.cus, at = blockIdx.x - round * a.cus;
  const int i = round * a.cus + (round & 1 ? a.cus - 1 - at : at), rank = i / H;
  head = i - rank * H;
  int b = -1;
#pragma unroll
  for (int g = 0; g < G; g++) {
    int r = 0;
#pragma unroll
    for (int w = 0; w < kTreeWaves; w++) r += ranks[(w * G + g) * 64 + lane];
    const uint64_t who = __ballot(key[g] != 0u && r == rank);
    if (who) {
      b = __ffsll((unsigned long long)who) - 1;
      group = g;
    }
  }
  p0_of = __builtin_amdgcn_readlane(p0, max(b, 0));
  n_of = __builtin_amdgcn_readlane(n, max(b, 0));
  return b;
}
// A workgroup's states of its place 0 or 1.
__device__ __forceinline__ float* states(const TreeIn& a, int share, int group, int groups, int rows, int place) {
  return a.part + (((int64_t)share * groups + group) * 2 + place) * rows * PART;
}

// Lane i, of parent `par`: the ancestors of node i, itself among them, one bit
// each.  Every
// round doubles the length of chain that a lane's mask covers.  A parent that
// is not an earlier node counts as none.
__device__ __forceinline__ uint64_t ancestors(int32_t par, int n, int lane) {
  if (lane >= n || par >= lane || par < 0) par = -1;
  uint64_t mask = 1ull << lane;
  while (__ballot(par >= 0)) {
    const int from = par >= 0 ? par : lane;
    const uint32_t lo = __shfl((uint32_t)mask, from), hi = __shfl((uint32_t)(mask >> 32), from);
    const int up = __shfl(par, from);
    mask |= (uint64_t)hi << 32 | lo;
    par = par >= 0 ? up : -1;
  }
  return mask;
}

// cos and sin of pair i at a position beyond the table: those of rope_cs, the
// angle reduced by multiples of pi/2 (held in two doubles: the position's 31 bits
// leave the remainder exact to 2^-53) and the Taylor series in double, its
// coefficients read as it goes.  (The library's double functions, inlined in the
// sequences' loop, keep some forty registers of constants through it.)
__device__ const double kTrig[21] = {
    // (-1)^n / (2n + 1)! and (-1)^n / (2n)!, n from 8 down
    1.0 / 355687428096000.0, -1.0 / 1307674368000.0, 1.0 / 6227020800.0, -1.0 / 39916800.0, 1.0 / 362880.0,
    -1.0 / 5040.0, 1.0 / 120.0, -1.0 / 6.0, 1.0,
    1.0 / 20922789888000.0, -1.0 / 87178291200.0, 1.0 / 479001600.0, -1.0 / 3628800.0, 1.0 / 40320.0,
    -1.0 / 720.0, 1.0 / 24.0, -1.0 / 2.0, 1.0,
    // 2/pi, pi/2 and what pi/2 is above it
    0x1.45f306dc9c883p-1, 0x1.921fb54442d18p+0, 0x1.1a62633145c07p-54};
__device__ __forceinline__ float2 far_cs(int32_t pos, int i) {
  const double a = (double)__fmul_rn((float)pos, __uint_as_float(c_inv_freq_bits[i]));
  const double k = rint(a * kTrig[18]);
  double r = fma(-k, kTrig[19], a);
  r = fma(-k, kTrig[20], r);
  const double r2 = r * r;
  double sn = 0.0, cn = 0.0;
#pragma unroll 1
  for (int n = 0; n < 9; n++) {
    sn = fma(sn, r2, kTrig[n]);
    cn = fma(cn, r2, kTrig[9 + n]);
  }
  sn *= r;
  const int q = (int)((int64_t)k & 3);
  const double c = q & 1 ? sn : cn, s = q & 1 ? cn : sn;
  return make_float2((float)(q == 1 || q == 2 ? -c : c), (float)(q >= 2 ? -s : s));
}

// cos and sin of the four pairs from dim d0 on, all read at once; those of a
// position beyond the table one after another (one copy of that code).
template <bool FAR_TAYLOR>
__device__ __forceinline__ void rope4_cs(const float2* tab, int32_t pos, int d0, float2 (&t)[4]) {
  const float4* r = (const float4*)(tab + (int64_t)min(pos, kRopeTab - 1) * 32 + (d0 >> 1));
  const float4 u = r[0], v = r[1];
  t[0] = make_float2(u.x, u.y);
  t[1] = make_float2(u.z, u.w);
  t[2] = make_float2(v.x, v.y);
  t[3] = make_float2(v.z, v.w);
  if (pos >= kRopeTab) {
#pragma unroll 1
    for (int j = 0; j < 4; j++) {
      float2 cs;
      if constexpr (FAR_TAYLOR) cs = far_cs(pos, (d0 >> 1) + j);
      else rope_cs(tab, pos, (d0 >> 1) + j, cs.x, cs.y);
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (j == k) t[k] = cs;
    }
  }
}
__device__ __forceinline__ void rope8(const float2 (&t)[4], float* x) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    float a, b;
    rope_pair(x[2 * j], x[2 * j + 1], t[j].x, t[j].y, a, b);
    x[2 * j] = a;
    x[2 * j + 1] = b;
  }
}

// The first `bytes` bytes from p on, as a buffer whose loads past the end give zeros.
__device__ __forceinline__ auto buffer_of(const char* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00027000);
}

// One element of a K or V row.
template <bool BF16>
__device__ __forceinline__ float elem(const char* row, int d) {
  return BF16 ? bf16_lo(((const uint16_t*)row)[d]) : ((const float*)row)[d];
}

// One workgroup per head and sequence, or piece of the line, and group of nodes (all
// up to 32 rows, 32 each beyond).  A wave takes batches of SB slots (8 KB of K and V)
// in turn with the other waves of its (sequence, head), forms the scores of all
// nodes, 16 to a tile, and keeps its own softmax state per node; the waves' states
// are joined in LDS at the end, and those of several workgroups by k_tree_merge.
// (With all 64 nodes' states a wave runs alone on its SIMD: 24 voices of up to 61 nodes
// over 1001 fp32 slots 97 us; groups of 32, three waves to a SIMD, and the rope
// table's rows read at once, 72.)
//
// What bounds it, by the kernel's own time: 64 voices x 16 nodes over up to 2048 bf16
// slots, 62 us: HBM, 335 MB at 5.4 TB/s.  24 x 17 .. 61 over up to 1001 fp32 slots, 44
// us: the fp32 matrix instructions, 18.7 us a SIMD on average and a quarter more
// on the CU with the most, between the starts and the joins.  3 x 40 .. 64 over up to
// 16384 bf16 slots, 45 us: two waves a SIMD take 19 us of vector instructions (the
// exponentials and the planes of the weights) and 9 of matrix ones, in one chain
// a wave.  1 x 8 over 1024 fp32 slots, 5.6 us: three trips to memory.
//
// Scores are formed as S^T = K Q^T, 16 slots x 16 nodes: lane (c = lane % 16,
// g = lane / 16) of the accumulator holds slots 4g .. 4g + 3 of node c, which is
// the layout in which the next product O^T = V^T P^T takes P^T, so nothing
// passes between lanes but the nodes' maxima.
//  - bf16 rings: v_mfma_f32_16x16x32_bf16, a batch of 32 slots.  q and the
//    weights are three bf16 planes each (split3), so the products are fp32
//    products of the bf16 K and V.  Lane (c, g) holds V of its 8 slots at dims
//    4c .. 4c + 3 (eight 8-byte loads, whole rows of 128 B per instruction), and a
//    byte permute makes them the four V^T operands of dims 4c + dt.
//  - fp32 rings: v_mfma_f32_16x16x4_f32, a batch of 16 slots, every operand as
//    it is loaded (16 bytes a lane).
// In both, lane (c, g) ends with dims 16g .. 16g + 15 of node c.
//
// The next batch's K is loaded once the scores are formed, its V once the
// weights are applied, so a wave always has half a batch under way.
//
// A batch whose slots are all live for every node needs no test per slot; one
// ballot of the stored positions finds that out.
//
// Infinities and NaN: a product of a weight 0 with a V that is not finite, a
// plane of an infinite q, and a difference of infinities are NaN where the sum
// over the seen slots alone may not be.  Where anything that is not finite
// comes out, the workgroup takes its rows again one node at a time, leaving
// unseen slots out (exact_rows).
template <bool KV_BF16, int NT>
struct TreeState {
  f32x4_t o[NT][4];  // dims 16g + 4i + dt of node c: o[t][dt][i]
  float m[NT], l[NT];
};

template <bool KV_BF16>
struct TreeBatch {
  u32x4_t k[4];                                           // bf16: [u][h]; fp32: [q]
  std::conditional_t<KV_BF16, u32x2_t, u32x4_t> v[KV_BF16 ? 8 : 4];
};

// The same rows again, for inputs that are not finite: lane = slot for the
// scores, lane = dim for the sums.
template <bool KV_BF16>
__device__ __forceinline__ void exact_rows(const TreeIn& a, int tid, int b, int head, int lo, int hi,
                                           bool drafts, float* part, int node0, int n, int p0,
                                           uint64_t anc, const char* dk, const char* dv, int dpitch) {
  constexpr int E = KV_BF16 ? 2 : 4;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t off = ((int64_t)b * a.seq_stride + (int64_t)head * a.C * HD) * E;
  const char *kb = a.k + off, *vb = a.v + off;
  const int32_t* sp = a.sp + (int64_t)b * a.C;
  for (int node = node0 + wave; node < n; node += kTreeWaves) {
    const uint64_t mine = __shfl((uint64_t)anc, node);
    const int pos = p0 + __popcll(mine) - 1;
    const int64_t qoff = ((int64_t)b * a.rows + node) * a.row_stride + head * HD + lane;
    const float x = a.qkv_bf16 ? bf16_lo(((const uint16_t*)a.qkv)[qoff]) : ((const float*)a.qkv)[qoff];
    const float y = __shfl_xor(x, 1);
    float r0, r1;
    const float2 cs = pos < kRopeTab ? a.rope[(int64_t)pos * 32 + (lane >> 1)] : far_cs(pos, lane >> 1);
    rope_pair(lane & 1 ? y : x, lane & 1 ? x : y, cs.x, cs.y, r0, r1);
    const float q = (lane & 1 ? r1 : r0) * 0.125f;
    float m = -INFINITY, l = 0.f, acc = 0.f;
    auto rows = [&](const char* kr, const char* vr, int64_t pitch, bool live) {
      float dot = 0.f;
      for (int d = 0; d < HD; d++) {
        const float qd = __shfl(q, d);
        if (live) dot = fmaf(qd, elem<KV_BF16>(kr + lane * pitch, d), dot);
      }
      float mx = live ? dot : -INFINITY;
      for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      mx = fmaxf(mx, m);
      const float at = mx == -INFINITY ? 0.f : mx;
      const float w = live ? __expf(dot - at) : 0.f, by = __expf(m - at);
      l = l * by + w;
      acc *= by;
      m = mx;
      const uint64_t who = __ballot(live);
      for (int j = 0; j < 64; j++) {
        const float wj = __shfl(w, j);
        if ((who >> j) & 1) acc = fmaf(wj, elem<KV_BF16>(vr + j * pitch, lane), acc);
      }
    };
    for (int base = lo; base < hi; base += 64) {
      const int p = base + lane < hi ? sp[base + lane] : -1;
      const bool live = p >= 0 && p < p0 && (int64_t)pos - p < a.C;
      if (__ballot(live)) rows(kb + (int64_t)base * HD * E, vb + (int64_t)base * HD * E, HD * E, live);
    }
    if (drafts)
      rows(dk, dv, dpitch, lane < n && ((mine >> lane) & 1) && __popcll(mine) - __popcll(anc) < a.C);
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    if (part) {
      float* pp = part + (node - node0) * PART;
      pp[lane] = acc;
      if (lane == 0) {
        pp[64] = m;
        pp[65] = l;
      }
    } else {
      a.out[((int64_t)b * a.rows + node) * a.out_stride + head * HD + lane] = l == 0.f ? 0.f : acc / l;
    }
  }
}

template <bool KV_BF16, int NT, int G>
__global__ __launch_bounds__(64 * kTreeWaves, 3) void k_tree(const TreeIn a) {
  constexpr int SB = KV_BF16 ? 32 : 16;       // slots per batch
  constexpr int E = KV_BF16 ? 2 : 4;          // bytes per element
  constexpr int ROWB = HD * E;                // bytes per slot
  constexpr int NS = SB / 4;                  // slots of a batch per lane
  constexpr int NN = NT * 16;
  constexpr int DR = (NN * G + SB - 1) / SB * SB; // drafted rows kept, in whole batches
  constexpr int QP = HD + 4;                  // floats per q row in LDS
  constexpr int DP = ROWB + 16;               // bytes per drafted row in LDS
  constexpr int FOLD = kTreeWaves * 16 * PART;
  constexpr int NSQ = NN * QP > FOLD ? NN * QP : FOLD;
  __shared__ __align__(16) float sq[NSQ];
  __shared__ __align__(16) char sdk[DR * DP], sdv[DR * DP];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // All pieces of the first group of nodes, then all of the second: a multiple of
  // 8 apart, a piece's two are on one XCD, reading alike.  (8 apart themselves, the
  // first group, which has the more nodes, fell to every other CU.)
  constexpr int QS = kTreeWaves * SB;
  const int shares = G == 1 ? gridDim.x : gridDim.x / G;
  int group = G == 1 ? 0 : blockIdx.x / shares;
  const int share = blockIdx.x - group * shares, piece = share / H;
  int head = share % H;
  __shared__ Line line;
  __shared__ int32_t flag[kTreeWaves];
  int first = piece, end = a.B, from = 0, to = 0;  // the piece: quanta [from, to) from sequence `first` on
  int one_p0 = 0, one_n = 0;
  if (a.pieces) {
    if (G > 1 && piece >= a.pieces) return;
    int length;
    const int total = lay_line<QS>(a, piece, lane, wave == 0, line, length, first);
    __syncthreads();
    if (blockIdx.x == 0) {  // for the merge
      for (int i = threadIdx.x; i <= kLineSeqs; i += 64 * kTreeWaves) a.plan[i] = line.starts[i];
      if (threadIdx.x < kLineSeqs) a.plan[kLineSeqs + 1 + threadIdx.x] = line.n[threadIdx.x];
      if (threadIdx.x == 0) a.plan[2 * kLineSeqs + 1] = length;
    }
    from = piece * length;
    to = min(total, from + length);
    if (from >= to) return;
  } else {
    if (a.cus) {
      // (the counts where q's rows will be)
      static_assert(kTreeWaves * G * 64 <= NN * QP, "the angles are written while others read them");
      first = by_work<QS, NT, G>(a, lane, wave, (int32_t*)sq, head, group, one_p0, one_n);
      if (first < 0) return;
    } else {
      if (G > 1 && piece >= a.B) return;
      one_n = tree_size(a.pos0, a.n_nodes, a.rows, first, one_p0);
    }
    end = first + 1;
  }
  const int node0 = group * NN;  // this group's first node

  for (int b = first; b < end; b++) {
    // (the thread's places are worked out anew for each sequence: kept over the
    // loop they would take more registers than there are)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, c = lane & 15, g = lane >> 4;
    int p0, n;
    if (a.pieces) {
      p0 = line.p0[b];
      n = line.n[b];
    } else {
      p0 = one_p0;
      n = one_n;
    }
    p0 = __builtin_amdgcn_readfirstlane(p0);
    n = __builtin_amdgcn_readfirstlane(n);
    if (n <= node0) continue;  // the whole workgroup
    const int32_t par = a.parent[(int64_t)b * a.rows + min(lane, a.rows - 1)];
    const int nvalid = min(p0, a.C);
    int lo = 0, hi = nvalid;  // this workgroup's slots of the window
    bool drafts = true;       // and whether it has the drafted rows
    float* part = nullptr;    // where its states go; null: it has the whole sequence
    if (a.pieces) {
      const int s0 = __builtin_amdgcn_readfirstlane(line.starts[b]),
                s1 = __builtin_amdgcn_readfirstlane(line.starts[b + 1]);
      if (s0 >= to) break;
      const int j0 = max(from - s0, 0), j1 = min(to, s1) - s0;
      drafts = j0 == 0;
      lo = max(j0 - 1, 0) * QS;
      hi = min(nvalid, (j1 - 1) * QS);
      if (s0 < from || s1 > to) part = states(a, share, group, G, min(a.rows, NN), s0 < from ? 0 : 1);
    }
    const int64_t off = ((int64_t)b * a.seq_stride + (int64_t)head * a.C * HD) * E;
    const char *kb = a.k + off, *vb = a.v + off;
    const int32_t* sp = a.sp + (int64_t)b * a.C;

    // The nodes' rows: q of this group's, and with the drafted rows K and V of every
    // node that they may descend from; thread -> row i / 8, dims 8 (i % 8) on.  The
    // angles of the positions p0 .. p0 + 31, whichever of them the tree has.  Loads
    // return in the order they are issued, so these go before the window's, and
    // none waits for another.  (Angles read once the nodes' depths were known, and the
    // position and count once more per sequence: three trips to memory, 7 us of
    // the 12 that 8 voices' workgroups took.)
    const int row0 = drafts ? 0 : node0, at_row = tid >> 3, d0 = (tid & 7) * 8;
    const bool two = G > 1 && row0 < node0;  // the second group's keys begin with the first's rows
    float rq[8] = {}, rk[8] = {}, rv[8] = {}, rk0[G > 1 ? 8 : 1] = {}, rv0[G > 1 ? 8 : 1] = {};
    auto load_row = [&](int row, int part, float* r) {
      const int64_t roff = ((int64_t)b * a.rows + min(row, a.rows - 1)) * a.row_stride + part * D + head * HD + d0;
      if (a.qkv_bf16) load8<true>(a.qkv, roff, r);
      else load8<false>(a.qkv, roff, r);
    };
    load_row(node0 + at_row, 0, rq);
    if (drafts) {
      load_row(node0 + at_row, 1, rk);
      load_row(node0 + at_row, 2, rv);
    }
    if constexpr (G > 1)
      if (two) {
        load_row(at_row, 1, rk0);
        load_row(at_row, 2, rv0);
      }
    float2 cs[4];
    rope4_cs<true>(a.rope, p0 + at_row, d0, cs);
    __builtin_amdgcn_sched_barrier(0);

    TreeBatch<KV_BF16> x;
    int32_t spl;  // lane l: the stored position of the batch's slot l % SB
    // Slots from hi on are past the buffers' ends: they load as zeros and are dead by
    // their number.  (A head's run is at most 2^28 bytes.)
    const auto kr = buffer_of(kb, hi * ROWB), vr = buffer_of(vb, hi * ROWB), pr = buffer_of((const char*)sp, hi * 4);
    constexpr int ONCE = G == 1 ? 2 : 0;  // the streaming hint where the launch reads a row once
    auto load_k = [&](int base) {
      spl = (int32_t)__builtin_amdgcn_raw_buffer_load_b32(pr, (base + (lane & (SB - 1))) * 4, 0, 0);
      const int at = base * ROWB + c * ROWB + g * 16;
#pragma unroll
      for (int i = 0; i < 4; i++)
        x.k[i] = __builtin_bit_cast(
            u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                         kr, at + (KV_BF16 ? 16 * ROWB * (i >> 1) + 64 * (i & 1) : 64 * i), 0, ONCE));
    };
    auto load_v = [&](int base) {
      const int at = base * ROWB + 4 * g * ROWB + c * 4 * E;
#pragma unroll
      for (int j = 0; j < NS; j++) {
        const int row = at + (16 * (j >> 2) + (j & 3)) * ROWB;
        if constexpr (KV_BF16)
          x.v[j] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(vr, row, 0, ONCE));
        else
          x.v[j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(vr, row, 0, ONCE));
      }
    };
    const int s0 = lo + wave * SB, step = kTreeWaves * SB;
    load_k(s0);
    load_v(s0);
    __builtin_amdgcn_sched_barrier(0);

    const int tiles = min(NT, (n - node0 + 15) / 16);
    const int keys = drafts ? min((min(n, node0 + NN) + SB - 1) / SB * SB, DR) : 0;  // drafted rows, in batches
    const uint64_t anc = ancestors(par, n, lane);
    // the angles, by depth: in the part of sq that q leaves
    static_assert(NN <= 8 * kTreeWaves && NN * QP + 32 * HD <= NSQ, "a group's rows are read at once");
    float* const angles = sq + NN * QP;
#pragma unroll
    for (int j = 0; j < 4; j++) *(float2*)(angles + at_row * HD + d0 + 2 * j) = cs[j];
    __syncthreads();
    auto cs_of = [&](int node) {
      const int src = min(node, n - 1);
      const uint32_t al = __shfl((uint32_t)anc, src), ah = __shfl((uint32_t)(anc >> 32), src);
      const int depth = __popc(al) + __popc(ah) - 1;
      if (G == 1 || depth < 32) {
#pragma unroll
        for (int j = 0; j < 4; j++) cs[j] = *(const float2*)(angles + (depth & 31) * HD + d0 + 2 * j);
      } else {
        rope4_cs<true>(a.rope, p0 + depth, d0, cs);
      }
    };
    auto store_kv = [&](int node, float (&k)[8], float (&v)[8]) {
      rope8(cs, k);
      if (node >= n)
#pragma unroll
        for (int j = 0; j < 8; j++) k[j] = v[j] = 0.f;
      store8<KV_BF16>(sdk + node * DP, d0, k);
      store8<KV_BF16>(sdv + node * DP, d0, v);
    };
    cs_of(node0 + at_row);
    if (at_row < NN) {
      rope8(cs, rq);
#pragma unroll
      for (int j = 0; j < 8; j++) sq[at_row * QP + d0 + j] = rq[j] * 0.125f;  // exact
    }
    if (node0 + at_row < keys) store_kv(node0 + at_row, rk, rv);
    if constexpr (G > 1)
      if (two) {
        cs_of(at_row);
        store_kv(at_row, rk0, rv0);
      }
    auto masks_of = [&](uint64_t mask, int t) {  // of node c of the tile
      const int node = node0 + 16 * t + c;
      const uint32_t lo = __shfl((uint32_t)mask, node), hi = __shfl((uint32_t)(mask >> 32), node);
      return (uint64_t)hi << 32 | lo;
    };
    int deepest = lane < n ? __popcll(anc) - 1 : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) deepest = max(deepest, __shfl_xor(deepest, o));
    deepest = __builtin_amdgcn_readfirstlane(deepest);
    __syncthreads();

    // q as the second operand of the scores: in registers, or with two tiles of
    // bf16 planes in LDS, in the lanes' order (48 registers less)
    constexpr bool QLDS = KV_BF16 && NT > 1;
    __shared__ uint4 sqp[QLDS ? NT * 2 : 1][3][QLDS ? 64 : 1];
    std::conditional_t<KV_BF16, Planes[QLDS ? 1 : NT][2], f32x4_t[NT][4]> q;
    auto planes = [&](int t, int h) {
      const float* r = sq + (16 * t + c) * QP + 32 * h + 8 * g;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = r[j];
      return split3(v);
    };
    if constexpr (QLDS) {
      for (int i = wave; i < NT * 2; i += kTreeWaves) {
        const Planes p = planes(i >> 1, i & 1);
#pragma unroll
        for (int k = 0; k < 3; k++) sqp[i][k][lane] = __builtin_bit_cast(uint4, p.p[k]);
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int t = 0; t < NT; t++) {
        if constexpr (KV_BF16) {
#pragma unroll
          for (int h = 0; h < 2; h++) q[t][h] = planes(t, h);
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) q[t][j] = *(const f32x4_t*)(sq + (16 * t + c) * QP + 16 * j + 4 * g);
        }
      }
    }
    auto plane = [&](auto& q, int t, int h, int k) {
      if constexpr (QLDS) return __builtin_bit_cast(bf16x8_t, sqp[2 * t + h][k][lane]);
      else return q[t][h].p[k];
    };

    TreeState<KV_BF16, NT> st;
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int dt = 0; dt < 4; dt++) st.o[t][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      st.m[t] = -INFINITY;
      st.l[t] = 0.f;
    }

    // scores s[t][j] of slot 16 (j / 4) + 4g + j % 4 of the batch
    float s[NT][NS];
    auto scores = [&]() {
#pragma unroll
      for (int t = 0; t < NT; t++) {
        if (NT > 1 && t >= tiles) break;  // uniform
        if constexpr (KV_BF16) {
          f32x4_t d[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int k = 2; k >= 0; k--)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const bf16x8_t p = plane(q, t, h, k);
#pragma unroll
              for (int u = 0; u < 2; u++)
                d[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x.k[2 * u + h]), p,
                                                               d[u], 0, 0, 0);
            }
#pragma unroll
          for (int j = 0; j < 8; j++) s[t][j] = d[j >> 2][j & 3];
        } else {
          f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              d = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.k[j][e]), q[t][j][e], d, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; j++) s[t][j] = d[j];
        }
      }
    };
    // the batch's scores into the states
    auto apply = [&]() {
      bf16x8_t vt[4];
      if constexpr (KV_BF16) {
#pragma unroll
        for (int dt = 0; dt < 4; dt++) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; j++)
            w[j] = __builtin_amdgcn_perm(x.v[2 * j + 1][dt >> 1], x.v[2 * j][dt >> 1],
                                         dt & 1 ? 0x07060302u : 0x05040100u);
          vt[dt] = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
        }
      }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        if (NT > 1 && t >= tiles) break;
        float mx = s[t][0];
#pragma unroll
        for (int j = 1; j < NS; j++) mx = fmaxf(mx, s[t][j]);
        mx = fmaxf(col_max(mx), st.m[t]);
        if (__ballot(mx > st.m[t])) {  // uniform
          const float by = mx == -INFINITY ? 1.f : __expf(st.m[t] - mx);
          st.l[t] *= by;
#pragma unroll
          for (int dt = 0; dt < 4; dt++) st.o[t][dt] *= by;
          st.m[t] = mx;
        }
        const float m = mx == -INFINITY ? 0.f : mx;
        float p[NS];
#pragma unroll
        for (int j = 0; j < NS; j++) {
          p[j] = __expf(s[t][j] - m);
          st.l[t] += p[j];
        }
        if constexpr (KV_BF16) {
          const Planes pp = split3(p);
#pragma unroll
          for (int k = 2; k >= 0; k--)
#pragma unroll
            for (int dt = 0; dt < 4; dt++)
              st.o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt[dt], pp.p[k], st.o[t][dt], 0, 0, 0);
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int dt = 0; dt < 4; dt++)
              st.o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.v[j][dt]), p[j],
                                                                 st.o[t][dt], 0, 0, 0);
        }
      }
    };

    for (int base = s0; base < hi; base += step) {
      const int32_t sc = base + (lane & (SB - 1)) < hi ? spl : -1;
      scores();
      // (loaded past the last batch too, from the last slot: a branch around the
      // loads would have the next wait drain them all)
      load_k(base + step);
      const uint64_t all = __ballot((sc >= 0) & (sc < p0) & (p0 + deepest - sc < a.C));
      if (~all) {  // uniform
#pragma unroll
        for (int t = 0; t < NT; t++) {
          const int32_t at = p0 + __popcll(masks_of(anc, t)) - 1;
#pragma unroll
          for (int j = 0; j < NS; j++) {
            const int32_t p = __shfl(sc, 16 * (j >> 2) + 4 * g + (j & 3));
            s[t][j] = ((p >= 0) & (p < p0) & (at - p < a.C)) ? s[t][j] : -INFINITY;
          }
        }
      }
      apply();
      load_v(base + step);
    }
    uint64_t kept = anc;
    if (deepest >= a.C) {  // uniform: chains longer than the ring lose their first nodes, as appended rows do
      const int depth = __popcll(anc);
      for (int i = 0; i < n; i++)
        if (depth - __builtin_amdgcn_readlane(depth, i) >= a.C) kept &= ~(1ull << i);
    }
    for (int base = wave * SB; base < keys; base += kTreeWaves * SB) {
      if constexpr (KV_BF16) {
#pragma unroll
        for (int i = 0; i < 4; i++)
          x.k[i] = *(const u32x4_t*)(sdk + (base + 16 * (i >> 1) + c) * DP + g * 16 + 64 * (i & 1));
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x.k[i] = *(const u32x4_t*)(sdk + (base + c) * DP + g * 16 + 64 * i);
      }
#pragma unroll
      for (int j = 0; j < NS; j++)
        x.v[j] = *(const std::remove_reference_t<decltype(x.v[0])>*)(
            sdv + (base + 16 * (j >> 2) + 4 * g + (j & 3)) * DP + c * 4 * E);
      scores();
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const uint64_t sees = masks_of(kept, t);
#pragma unroll
        for (int j = 0; j < NS; j++) {
          const int row = base + 16 * (j >> 2) + 4 * g + (j & 3);
          if (!((sees >> row) & 1)) s[t][j] = -INFINITY;
        }
      }
      apply();
    }

    // join the waves' states, a tile of 16 nodes at a time
    bool bad = false;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const float l = col_sum(st.l[t]);
      __syncthreads();
      float* f = sq + (wave * 16 + c) * PART;
#pragma unroll
      for (int i = 0; i < 4; i++)
        *(f32x4_t*)(f + 16 * g + 4 * i) = f32x4_t{st.o[t][0][i], st.o[t][1][i], st.o[t][2][i], st.o[t][3][i]};
      if (g == 0) {
        f[64] = st.m[t];
        f[65] = l;
      }
      __syncthreads();
      const int i = tid >> 4, d = (tid & 15) * 4, node = node0 + 16 * t + i;
      float M = -INFINITY, L = 0.f;
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kTreeWaves; w++) M = fmaxf(M, sq[(w * 16 + i) * PART + 64]);
#pragma unroll
      for (int w = 0; w < kTreeWaves; w++) {
        const float* r = sq + (w * 16 + i) * PART;
        const float by = M == -INFINITY ? 0.f : __expf(r[64] - M);
        L += by * r[65];
        o += by * *(const f32x4_t*)(r + d);
      }
      if (node < n) {
        bad |= !(fabsf(o[0]) < INFINITY && fabsf(o[1]) < INFINITY && fabsf(o[2]) < INFINITY &&
                 fabsf(o[3]) < INFINITY && fabsf(L) < INFINITY && M < INFINITY);
        if (part) {
          float* pp = part + (node - node0) * PART;
          *(f32x4_t*)(pp + d) = o;
          if (d == 0) {
            pp[64] = M;
            pp[65] = L;
          }
        } else {
          float* op = a.out + ((int64_t)b * a.rows + node) * a.out_stride + head * HD + d;
          const float by = L == 0.f ? 0.f : 1.f / L;
          *(f32x4_t*)op = o * by;
        }
      }
    }
    const bool any = __ballot(bad) != 0;
    if (lane == 0) flag[wave] = any;
    __syncthreads();
    static_assert(kTreeWaves == 4, "four flags");
    if (flag[0] | flag[1] | flag[2] | flag[3]) {
      exact_rows<KV_BF16>(a, tid, b, head, lo, hi, drafts, part, node0, min(n, node0 + NN), p0, anc, sdk, sdv, DP);
      __syncthreads();
    }
  }
}

// The states of a sequence that was cut: a wave per node of one (sequence,
// head), lane (g, quad) taking every fourth state's dims 4 quad .. + 3, 16 states
// on their way at once: two trips to memory, 4.0 us over 8 sequences of 16 nodes, 4.9
// over 3 of 64.
__global__ __launch_bounds__(256) void k_tree_merge(const TreeIn a, int groups) {
  const int b = blockIdx.x / H, head = blockIdx.x % H;
  const int lane = threadIdx.x & 63, g = lane >> 4, d = (lane & 15) * 4;
  const int s = a.plan[b], e = a.plan[b + 1], n = a.plan[kLineSeqs + 1 + b], length = a.plan[2 * kLineSeqs + 1];
  const int node = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (node >= n || e == s) return;
  const int first = s / length, splits = (e - 1) / length - first + 1;
  if (splits == 1) return;
  const int rows = min(a.rows, 32), group = node / 32;
  // the first piece's place 1, the others' place 0
  auto state = [&](int i) {
    return states(a, (first + i) * H + head, group, groups, rows, i == 0) + (node - 32 * group) * PART;
  };
  float M = -INFINITY, L = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < splits; s0 += 16) {
    f32x4_t v[4];
    float m[4], l[4], mx = M;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float* p = state(min(s0 + 4 * j + g, splits - 1));
      v[j] = *(const f32x4_t*)(p + d);
      m[j] = p[64];
      l[j] = p[65];
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (s0 + 4 * j + g >= splits) m[j] = -INFINITY;
      mx = fmaxf(mx, m[j]);
    }
    const float by = M == -INFINITY ? 0.f : __expf(M - mx);
    L *= by;
    o *= by;
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (m[j] != -INFINITY) {  // (a state that saw nothing may not be finite)
        const float w = __expf(m[j] - mx);
        L += w * l[j];
        o += w * v[j];
      }
    M = mx;
  }
  // the four lane groups
  const float mx = col_max(M), by = M == -INFINITY ? 0.f : __expf(M - mx);
  L = col_sum(L * by);
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] = col_sum(M == -INFINITY ? 0.f : o[i] * by);
  if (g == 0) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
    *(f32x4_t*)(a.out + ((int64_t)b * a.rows + node) * a.out_stride + head * HD + d) = o * inv;
  }
}

// Workgroups per head of a launch whose work is cut as a line: with the groups
// and heads two per CU.  (us for 24 voices of up to 61 nodes in fp32 / 3 of 64 over
// 16384 slots / 8 of 16 over 2048, bf16: one per CU 57.2 / 55.4 / 17.3, two 57.1 /
// 48.0 / 17.8, three, as many as fit, 61.1 / 49.3 / 18.2.)  0: a workgroup for each
// sequence, where a piece is not shorter than the longest window by what the line
// costs: kLineGain quanta for the second launch and the sequences that begin
// inside a piece, and up to kLineShare for two pieces on a CU that has one
// sequence.  (us as a line / as sequences, by voices x nodes x slots: 1 x 8 x 1024 fp32
// 9.4 / 17.5, 4 x 32 x 512 fp32 12.4 / 16.9, 8 x 16 x 2048 bf16 18.8 / 20.4, 12 x 16 x 4000
// bf16 31.7 / 40.0, 28 x 16 x 8000 bf16 103 / 119, 10 x 64 x 4096 fp32 87 / 92; 10 x 2 x
// 1139 bf16 15.6 / 14.0, 16 x 16 x 1024 bf16 19.1 / 13.9, 24 x 30 x 1001 fp32 41.3 / 36.9,
// 12 x 64 x 2000 bf16 34.9 / 30.2, 21 x 64 x 1001 fp32 62.7 / 54.6; 24 x 8 x 4096 fp32, 86.5
// / 83.6, is taken as a line.)
constexpr int kLineGain = 5, kLineShare = 15;
static int tree_cus(const mb_ctx* ctx) { return ctx->cus_per_xcd > 0 ? ctx->xcds * ctx->cus_per_xcd : 256; }
static int tree_groups(int rows) { return rows <= 32 ? 1 : 2; }
static int tree_pieces(const mb_ctx* ctx, int B, int rows, int32_t max_pos) {
  const int cus = tree_cus(ctx);
  const int pieces = std::max(1, 2 * cus / (H * tree_groups(rows)));
  const int qs = kTreeWaves * (ctx->cfg.kv_dtype == MB_KV_BF16 ? 32 : 16);
  const int window = (std::min(max_pos, ctx->cfg.capacity) + qs - 1) / qs;
  const int piece = (int)(((int64_t)B * (1 + window) + pieces - 1) / pieces);
  return B <= kLineSeqs && window - piece >= kLineGain + std::min(piece, kLineShare) ? pieces : 0;
}

int64_t tree_work_bytes(const mb_ctx* ctx, int B, int rows, int32_t max_pos) {
  if (B < 1) return 0;
  const int64_t g = tree_groups(rows), p = tree_pieces(ctx, B, rows, max_pos);
  return p ? 4 * (kPlanWords + p * H * g * 2 * std::min(rows, 32) * PART) : 0;
}

int launch_tree_attention(mb_ctx* ctx, const RingView& ring, int B, int rows, const void* qkv,
                          int qkv_dtype, int64_t qkv_stride, const int32_t* parent,
                          const int32_t* pos0, const int32_t* n_nodes, int32_t max_pos, float* out,
                          int64_t out_stride, void* work) {
  TreeIn a;
  a.qkv = qkv;
  a.row_stride = qkv_stride;
  a.qkv_bf16 = qkv_dtype == MB_DT_BF16;
  a.rows = rows;
  a.parent = parent;
  a.pos0 = pos0;
  a.n_nodes = n_nodes;
  a.k = (const char*)ring.k;
  a.v = (const char*)ring.v;
  a.sp = ring.sp;
  a.seq_stride = ring.seq_stride;
  a.C = ring.C;
  a.rope = ctx->rope_tab;
  a.out = out;
  a.out_stride = out_stride;
  a.B = B;
  a.pieces = tree_pieces(ctx, B, rows, max_pos);
  a.plan = (int32_t*)work;
  a.part = (float*)work + kPlanWords;
  const int groups = tree_groups(rows);
  const int cus = tree_cus(ctx);
  a.cus = a.pieces == 0 && B <= kLineSeqs && B * H * groups > cus ? cus : 0;
  const unsigned shares = (unsigned)((a.pieces ? a.pieces : B) * H);
  auto go = [&](auto nt, auto g) {
    constexpr int NT = decltype(nt)::value, G = decltype(g)::value;
    const dim3 grid(a.cus ? (shares * G + a.cus - 1) / a.cus * a.cus : G == 1 ? shares : (shares + 7) / 8 * 8 * G);
    if (ring.bf16) hipLaunchKernelGGL((k_tree<true, NT, G>), grid, dim3(64 * kTreeWaves), 0, ctx->stream, a);
    else hipLaunchKernelGGL((k_tree<false, NT, G>), grid, dim3(64 * kTreeWaves), 0, ctx->stream, a);
  };
  std::integral_constant<int, 1> one;
  std::integral_constant<int, 2> two;
  if (rows <= 16) go(one, one);
  else if (rows <= 32) go(two, one);
  else go(two, two);
  MB_HIP(ctx, hipGetLastError());
  if (a.pieces) {
    hipLaunchKernelGGL(k_tree_merge, dim3((unsigned)(B * H), (unsigned)((rows + 3) / 4)), dim3(256), 0,
                       ctx->stream, a, groups);
    MB_HIP(ctx, hipGetLastError());
  }
  return MB_OK;
}

// ----------------------------------------------------------------- commit

// Row i of sequence b's path, node path[b][i] of its drafted rows, goes to
// position pos0[b] + i of every layer's ring as k_ring_write would write it.
// Each thread owns 8 dims of one head of one row of one layer; a row that a
// later one of the same path overwrites is not stored, nor one whose node is
// not a drafted row or whose position the ring cannot hold.
// 64 voices x up to 8 rows x 12 layers in bf16 (21 MB): 8.0 us, 2.6 TB/s: two dependent
// trips to memory (the path, the rows), in two rounds of waves: the rings' own cos
// and sin of positions beyond the table, bit for bit, take 86 registers (as a
// series, which may end a bit away, 45).  One voice: 3.4 us, a launch.
template <bool IN_BF16, bool KV_BF16>
__global__ __launch_bounds__(256) void k_tree_commit(
    const void* __restrict__ qkv, int64_t row_stride, int64_t layer_stride, int rows,
    const int32_t* __restrict__ pos0, const int32_t* __restrict__ path, int path_max,
    const int32_t* __restrict__ n_path, int B, void* __restrict__ ring_k,
    void* __restrict__ ring_v, int32_t* __restrict__ slot_pos, int64_t seq_stride,
    int64_t layer_seqs, int C, int wrap, const float2* __restrict__ rope_tab) {
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  const int i = (int)(t / (H * 8)), part = (int)(t % (H * 8)), head = part >> 3, d0 = (part & 7) * 8;
  if (i >= path_max) return;
  const int layer = blockIdx.z;
  for (int b = blockIdx.y; b < B; b += gridDim.y) {
    // (the path's entry is read before its count is known: path_max bounds both)
    const int n = min(n_path ? n_path[b] : path_max, path_max);
    const int node = path[(int64_t)b * path_max + i];
    const int32_t p0 = pos0[b];
    const int64_t p64 = (int64_t)p0 + i;
    if (i >= n || (n > C && i < n - C) || node < 0 || node >= rows || p0 < 0 || p64 > INT32_MAX ||
        (!wrap && p64 >= C))
      continue;
    const int32_t pos = (int32_t)p64;
    const int64_t roff = layer * layer_stride + ((int64_t)b * rows + node) * row_stride + head * HD + d0;
    float k[8], v[8];
    load8<IN_BF16>(qkv, roff + D, k);
    load8<IN_BF16>(qkv, roff + 2 * D, v);
    float2 cs[4];
    rope4_cs<false>(rope_tab, pos, d0, cs);
    rope8(cs, k);
    const int slot = wrap ? (int)((uint32_t)pos % (uint32_t)C) : pos;
    const int64_t seq = layer * layer_seqs + b;
    const int64_t koff = seq * seq_stride + ((int64_t)head * C + slot) * HD + d0;
    store8<KV_BF16>(ring_k, koff, k);
    store8<KV_BF16>(ring_v, koff, v);
    if (part == 0) slot_pos[seq * C + slot] = pos;
  }
}

int launch_tree_commit(mb_ctx* ctx, int layer0, int n_layers, int B, int rows, const void* qkv,
                       int qkv_dtype, int64_t qkv_stride, int64_t layer_stride, const int32_t* pos0,
                       int path_max, const int32_t* path, const int32_t* n_path) {
  const int64_t blocks = ((int64_t)path_max * H * 8 + 255) / 256;
  if (blocks > INT32_MAX / 256) return fail(ctx, MB_ERR_ARG, "too many rows in one call");
  const RingView ring = global_ring(ctx, layer0);
  const dim3 grid((unsigned)blocks, (unsigned)std::min(B, 65535), (unsigned)n_layers);
  auto go = [&](auto in, auto kv) {
    hipLaunchKernelGGL((k_tree_commit<decltype(in)::value, decltype(kv)::value>), grid,
                       dim3(256), 0, ctx->stream, qkv, qkv_stride, layer_stride, rows, pos0, path,
                       path_max, n_path, B, ring.k, ring.v, ring.sp, ring.seq_stride,
                       (int64_t)ctx->cfg.max_seqs, ring.C, ring.wrap, ctx->rope_tab);
  };
  std::true_type yes;
  std::false_type no;
  if (qkv_dtype == MB_DT_BF16) { if (ring.bf16) go(yes, yes); else go(yes, no); }
  else { if (ring.bf16) go(no, yes); else go(no, no); }
  MB_HIP(ctx, hipGetLastError());
  return MB_OK;
}

}  // namespace mb
