// Beam search over the rings: the choice of the best continuations of a
// voice's beams, and the move of the rings to the beams that go on.
#include <algorithm>
#include <type_traits>

#include "kv_types.h"
#include "mb_internal.h"

namespace mb {

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------ wave reduces

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}
// op over the wave's 64 lanes; every lane has the result
template <class Op>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t x, Op op) {
  x = op(x, dpp_u32<0xB1>(x));   // quad_perm [1,0,3,2]
  x = op(x, dpp_u32<0x4E>(x));   // quad_perm [2,3,0,1]
  x = op(x, dpp_u32<0x141>(x));  // row_half_mirror
  x = op(x, dpp_u32<0x140>(x));  // row_mirror
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = op(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return op(b[0], b[1]);
}
__device__ __forceinline__ float wave_max(float x) {
  return __uint_as_float(wave_reduce(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ uint32_t wave_min(uint32_t x) {
  return wave_reduce(x, [](uint32_t a, uint32_t b) { return min(a, b); });
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
  return wave_reduce(x, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// ------------------------------------------------------------- one row

// The choice over one voice's W beams and V ids takes the n best of
//   c(w, v) = score_w + (z_wv - m_w) - log sum_u exp(z_wu - m_w)
// with z the logits (penalised where seen, in fp32) and m_w their maximum.
// Within a beam c falls with z, so a row needs its n best logits only, found by
// fp32 compares (the lower id on ties), its maximum and its sum; c itself is
// formed and compared in 64 bits, for the n best of each beam.
constexpr uint32_t kNoId = 0x7fffffffu;
constexpr int kScan = 1024;  // ids a wave reads at a time, 16 to a lane

// What a wave knows of a row: lane k < n holds the k-th best logit so far and
// its id, (-inf, kNoId) where there is none; the maximum; the lane's share of
// the sum.
struct RowTop {
  float v = -INFINITY;
  uint32_t id = kNoId;
  float m = -INFINITY;
  double sum = 0.0;
};

// Merge 16 values a lane into the list: n rounds of the wave's best.
template <class Id>
__device__ __forceinline__ void take_top(float (&z)[16], Id id, int n, int lane, RowTop& t) {
  float nv = -INFINITY;
  uint32_t ni = kNoId;
  for (int r = 0; r < n; r++) {
    float bv = t.v;
    uint32_t bi = t.id;
#pragma unroll
    for (int j = 0; j < 16; j++)
      if (z[j] > bv || (z[j] == bv && id(j) < bi)) {
        bv = z[j];
        bi = id(j);
      }
    const float top = wave_max(bv);
    if (top == -INFINITY) break;  // uniform
    const uint64_t who = __ballot(bv == top);
    const uint32_t win = __popcll(who) == 1
                             ? (uint32_t)__builtin_amdgcn_readlane((int)bi, __ffsll((unsigned long long)who) - 1)
                             : wave_min(bv == top ? bi : kNoId);
    if (lane == r) {
      nv = top;
      ni = win;
    }
    if (t.id == win) t.v = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; j++)
      if (id(j) == win) z[j] = -INFINITY;
  }
  t.v = nv;
  t.id = ni;
}

// Ids [lo, hi) of a row of V logits.  A NaN counts as -inf.  An infinite
// maximum leaves the whole sum to the ids that reach it.
template <bool BF16>
__device__ __forceinline__ void scan_row(const void* row, const uint32_t* seen, float penalty, int lo,
                                         int hi, int n, int lane, RowTop& t) {
  constexpr int PER = BF16 ? 8 : 4;  // consecutive ids of a lane's load
  float least = -INFINITY;           // the n-th best so far
  for (int base = lo; base < hi; base += kScan) {
    auto id = [&](int j) { return (uint32_t)(base + 64 * (j / PER * PER) + lane * PER + j % PER); };
    float z[16];
#pragma unroll
    for (int q = 0; q < 16 / PER; q++) {
      const int at = (int)id(q * PER);
      if (at + PER <= hi) {
        // 16 bytes at the elements' own alignment
        uint4 w;
        __builtin_memcpy(&w, (const char*)row + (int64_t)at * (BF16 ? 2 : 4), 16);
        unpack<BF16>(w, z + q * PER);
      } else {
#pragma unroll
        for (int e = 0; e < PER; e++)
          z[q * PER + e] = at + e >= hi ? -INFINITY
                           : BF16       ? bf16_lo(((const uint16_t*)row)[at + e])
                                        : ((const float*)row)[at + e];
      }
    }
    if (seen) {  // uniform
#pragma unroll
      for (int q = 0; q < 16 / PER; q++) {
        const int at = (int)id(q * PER);
        const uint32_t bits = at < hi ? seen[at >> 5] >> (at & 31) : 0u;
#pragma unroll
        for (int e = 0; e < PER; e++) {
          float& x = z[q * PER + e];
          if ((bits >> e) & 1) x = x < 0.f ? x * penalty : x / penalty;
        }
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; j++) {
      z[j] = z[j] == z[j] ? z[j] : -INFINITY;
      mx = fmaxf(mx, z[j]);
    }
    mx = wave_max(mx);
    if (mx == -INFINITY) continue;  // uniform
    if (mx > t.m) {
      t.sum *= (double)__expf(t.m - mx);
      t.m = mx;
    }
    float p[16];
#pragma unroll
    for (int j = 0; j < 16; j++) p[j] = z[j] == t.m ? 1.f : __expf(z[j] - t.m);
#pragma unroll
    for (int w = 8; w > 0; w >>= 1)
#pragma unroll
      for (int j = 0; j < w; j++) p[j] += p[j + w];
    t.sum += (double)p[0];
    if (mx > least) {
      take_top(z, id, n, lane, t);
      least = __shfl(t.v, n - 1);
    }
  }
}

struct BeamIn {
  const void* logits;  // [B * W] rows, stride elements apart
  int64_t stride;
  int bf16, W, V, n, words;
  const float* scores;    // [B][W]
  const int32_t* done;    // [B][W] or null
  const uint32_t* seen;   // [B][W][words] or null
  int32_t end_id;
  float penalty;
  float* scores_out;  // [B][n]
  int32_t *parent, *token, *done_out;
  uint32_t* seen_out;  // [B][n][words] or null
  char* part;          // chunks > 1: [B * W][chunks] PartRow
  int chunks, chunk;   // parts of a row, ids of a part
};

// One part of a row, in the workspace: 16 bytes, then n (value, id) pairs.
struct PartRow {
  double sum;
  float m;
  uint32_t pad;
};
__device__ __forceinline__ char* part_row(const BeamIn& a, int64_t row, int chunk) {
  return a.part + (row * a.chunks + chunk) * (int64_t)(sizeof(PartRow) + a.n * 8);
}

__device__ __forceinline__ void scan(const BeamIn& a, int64_t row, int lo, int hi, int lane, RowTop& t) {
  const char* p = (const char*)a.logits + row * a.stride * (a.bf16 ? 2 : 4);
  const uint32_t* seen = a.seen ? a.seen + row * a.words : nullptr;
  if (a.bf16) scan_row<true>(p, seen, a.penalty, lo, hi, a.n, lane, t);
  else scan_row<false>(p, seen, a.penalty, lo, hi, a.n, lane, t);
  t.sum = wave_sum(t.sum);
}

// A wave per part of a row.
__global__ __launch_bounds__(256) void k_beam_scan(const BeamIn a, int64_t parts) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= parts) return;
  const int64_t row = i / a.chunks;
  const int c = (int)(i % a.chunks);
  if (a.done && a.done[row]) return;  // an ended beam's logits are not looked at
  RowTop t;
  scan(a, row, c * a.chunk, min(a.V, (c + 1) * a.chunk), lane, t);
  char* p = part_row(a, row, c);
  if (lane == 0) *(PartRow*)p = PartRow{t.sum, t.m, 0u};
  if (lane < a.n) ((uint2*)(p + sizeof(PartRow)))[lane] = make_uint2(__float_as_uint(t.v), t.id);
}

// The parts of a row joined.
__device__ __forceinline__ void join(const BeamIn& a, int64_t row, int lane, RowTop& t) {
  PartRow h{0.0, -INFINITY, 0u};
  if (lane < a.chunks) h = *(const PartRow*)part_row(a, row, lane);
  t.m = wave_max(h.m);
  // (an infinite maximum is the maximum of a part only where it was reached)
  const double by = h.m == t.m ? 1.0 : (double)__expf(h.m - t.m);
  t.sum = wave_sum(h.sum * by);
  const int all = a.chunks * a.n;
  for (int base = 0; base < all; base += kScan) {
    float z[16];
    uint32_t ids[16];
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const int i = base + 64 * j + lane;
      uint2 w = make_uint2(__float_as_uint(-INFINITY), kNoId);
      if (i < all) w = ((const uint2*)(part_row(a, row, i / a.n) + sizeof(PartRow)))[i % a.n];
      z[j] = __uint_as_float(w.x);
      ids[j] = w.y;
    }
    take_top(z, [&](int j) { return ids[j]; }, a.n, lane, t);
  }
}

// A double as an integer of the same order (-0 as 0).
__device__ __forceinline__ uint64_t order_of(double c) {
  const uint64_t u = __builtin_bit_cast(uint64_t, c + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// One workgroup per voice, its waves taking the beams' rows in turn; then the
// first wave merges the beams' lists, lane w holding the head of beam w's.
constexpr int kBeamWaves = 16;
template <bool FUSED>
__global__ __launch_bounds__(64 * kBeamWaves) void k_beam_pick(const BeamIn a) {
  __shared__ float lv[kBeamMax][kBeamMax];
  __shared__ uint32_t li[kBeamMax][kBeamMax];
  __shared__ float lm[kBeamMax];
  __shared__ double ls[kBeamMax];
  __shared__ int32_t from[kBeamMax], tok[kBeamMax];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int b = blockIdx.x;
  for (int w = wave; w < a.W; w += nw) {
    const int64_t row = (int64_t)b * a.W + w;
    if (a.done && a.done[row]) continue;
    RowTop t;
    if (FUSED) scan(a, row, 0, a.V, lane, t);
    else join(a, row, lane, t);
    if (lane < a.n) {
      lv[w][lane] = t.v;
      li[w][lane] = t.id;
    }
    if (lane == 0) {
      lm[w] = t.m;
      ls[w] = t.sum;
    }
  }
  __syncthreads();
  if (wave == 0) {
    const bool mine = lane < a.W;
    const double score = mine ? (double)a.scores[(int64_t)b * a.W + lane] : -INFINITY;
    const bool ended = mine && a.done && a.done[(int64_t)b * a.W + lane];
    const float m = mine && !ended ? lm[lane] : 0.f;
    const double lsum = mine && !ended ? log(ls[lane]) : 0.0;
    int at = 0;  // of the beam's list
    auto head = [&](uint32_t& id) {
      id = kNoId;
      if (!mine || at >= a.n) return (double)-INFINITY;
      if (ended) {
        if (at) return (double)-INFINITY;
        id = (uint32_t)a.end_id;
        return score;
      }
      id = li[lane][at];
      if (id == kNoId) return (double)-INFINITY;
      const float v = lv[lane][at];
      return score + ((v == m ? 0.0 : (double)v - (double)m) - lsum);
    };
    uint32_t id;
    double c = head(id);
    for (int k = 0; k < a.n; k++) {
      const uint64_t key = c > -INFINITY ? order_of(c) : 0ull;  // NaN: none
      const uint32_t hi = wave_umax((uint32_t)(key >> 32));
      const uint32_t lo = wave_umax((uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
      const uint64_t who = __ballot(key && (uint32_t)(key >> 32) == hi && (uint32_t)key == lo);
      const int w = who ? __ffsll((unsigned long long)who) - 1 : -1;  // the lowest beam on ties
      const int64_t o = (int64_t)b * a.n + k;
      if (w < 0 ? lane == 0 : lane == w) {
        const int32_t id_out = w < 0 ? -1 : (int32_t)id;
        a.scores_out[o] = w < 0 ? -INFINITY : (float)c;
        a.parent[o] = w;
        a.token[o] = id_out;
        if (a.done_out) a.done_out[o] = w < 0 || (a.end_id >= 0 && id_out == a.end_id);
        from[k] = w;
        tok[k] = id_out;
      }
      if (lane == w) {
        at++;
        c = head(id);
      }
    }
  }
  if (!a.seen_out) return;
  __syncthreads();
  // every chosen beam's history: its parent's and the chosen id
  for (int i = threadIdx.x; i < a.n * a.words; i += blockDim.x) {
    const int k = i / a.words, j = i % a.words;
    const int w = from[k], v = tok[k];
    uint32_t bits = 0u;
    if (w >= 0) {
      bits = a.seen[((int64_t)b * a.W + w) * a.words + j];
      if (v >> 5 == j) bits |= 1u << (v & 31);
    }
    a.seen_out[((int64_t)b * a.n + k) * a.words + j] = bits;
  }
}

// Ids of a row that one wave reads: all where the voice's own workgroup scans
// its rows, else a 64th of the row at least.
constexpr int kBeamFusedVocab = 4096;
static void beam_parts(int V, int& chunks, int& chunk) {
  chunk = V <= kBeamFusedVocab ? V : std::max(1, (V + 64 * kScan - 1) / (64 * kScan)) * kScan;
  chunks = (V + chunk - 1) / chunk;
}

int64_t beam_work_bytes(int B, int W, int V, int n) {
  int chunks, chunk;
  beam_parts(V, chunks, chunk);
  return chunks > 1 ? (int64_t)B * W * chunks * (int64_t)(sizeof(PartRow) + n * 8) : 0;
}

int launch_beam_select(mb_ctx* ctx, int B, int W, int V, int n, const void* logits, int logits_dtype,
                       int64_t logits_stride, const float* scores, const int32_t* done,
                       int32_t end_id, const uint32_t* seen, double penalty, float* scores_out,
                       int32_t* parent, int32_t* token, int32_t* done_out, uint32_t* seen_out,
                       void* work) {
  BeamIn a;
  a.logits = logits;
  a.stride = logits_stride;
  a.bf16 = logits_dtype == MB_DT_BF16;
  a.W = W;
  a.V = V;
  a.n = n;
  a.words = (V + 31) / 32;
  a.scores = scores;
  a.done = done;
  a.seen = seen;
  a.end_id = end_id;
  a.penalty = (float)penalty;
  a.scores_out = scores_out;
  a.parent = parent;
  a.token = token;
  a.done_out = done_out;
  a.seen_out = seen_out;
  a.part = (char*)work;
  beam_parts(V, a.chunks, a.chunk);
  const dim3 block(64 * std::min(W, kBeamWaves));
  if (a.chunks == 1) {
    hipLaunchKernelGGL(k_beam_pick<true>, dim3((unsigned)B), block, 0, ctx->stream, a);
  } else {
    const int64_t parts = (int64_t)B * W * a.chunks;
    hipLaunchKernelGGL(k_beam_scan, dim3((unsigned)((parts + 3) / 4)), dim3(256), 0, ctx->stream, a, parts);
    MB_HIP(ctx, hipGetLastError());
    hipLaunchKernelGGL(k_beam_pick<false>, dim3((unsigned)B), block, 0, ctx->stream, a);
  }
  MB_HIP(ctx, hipGetLastError());
  return MB_OK;
}

// ---------------------------------------------------------------- reorder

struct ReorderIn {
  char *k, *v;
  int32_t* sp;
  int64_t seq_bytes;  // K (or V) bytes of one sequence's ring
  int64_t head_bytes;
  int max_seqs, groups, W, C, wrap;
  const int32_t *parent, *from, *to;
};

// One thread owns 16 bytes of one slot of one head for all W sequences of a
// group: it reads the parents' before it writes any, so the move is in place
// and every byte is read where its parent still has it.  A group's slots are
// cut into blockDim.x-thread pieces along blockIdx.y.
template <int MW>
__global__ __launch_bounds__(256) void k_ring_reorder(const ReorderIn a, int row_chunks) {
  const int head = blockIdx.x % H;
  const int gl = blockIdx.x / H, group = gl % a.groups, layer = gl / a.groups;
  int64_t first = 0, n = a.C;
  if (a.from) {
    first = max(a.from[group], 0);
    const int64_t to = a.wrap ? (int64_t)a.to[group] : (int64_t)min(a.to[group], a.C);
    n = min(to - first, (int64_t)a.C);
  }
  int from[MW];  // the sequence of the group that w's rows come from; -1: they stay
#pragma unroll
  for (int w = 0; w < MW; w++) {
    const int p = w < a.W ? a.parent[(int64_t)group * a.W + w] : -1;
    from[w] = p >= 0 && p < a.W && p != w ? p : -1;
  }
  const int64_t seq0 = (int64_t)layer * a.max_seqs + (int64_t)group * a.W;
  const int64_t step = (int64_t)gridDim.y * 256;
  for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < n * row_chunks; i += step) {
    const int64_t slot = (first + i / row_chunks) % a.C;
    const int piece = (int)(i % row_chunks);
    const int64_t off = seq0 * a.seq_bytes + head * a.head_bytes + (slot * row_chunks + piece) * 16;
    u32x4_t kk[MW], vv[MW];
#pragma unroll
    for (int w = 0; w < MW; w++) {
      kk[w] = vv[w] = u32x4_t{0u, 0u, 0u, 0u};
      if (from[w] >= 0) {  // uniform
        kk[w] = *(const u32x4_t*)(a.k + off + from[w] * a.seq_bytes);
        vv[w] = *(const u32x4_t*)(a.v + off + from[w] * a.seq_bytes);
      }
    }
    asm volatile("" ::: "memory");  // no store before the last load
#pragma unroll
    for (int w = 0; w < MW; w++)
      if (from[w] >= 0) {
        *(u32x4_t*)(a.k + off + w * a.seq_bytes) = kk[w];
        *(u32x4_t*)(a.v + off + w * a.seq_bytes) = vv[w];
      }
    if (head == 0 && piece == 0) {
      int32_t s[MW];
      int32_t* sp = a.sp + seq0 * a.C + slot;
#pragma unroll
      for (int w = 0; w < MW; w++) s[w] = sp[(int64_t)max(from[w], 0) * a.C];
      asm volatile("" ::: "memory");
#pragma unroll
      for (int w = 0; w < MW; w++)
        if (from[w] >= 0) sp[(int64_t)w * a.C] = s[w];
    }
  }
}

int launch_ring_reorder(mb_ctx* ctx, int layer0, int n_layers, int B, int W, const int32_t* parent,
                        const int32_t* from, const int32_t* to, int64_t max_rows) {
  const RingView ring = global_ring(ctx, layer0);
  const int64_t e = kv_elem_bytes(ctx);
  ReorderIn a;
  a.k = (char*)ring.k;
  a.v = (char*)ring.v;
  a.sp = ring.sp;
  a.seq_bytes = ring.seq_stride * e;
  a.head_bytes = (int64_t)ring.C * HD * e;
  a.max_seqs = ctx->cfg.max_seqs;
  a.groups = B / W;
  a.W = W;
  a.C = ring.C;
  a.wrap = ring.wrap;
  a.parent = parent;
  a.from = from;
  a.to = to;
  const int row_chunks = (int)(HD * e / 16);
  const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(max_rows, ring.C));
  const int64_t bx = (int64_t)n_layers * a.groups * H;
  const int64_t by = std::min<int64_t>(65535, (rows * row_chunks + 255) / 256);
  if (bx > INT32_MAX) return fail(ctx, MB_ERR_ARG, "too many rings in one call");
  const dim3 grid((unsigned)bx, (unsigned)by);
  auto go = [&](auto mw) {
    hipLaunchKernelGGL(k_ring_reorder<decltype(mw)::value>, grid, dim3(256), 0, ctx->stream, a, row_chunks);
  };
  if (W <= 2) go(std::integral_constant<int, 2>{});
  else if (W <= 4) go(std::integral_constant<int, 4>{});
  else if (W <= 8) go(std::integral_constant<int, 8>{});
  else if (W <= 16) go(std::integral_constant<int, 16>{});
  else go(std::integral_constant<int, 32>{});
  MB_HIP(ctx, hipGetLastError());
  return MB_OK;
}

}  // namespace mb
