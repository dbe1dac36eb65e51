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
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, (uint64_t)dpp_u32<CTRL>((uint32_t)(u >> 32)) << 32 | dpp_u32<CTRL>((uint32_t)u));
}
__device__ __forceinline__ double wave_sum(double x) {
  x += dpp_f64<0xB1>(x);
  x += dpp_f64<0x4E>(x);
  x += dpp_f64<0x141>(x);
  x += dpp_f64<0x140>(x);
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Integers in the order of the floats (-0 as 0), above 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t order_of(double c) {
  const uint64_t u = __builtin_bit_cast(uint64_t, c + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// Raises lo, which at_lo >= n of some keys reach, until hardly more than n do, by
// the counts of keys that reach WAYS - 1 bounds between lo and hi (which no key
// exceeds).  count(bound) is uniform.  (A step is a chain of compare, count and
// branch of some 300 cycles whatever WAYS is, so few steps of many bounds.)
constexpr int kSlack = 8;
template <int WAYS, class Count>
__device__ __forceinline__ void raise(uint32_t& lo, int& at_lo, uint32_t hi, int n, Count count) {
  while (at_lo > n + kSlack && lo < hi) {
    const uint32_t step = (hi - lo) / WAYS + 1, from = lo;
    uint32_t k = 0;
#pragma unroll
    for (int w = 1; w < WAYS; w++) {
      const int c = count(from + w * step);
      if (c >= n) {
        k = w;
        at_lo = c;
      }
    }
    lo = from + k * step;
    hi = min(hi, lo + step - 1);
  }
}
// Lanes of `who` below this one.
__device__ __forceinline__ int rank_in(uint64_t who) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
}
// The rank of the lane's key among the 64 in LDS, of which the first `count` may
// be other than 0, the lower lane first on equal ones (UNIQUE: there are none).
// Read back as broadcasts, 8 at a time: some 20 cycles a key, where reading lanes
// into scalar registers took 75.
template <bool UNIQUE>
__device__ __forceinline__ int rank_of(const uint64_t* keys, uint64_t key, int count, int lane) {
  int r = 0;
  for (int k0 = 0; k0 < count; k0 += 8) {  // uniform
    ulonglong2 o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = ((const ulonglong2*)(keys + k0))[i];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint64_t k = i & 1 ? o[i >> 1].y : o[i >> 1].x;
      r += k > key || (!UNIQUE && k == key && k0 + i < lane);
    }
  }
  return r;
}
// LDS accesses of one wave before and after this one stay in their order.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
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

// Merge 16 values a lane into the list.  A bound that n lanes' best values reach
// leaves hardly more than n values; with the list's they are collected in LDS,
// one to a lane, and ranked by counting.  Where more than 64 reach it the bound is
// raised by counting values instead of lanes, and where that does not help
// (equal values) the list is taken in n rounds of the wave's best.
template <class Id>
__device__ __forceinline__ void take_top(float (&z)[16], Id id, int n, int lane, uint64_t* buf, RowTop& t) {
  auto key_of = [](float v, uint32_t id) { return (uint64_t)order_of(v) << 32 | ~id; };
  float best = z[0];
#pragma unroll
  for (int j = 1; j < 16; j++) best = fmaxf(best, z[j]);
  const bool mine = lane < n && t.id != kNoId;
  const int listed = __popcll(__ballot(mine));
  const uint32_t top = order_of(best), held = mine ? order_of(t.v) : 0u;
  // values up to the list's last can not enter a full list
  uint32_t lo = 1 + (listed == n ? (uint32_t)__builtin_amdgcn_readlane((int)held, n - 1) : order_of(-INFINITY));
  const uint32_t hi = wave_umax(top);
  if (hi < lo) return;  // uniform: nothing enters the list
  int at_lo = __popcll(__ballot(top >= lo));
  bool whole = at_lo < n;  // too few for a bound: every value that may enter
  if (!whole) {
    lo = wave_min(top >= lo ? top : ~0u);  // (the values in use span few of the keys)
    raise<8>(lo, at_lo, hi, n, [&](uint32_t k) { return __popcll(__ballot(top >= k)); });
  }
  int count = 0, all = 0;
  for (int pass = 0; pass < 2; pass++) {
    const float bound = value_of(lo);
    count = 0;
#pragma unroll
    for (int j = 0; j < 16; j++) {
      // (every lane stores, what is not taken to place 64: no branches)
      const bool in = z[j] >= bound;
      const uint64_t who = __ballot(in);
      buf[in ? min(count + rank_in(who), 64) : 64] = key_of(z[j], id(j));
      count += __popcll(who);
    }
    const bool in = mine && (whole || held >= lo);
    const uint64_t who = __ballot(in);
    buf[in ? min(count + rank_in(who), 64) : 64] = key_of(t.v, t.id);
    all = count + __popcll(who);
    if (all <= 64 || pass) break;  // uniform
    const uint32_t first = (uint32_t)__builtin_amdgcn_readfirstlane((int)held);  // the list's best
    whole = false;
    at_lo = all;
    if (at_lo > n)
      raise<2>(lo, at_lo, max(hi, first), n, [&](uint32_t k) {
        const float v = value_of(k);
        int c = __popcll(__ballot(held >= k));
#pragma unroll
        for (int j = 0; j < 16; j++) c += __popcll(__ballot(z[j] >= v));
        return c;
      });
  }
  if (all <= 64) {  // uniform
    wave_order();
    if (lane >= all) buf[lane] = 0ull;
    wave_order();
    uint64_t key = buf[lane];
    const int r = rank_of<true>(buf, key, all, lane);
    wave_order();
    if (lane < all && r < n) buf[r] = key;
    wave_order();
    key = buf[lane];
    wave_order();
    const bool some = lane < min(n, all);
    t.v = some ? value_of((uint32_t)(key >> 32)) : -INFINITY;
    t.id = some ? ~(uint32_t)key : kNoId;
    return;
  }
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
    const uint32_t win = wave_min(bv == top ? bi : kNoId);
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
                                         int hi, int n, int lane, uint64_t* buf, RowTop& t) {
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
      const double by = 1.0 / (double)penalty;
#pragma unroll
      for (int q = 0; q < 16 / PER; q++) {
        const int at = (int)id(q * PER);
        const uint32_t bits = at < hi ? seen[at >> 5] >> (at & 31) : 0u;
#pragma unroll
        for (int e = 0; e < PER; e++) {
          // (the double product rounds once to the fp32 product, and with the
          // reciprocal to the fp32 quotient: no quotient of two floats is
          // within 2^-50 of the middle between two normal floats)
          float& x = z[q * PER + e];
          const float y = (float)((double)x * (x < 0.f ? (double)penalty : by));
          x = (bits >> e) & 1 ? y : x;
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
    if (t.m < INFINITY) {  // uniform
#pragma unroll
      for (int j = 0; j < 16; j++) p[j] = __expf(z[j] - t.m);
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++) p[j] = z[j] == t.m ? 1.f : 0.f;
    }
#pragma unroll
    for (int w = 8; w > 0; w >>= 1)
#pragma unroll
      for (int j = 0; j < w; j++) p[j] += p[j + w];
    t.sum += (double)p[0];
    if (mx > least) {
      take_top(z, id, n, lane, buf, t);
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
  int chunks, chunk;   // parts of a row in the workspace, ids of a part
  int parts;           // parts of a row within its voice's workgroup (chunks 1)
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

__device__ __forceinline__ void scan(const BeamIn& a, int64_t row, int lo, int hi, int lane, uint64_t* buf,
                                     RowTop& t) {
  const char* p = (const char*)a.logits + row * a.stride * (a.bf16 ? 2 : 4);
  const uint32_t* seen = a.seen ? a.seen + row * a.words : nullptr;
  if (a.bf16) scan_row<true>(p, seen, a.penalty, lo, hi, a.n, lane, buf, t);
  else scan_row<false>(p, seen, a.penalty, lo, hi, a.n, lane, buf, t);
  t.sum = wave_sum(t.sum);
}

// What a part holds whose row is not looked at.
__device__ __forceinline__ void part_empty(const BeamIn& a, int64_t row, int chunk, int lane) {
  char* p = part_row(a, row, chunk);
  if (lane == 0) *(PartRow*)p = PartRow{0.0, -INFINITY, 0u};
  if (lane < a.n) ((uint2*)(p + sizeof(PartRow)))[lane] = make_uint2(__float_as_uint(-INFINITY), kNoId);
}

// A wave per part of a row.  16 voices x 8 beams x 32000 fp32 ids, 16 chosen (16.4 MB): 9.1
// us, where reading them takes 2.4: four waves a SIMD, each one part, whose
// exponentials, bound and list are some 4000 cycles of vector instructions in
// one chain (with n rounds of the wave's best instead of the bound and the ranks,
// here and in the choice, the two launches took 56 us, not 19).
__global__ __launch_bounds__(256) void k_beam_scan(const BeamIn a, int64_t parts) {
  __shared__ __align__(16) uint64_t buf[4][66];
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= parts) return;
  const int64_t row = i / a.chunks;
  const int c = (int)(i % a.chunks);
  if (a.done && a.done[row]) {  // its logits are not looked at
    part_empty(a, row, c, lane);
    return;
  }
  RowTop t;
  scan(a, row, c * a.chunk, min(a.V, (c + 1) * a.chunk), lane, buf[threadIdx.x >> 6], t);
  char* p = part_row(a, row, c);
  if (lane == 0) *(PartRow*)p = PartRow{t.sum, t.m, 0u};
  if (lane < a.n) ((uint2*)(p + sizeof(PartRow)))[lane] = make_uint2(__float_as_uint(t.v), t.id);
}

// The maximum and sum of a row's parts, one to a lane (h.m = -inf elsewhere).
__device__ __forceinline__ void join_sums(const PartRow& h, RowTop& t) {
  t.m = wave_max(h.m);
  // (an infinite maximum is the maximum of a part only where it was reached)
  const double by = h.m == t.m ? 1.0 : (double)__expf(h.m - t.m);
  t.sum = wave_sum(h.sum * by);
}
// The parts of a row joined.  Everything is read before anything is used.
__device__ __forceinline__ void join(const BeamIn& a, int64_t row, int lane, uint64_t* buf, RowTop& t) {
  PartRow h{0.0, -INFINITY, 0u};
  if (lane < a.chunks) h = *(const PartRow*)part_row(a, row, lane);
  const int all = a.chunks * a.n;
  const uint32_t per = (1u << 20) / a.n + 1;  // i / n as a product: i < 2^11, n <= 2^5
  for (int base = 0; base < all; base += kScan) {
    float z[16];
    uint32_t ids[16];
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const int i = base + 64 * j + lane;
      uint2 w = make_uint2(__float_as_uint(-INFINITY), kNoId);
      if (i < all) {
        const int c = (int)(i * per >> 20);
        w = ((const uint2*)(part_row(a, row, c) + sizeof(PartRow)))[i - c * a.n];
      }
      z[j] = __uint_as_float(w.x);
      ids[j] = w.y;
    }
    take_top(z, [&](int j) { return ids[j]; }, a.n, lane, buf, t);
  }
  join_sums(h, t);
}

// The n best of `all` <= 64 J keys in LDS, the lower index first on equal ones,
// as take_top finds a row's: lane k returns the k-th's index, or -1.
template <int J>
__device__ __forceinline__ int best_of(uint64_t* lk, int all, int n, int lane, uint64_t* buf, int32_t* at64) {
  int count, i = lane;
  if (J == 1) {
    count = all;
  } else {
    uint32_t hk[J], top = 0u;  // the keys' upper words
#pragma unroll
    for (int j = 0; j < J; j++) {
      const int at = 64 * j + lane;
      hk[j] = at < all ? (uint32_t)(lk[at] >> 32) : 0u;
      top = max(top, hk[j]);
    }
    auto reach = [&](uint32_t k) {
      int c = 0;
#pragma unroll
      for (int j = 0; j < J; j++) c += __popcll(__ballot(hk[j] >= k));
      return c;
    };
    uint32_t least = ~0u;
#pragma unroll
    for (int j = 0; j < J; j++) least = min(least, hk[j] ? hk[j] : ~0u);
    const uint32_t hi = wave_umax(top);
    uint32_t lo = max(1u, min(hi, wave_min(least)));
    count = reach(lo);
    raise<4>(lo, count, hi, n, reach);
    int at = 0;
#pragma unroll
    for (int j = 0; j < J; j++) {
      const bool in = hk[j] >= lo;
      const uint64_t who = __ballot(in);
      at64[in ? min(at + rank_in(who), 64) : 64] = 64 * j + lane;  // in the index's order
      at += __popcll(who);
    }
    wave_order();
    if (lane < min(count, 64)) i = at64[lane];
  }
  int mine = -1;
  if (count <= 64) {  // uniform
    const uint64_t k = lane < count ? lk[i] : 0ull;
    buf[lane] = k;
    wave_order();
    const int r = rank_of<false>(buf, k, count, lane);
    if (lane < n) at64[lane] = -1;
    wave_order();
    if (k && r < n) at64[r] = i;
    wave_order();
    if (lane < n) mine = at64[lane];
    return mine;
  }
  for (int r = 0; r < n; r++) {  // many equal keys: n rounds of the wave's best
    uint64_t bk = 0ull;
    uint32_t bi = kNoId;
    for (int at = lane; at < all; at += 64)
      if (lk[at] > bk) {
        bk = lk[at];
        bi = at;
      }
    const uint32_t hi = wave_umax((uint32_t)(bk >> 32));
    if (hi == 0u) break;
    const uint32_t low = wave_umax((uint32_t)(bk >> 32) == hi ? (uint32_t)bk : 0u);
    const uint32_t win = wave_min((uint32_t)(bk >> 32) == hi && (uint32_t)bk == low ? bi : kNoId);
    if (lane == r) mine = (int)win;
    wave_order();
    if (bi == win) lk[bi] = 0ull;
    wave_order();
  }
  return mine;
}

// One workgroup per voice, its waves taking the beams' rows in turn; then the
// first wave takes the n best of the W n candidates by c.  On equal c the lower
// beam goes first and, within a beam, the list's order holds.
// A chain that one workgroup a voice walks: 1 voice x 4 beams x 1024 ids 6.1 us, 64 x 8 x
// 1024 with a penalty 9.4 (2 MB of logits), the join of 16 x 8 rows in 32 parts of 16
// ids 11.3; the ranks by counting instead of rounds took 9.2 us to 5.3 and 17.5 to 8.6,
// calls of the first two.
constexpr int kBeamWaves = 16;
template <bool FUSED>
__global__ __launch_bounds__(64 * kBeamWaves) void k_beam_pick(const BeamIn a) {
  __shared__ float lv[kBeamMax * kBeamMax];
  __shared__ uint32_t li[kBeamMax * kBeamMax];
  __shared__ float lm[kBeamMax];
  __shared__ double ls[kBeamMax], sc[kBeamMax];
  __shared__ uint64_t lk[kBeamMax * kBeamMax];
  __shared__ int32_t from[kBeamMax], tok[kBeamMax], at64[65];
  __shared__ __align__(16) uint64_t buf[kBeamWaves][66];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int b = blockIdx.x, n = a.n;
  auto put = [&](int at, const RowTop& t) {
    if (lane < n) {
      lv[at * n + lane] = t.v;
      li[at * n + lane] = t.id;
    }
  };
  auto finish = [&](int w, RowTop& t, float score, bool ended) {
    if (ended) {  // as a row of one id, whose logarithm is 0
      t.m = 0.f;
      t.sum = 1.0;
      t.v = lane == 0 ? 0.f : -INFINITY;
      t.id = lane == 0 ? (uint32_t)a.end_id : kNoId;
    }
    put(w, t);
    if (lane == 0) {
      lm[w] = t.m;
      ls[w] = log(t.sum);
      sc[w] = (double)score;
    }
  };
  // (a row is read whether its beam has ended or not: waiting for the flag would
  // cost every row a trip to memory)
  if (FUSED && a.parts > 1) {  // W parts <= kBeamWaves: a wave for each part
    const int w = wave / a.parts, part = wave - w * a.parts;
    const int64_t row = (int64_t)b * a.W + w, mine = (int64_t)b * a.W + min(wave, a.W - 1);
    const float score = a.scores[mine];
    const bool ended = a.done && a.done[mine];
    RowTop t;
    scan(a, row, part * a.chunk, min(a.V, (part + 1) * a.chunk), lane, buf[wave], t);
    put(wave, t);
    if (lane == 0) {
      lm[wave] = t.m;
      ls[wave] = t.sum;
    }
    __syncthreads();
    // wave w < W joins row w's parts
    const int all = a.parts * n;  // <= 512
    PartRow h{0.0, -INFINITY, 0u};
    float z[16];
    uint32_t ids[16];
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const int i = 64 * j + lane;
      const bool in = j < 8 && i < all && wave < a.W;
      z[j] = in ? lv[wave * all + i] : -INFINITY;
      ids[j] = in ? li[wave * all + i] : kNoId;
    }
    if (wave < a.W && lane < a.parts) {
      h.m = lm[wave * a.parts + lane];
      h.sum = ls[wave * a.parts + lane];
    }
    __syncthreads();
    if (wave < a.W) {
      t = RowTop{};
      take_top(z, [&](int j) { return ids[j]; }, n, lane, buf[wave], t);
      join_sums(h, t);
      finish(wave, t, score, ended);
    }
  } else {
    for (int w = wave; w < a.W; w += nw) {
      const int64_t row = (int64_t)b * a.W + w;
      const float score = a.scores[row];
      const bool ended = a.done && a.done[row];
      RowTop t;
      if (FUSED) scan(a, row, 0, a.V, lane, buf[wave], t);
      else join(a, row, lane, buf[wave], t);
      finish(w, t, score, ended);
    }
  }
  __syncthreads();
  // c of every candidate, as a key (0: none)
  const int all = a.W * n;
  const uint32_t per = 65536 / n + 1;  // i / n as a product: i < 1024, n <= 32
  for (int i = threadIdx.x; i < all; i += blockDim.x) {
    const int w = (int)(i * per >> 16);
    const float v = lv[i], m = lm[w];
    const double c = sc[w] + ((v == m ? 0.0 : (double)v - (double)m) - ls[w]);
    lk[i] = li[i] != kNoId && c > -INFINITY ? order_of(c) : 0ull;
  }
  __syncthreads();
  if (wave == 0) {
    int mine;  // the candidate that lane k's output is
    if (all <= 64) mine = best_of<1>(lk, all, n, lane, buf[0], at64);  // uniform
    else if (all <= 128) mine = best_of<2>(lk, all, n, lane, buf[0], at64);
    else if (all <= 256) mine = best_of<4>(lk, all, n, lane, buf[0], at64);
    else mine = best_of<16>(lk, all, n, lane, buf[0], at64);
    if (lane < n) {
      const int64_t o = (int64_t)b * n + lane;
      const int w = mine < 0 ? -1 : (int)(mine * per >> 16);
      const int32_t id = mine < 0 ? -1 : (int32_t)li[mine];
      float score = -INFINITY;
      if (mine >= 0) {
        const float v = lv[mine], m = lm[w];
        score = (float)(sc[w] + ((v == m ? 0.0 : (double)v - (double)m) - ls[w]));
      }
      a.scores_out[o] = score;
      a.parent[o] = w;
      a.token[o] = id;
      if (a.done_out) a.done_out[o] = w < 0 || (a.end_id >= 0 && id == a.end_id);
      from[lane] = w;
      tok[lane] = id;
    }
  }
  if (!a.seen_out) return;
  __syncthreads();
  // every chosen beam's history: its parent's and the chosen id
  for (int k = wave; k < n; k += nw) {
    const int w = from[k], v = tok[k];
    const uint32_t* src = a.seen + ((int64_t)b * a.W + max(w, 0)) * a.words;
    uint32_t* dst = a.seen_out + ((int64_t)b * n + k) * a.words;
    for (int j = lane; j < a.words; j += 64) {
      uint32_t bits = w >= 0 ? src[j] : 0u;
      if (w >= 0 && v >> 5 == j) bits |= 1u << (v & 31);
      dst[j] = bits;
    }
  }
}

// How a row is cut.  One launch, a workgroup per voice, where its waves can read
// every row's 1024 ids at a time side by side (`parts` waves a row); else a scan by
// a wave per part of a row, and the choice in a second launch.  (Rows of 2477, 3383
// and 5489 ids of 14, 2 and 2 beams read by one wave each took 21.0, 12.8 and, in two
// launches, 11.1 us.)
static void beam_parts(int W, int V, int& chunks, int& chunk, int& parts) {
  const int reads = (V + kScan - 1) / kScan;
  chunks = parts = 1;
  chunk = V;
  if (reads == 1) return;
  if ((int64_t)W * reads <= kBeamWaves) {
    parts = reads;
    chunk = kScan;
    return;
  }
  chunk = (V + 64 * kScan - 1) / (64 * kScan) * kScan;
  chunks = (V + chunk - 1) / chunk;
}

int64_t beam_work_bytes(int B, int W, int V, int n) {
  int chunks, chunk, parts;
  beam_parts(W, V, chunks, chunk, parts);
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
  beam_parts(W, V, a.chunks, a.chunk, a.parts);
  // (a grid's work-items are counted in 32 bits)
  if (((int64_t)B * W * a.chunks + 3) / 4 > INT32_MAX / 256 || (int64_t)B * 64 * kBeamWaves > INT32_MAX)
    return fail(ctx, MB_ERR_ARG, "too many rows in one call");
  const dim3 block(64 * std::min(W * a.parts, kBeamWaves));
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
// 32 voices x 4 beams x 12 layers, 300 bf16 rows each (1.5 GB read and written): 290
// us, 5.2 TB/s, where a copy of 2 GiB reaches 4.87.
template <int MW>
__global__ __launch_bounds__(256) void k_ring_reorder(const ReorderIn a, int chunk_bits) {
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
  // (a row is 8 or 16 pieces, a head's run at most 2^28 bytes)
  const uint32_t at0 = (uint32_t)first % (uint32_t)a.C, pieces = n > 0 ? (uint32_t)n << chunk_bits : 0u;
  for (uint32_t i = blockIdx.y * 256 + threadIdx.x; i < pieces; i += gridDim.y * 256) {
    uint32_t slot = at0 + (i >> chunk_bits);
    if (slot >= (uint32_t)a.C) slot -= a.C;
    const uint32_t piece = i & ((1u << chunk_bits) - 1);
    const int64_t off = seq0 * a.seq_bytes + head * a.head_bytes + (((slot << chunk_bits) + piece) << 4);
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
  const int chunk_bits = e == 2 ? 3 : 4, row_chunks = 1 << chunk_bits;  // 16-byte pieces of a row
  const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(max_rows, ring.C));
  const int64_t bx = (int64_t)n_layers * a.groups * H;
  const int64_t by = std::min<int64_t>(65535, (rows * row_chunks + 255) / 256);
  if (bx > INT32_MAX / 256) return fail(ctx, MB_ERR_ARG, "too many rings in one call");
  const dim3 grid((unsigned)bx, (unsigned)by);
  auto go = [&](auto mw) {
    hipLaunchKernelGGL(k_ring_reorder<decltype(mw)::value>, grid, dim3(256), 0, ctx->stream, a, chunk_bits);
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
