// Token sampling with temperature, top-k, top-p and min-p from given random numbers (sm_100a).
//
// The weights are w = exp((l - max) / T).  In the order (logit falling, index rising) each
// filter keeps a head, so the kept tokens are the first n of that order and the sampled one is
// the first whose running sum exceeds u times the sum of those n.  A decision of either kind
// compares long sums, and one token's weight may be 1e-7 of them, so sums and weights are f64.
//
// No sort: 16-bit logits take at most 65536 values, and equal logits have equal weights.  A row
// is counted into a histogram over the logits' bits, in integers, so nothing depends on the order
// of atomics; a weight is then computed once per value that occurs (a few thousand of 1e5
// tokens), and every sum over tokens is a sum over values of count * weight.  The sampled value
// and its ordinal among equals known, one more pass over the row (from L2) finds the ordinal-th
// token with these bits.
//
// One cluster of up to eight CTAs per row.  A CTA holds a histogram of its slice of the row as
// 65536 16-bit counters (128 KB): word m counts the logits of magnitude m, all of them in its low
// half and the negative ones in its high half.  A slice of more tokens than a counter holds is
// counted in rounds: the counts that the atomics return tell whether one passed half of the range
// in a round, and then values counted 2048 times or more give all but one of their count to a list
// (one value in 2048 tokens at most gets there).
// So counting needs no reordering of the bits: the address is the magnitude, the increment 1 or
// 0x10001 (about three instructions of the half-rate integer pipe per token, which bounds it).  The values are taken in blocks of 64;
// block i, 0 <= i < 1024, is the i-th from the top (512 of falling positive, then 512 of rising
// negative magnitude).  Each CTA notes which blocks occur, the cluster's warps share out those
// that do, add the counters of its CTAs up over distributed shared memory and leave (count, mass)
// with CTA 0, which scans the blocks and whose first warp looks into the (at most four) blocks
// where a filter or the sample falls, and tells the CTA whose slice holds the token.
//
// Measured: 16 rows of 128256 15.9 us, one row of 32003 f16 logits 16.8 us, 192 rows of 152064, half
// of them masked, 73 us (0.12 of the measured copy rate for its 58 MB; 4 more with the counters looked
// through after every round).
// What bounds it: for few rows latency (three cluster barriers and the chain of searches, most
// of it code that runs once); for many rows counting, its instructions and one shared-memory
// atomic per token.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstddef>
#include <type_traits>

#include "common.cuh"
#include "pick.cuh"
#include "tma.cuh"

namespace cg = cooperative_groups;

namespace tq {
namespace sm {
constexpr int THREADS = 1024;
constexpr int WARPS = THREADS / 32;
constexpr int WORDS = 32768;           // magnitudes
constexpr int BLOCKS = 1024;           // of 64 values
constexpr int ROUND = 8 * THREADS;     // lines of 8 logits looked at together
constexpr int SHORT_ROUND = 4088;      // or, where rounds follow: what fits above half of a counter's range
constexpr int KEEP = 2048;             // a value's count from which all but one leave when some count passed half of the range
constexpr int MAX_VOCAB = 1 << 20;
constexpr int SPILLS = MAX_VOCAB / (KEEP - 1) + 8;
constexpr int MAX_CTAS = 8;
constexpr int CARDS = 64;              // blocks whose weights are kept for the searches
}  // namespace sm

// A block's values as one warp computed them, for the searches: lane l has the values 2 l and
// 2 l + 1 of the falling order.
struct BlockCard {
  double w[2][32];
  double before[32];  // mass of the block before the lane's first value
  uint32_t cnt[2][32];
};

struct SampleShared {
  uint32_t hist[sm::WORDS];
  BlockCard card[sm::CARDS];  // CTA 0: of the blocks of the largest magnitudes that occur
  // CTA 0, of the whole row: first each block's mass and count, then those before it
  double mass[sm::BLOCKS];
  uint32_t count[sm::BLOCKS];
  double red_m[32];
  uint32_t red_c[32];
  uint16_t card_of[sm::BLOCKS];  // CTA 0: a block's card (CARDS: none kept)
  double w, kept;            // of the sampled value, and the kept mass
  uint32_t spill_bits[sm::SPILLS], spill_count[sm::SPILLS];  // counts taken out of the histogram
  uint32_t spills;           // entries of this CTA's list
  uint32_t spilled;          // whether any CTA of the row has one
  uint32_t masked[2][32];    // by lane: logits that are -inf, and that are the type's lowest value
  uint32_t occur[32];        // which blocks of 64 magnitudes the row has, 16 positive and 16 negative ones an entry
  uint32_t top;              // order of the row's largest logit (see order_of; 0: nothing there)
  float temperature, top_p, min_p, u;  // the row's
  int top_k;
  int owner;                 // rank of the CTA that holds the sampled token
  uint32_t bits, ordinal;    // its bits and its place among this CTA's equals
};

template <int XT>
struct Bits {
  static constexpr uint32_t INF = XT == TQ_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  static constexpr uint32_t LOWEST = XT == TQ_DTYPE_BF16 ? 0xff7fu : 0xfbffu;  // the type's lowest value
};

// An order-preserving number of a logit's bits (-0 given as +0), never 0.
__device__ __forceinline__ uint32_t order_of(uint32_t b) { return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u); }
__device__ __forceinline__ uint32_t bits_of(uint32_t order) {
  return (order & 0x8000u) ? (order & 0x7fffu) : (~order & 0xffffu);
}

// Logits of one sign in a histogram word.  (Before words are read, those of NaN are cleared and -0
// counts as +0; -inf was never counted.)
__device__ __forceinline__ uint32_t count_in(uint32_t w, bool negative) {
  return negative ? w >> 16 : (w & 0xffffu) - (w >> 16);
}

// What a CTA's list holds of a value.
__device__ __forceinline__ uint32_t spilled_of(const SampleShared* o, uint32_t bits) {
  uint32_t c = 0u;
  for (uint32_t k = 0; k < o->spills; ++k)
    if (o->spill_bits[k] == bits) c += o->spill_count[k];
  return c;
}

// What a row's weights are computed from.
struct RowScale {
  uint32_t top_bits;  // the largest logit
  double vmax, inv_t;
  bool spike;         // only the largest value weighs (temperature <= 0, or the largest is +inf)
};

template <int XT>
__device__ __forceinline__ double weight_of(uint32_t bits, const RowScale& r) {
  if (bits == r.top_bits) return 1.0;
  return r.spike ? 0.0 : exp(((double)h2f((uint16_t)bits, XT) - r.vmax) * r.inv_t);
}

// Exclusive running sums over the block (thread order) of a count and a mass.
__device__ __forceinline__ void scan_pair(uint32_t& c, double& m, SampleShared& s, uint32_t& total_c, double& total_m) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t xc = c;
  double xm = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t yc = __shfl_up_sync(0xffffffffu, xc, o);
    const double ym = __shfl_up_sync(0xffffffffu, xm, o);
    if (lane >= o) {
      xc += yc;
      xm += ym;
    }
  }
  double em = __shfl_up_sync(0xffffffffu, xm, 1);  // not xm - m: masses differ by 300 orders
  if (lane == 0) em = 0.0;
  if (lane == 31) {
    s.red_c[warp] = xc;
    s.red_m[warp] = xm;
  }
  __syncthreads();
  uint32_t wc = s.red_c[lane];
  double wm = s.red_m[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t yc = __shfl_up_sync(0xffffffffu, wc, o);
    const double ym = __shfl_up_sync(0xffffffffu, wm, o);
    if (lane >= o) {
      wc += yc;
      wm += ym;
    }
  }
  total_c = __shfl_sync(0xffffffffu, wc, 31);
  total_m = __shfl_sync(0xffffffffu, wm, 31);
  const uint32_t bc = __shfl_sync(0xffffffffu, wc, (warp + 31) & 31);
  const double bm = __shfl_sync(0xffffffffu, wm, (warp + 31) & 31);
  c = xc - c + (warp ? bc : 0u);
  m = em + (warp ? bm : 0.0);
}

// The 8 logits from index `first` on (a 16-byte line of memory); those outside [lo, hi) come as NaN.
// Lines that cross an end are read value by value.
__device__ __noinline__ uint4 load_ragged_line(const uint16_t* row, int64_t first, int64_t lo, int64_t hi) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = 0x7fff7fffu;
    const int64_t j = first + 2 * e;
    if (j >= lo && j < hi) w[e] = (w[e] & 0xffff0000u) | row[j];
    if (j + 1 >= lo && j + 1 < hi) w[e] = (w[e] & 0xffffu) | ((uint32_t)row[j + 1] << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 load_line(const uint16_t* row, int64_t first, int64_t lo, int64_t hi) {
  if (first >= lo && first + 8 <= hi) return *reinterpret_cast<const uint4*>(row + first);
  return load_ragged_line(row, first, lo, hi);
}

// One warp's view of block i, lane order falling (lane 0 has the largest two values), with the
// counts of the whole row.
struct BlockView {
  uint32_t bits[2], cnt[2];
  double w[2];
  double before;  // mass of the block before the lane's first value
};

__device__ __forceinline__ void name_values(BlockView& v, int i) {
  const int lane = threadIdx.x & 31;
  const bool negative = i >= sm::BLOCKS / 2;
  const int m = negative ? (i - sm::BLOCKS / 2) * 64 + 2 * lane : (sm::BLOCKS / 2 - 1 - i) * 64 + 63 - 2 * lane;
  v.bits[0] = negative ? 0x8000u | (uint32_t)m : (uint32_t)m;
  v.bits[1] = negative ? v.bits[0] + 1 : v.bits[0] - 1;
}

// Counts from the cluster's histograms, weights, and the running mass; returns the block's mass.
template <int XT>
__device__ __forceinline__ double view_block(BlockView& v, SampleShared& s, int i, int ctas, const RowScale& r) {
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31;
  name_values(v, i);
  const bool negative = v.bits[0] & 0x8000u;
  const uint32_t m0 = v.bits[0] & 0x7fffu, m1 = v.bits[1] & 0x7fffu;
  v.cnt[0] = v.cnt[1] = 0u;
  auto gather = [&](auto many) {  // the words of up to `many` CTAs, their loads in flight together
    constexpr int MANY = decltype(many)::value;
    uint2 x[MANY];
#pragma unroll
    for (int c = 0; c < MANY; ++c) {
      x[c] = make_uint2(0u, 0u);
      if (c < ctas) x[c] = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(s.hist, c) + min(m0, m1));
    }
#pragma unroll
    for (int c = 0; c < MANY; ++c) {
      v.cnt[0] += count_in(negative ? x[c].x : x[c].y, negative);
      v.cnt[1] += count_in(negative ? x[c].y : x[c].x, negative);
    }
  };
  if (ctas <= 2)
    gather(std::integral_constant<int, 2>());
  else
    gather(std::integral_constant<int, sm::MAX_CTAS>());
  if (s.spilled)
    for (int c = 0; c < ctas; ++c) {
      const SampleShared* o = cluster.map_shared_rank(&s, c);
      v.cnt[0] += spilled_of(o, v.bits[0]);
      v.cnt[1] += spilled_of(o, v.bits[1]);
    }
  v.w[0] = v.w[1] = 0.0;
  if (v.cnt[0] | v.cnt[1]) {  // both at once: the two chains overlap
    v.w[0] = weight_of<XT>(v.bits[0], r);
    v.w[1] = weight_of<XT>(v.bits[1], r);
    if (!v.cnt[0]) v.w[0] = 0.0;
    if (!v.cnt[1]) v.w[1] = 0.0;
  }
  double xm = v.cnt[0] * v.w[0] + v.cnt[1] * v.w[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double ym = __shfl_up_sync(0xffffffffu, xm, o);
    if (lane >= o) xm += ym;
  }
  v.before = __shfl_up_sync(0xffffffffu, xm, 1);
  if (lane == 0) v.before = 0.0;
  return __shfl_sync(0xffffffffu, xm, 31);
}

// The last i in [0, 1024) for which `holds`, which is true up to some place; all lanes agree.
template <class F>
__device__ __forceinline__ int last_block(F holds) {
  const int lane = threadIdx.x & 31;
  const uint32_t coarse = __ballot_sync(0xffffffffu, holds(32 * lane));
  const int c = max(31 - __clz((int)coarse), 0);
  const uint32_t fine = __ballot_sync(0xffffffffu, holds(32 * c + lane));
  return 32 * c + max(31 - __clz((int)fine), 0);
}

// One warp: where the filters cut the order, and which value and ordinal the sample falls on.
// s.count / s.mass hold the tokens and mass before the i-th block.  One loop over the four
// searches, so that their common code (a double exp among it) is there once.
template <int XT>
__device__ __forceinline__ void pick(cg::cluster_group& cluster, SampleShared& s, int ctas, const RowScale& scale, bool greedy, uint32_t all_c, double all_m) {
  using namespace sm;
  const int lane = threadIdx.x & 31;
  const int k = s.top_k;
  const double p = (double)s.top_p, mp = (double)s.min_p;
  const double u = s.u > 0.0f ? fmin((double)s.u, 1.0) : 0.0;  // NaN: 0
  const uint32_t want = greedy ? 1u : k > 0 ? (uint32_t)k : 0u;
  uint32_t n = all_c;  // the kept head and its mass
  double kept = all_m;
  uint32_t at_most = all_c;  // where the sample falls if no value of its block passes the goal
  uint32_t bits = scale.top_bits, ord = 0u;
  double w = 1.0;
  bool done = false;
  if (want == 1u) {
    n = 1u;
    kept = 1.0;
  }
  enum { TOP_K, TOP_P, MIN_P, SAMPLE, LAST };
#pragma unroll 1
  for (int what = TOP_K; what <= LAST; ++what) {
    double goal = 0.0;   // a mass to reach (TOP_P) or pass (SAMPLE)
    uint32_t nth = 0u;   // a token to find, from 1
    int i = 0;
    if (n == 1u) {
      if (what < SAMPLE) continue;
      break;  // the first token
    }
    if (what == TOP_K) {
      if (!want || want >= n) continue;
      nth = want;
    } else if (what == TOP_P) {
      if (!(p < 1.0)) continue;
      goal = p * kept;
      if (goal <= 1.0) {  // the first token, of weight 1, is enough
        n = 1u;
        kept = 1.0;
        continue;
      }
    } else if (what == MIN_P) {
      if (!(mp > 0.0)) continue;
    } else if (what == SAMPLE) {
      goal = u * kept;
    } else {
      if (done) break;
      nth = min(n, at_most);  // (n: u times the sum reached the sum by rounding)
    }
    if (nth)
      i = last_block([&](int j) { return s.count[j] < nth; });
    else if (what != MIN_P)
      i = last_block([&](int j) { return what == TOP_P ? s.mass[j] < goal : s.mass[j] <= goal; });
    else  // the last block whose first value weighs enough
#pragma unroll 1
      for (int apart = 32, first = 0; apart; apart >>= 5, first = i) {  // (last_block with one exp)
        const int j = first + apart * lane;
        const uint32_t b = j < BLOCKS / 2 ? (uint32_t)(BLOCKS / 2 - 1 - j) * 64 + 63 : 0x8000u | (uint32_t)(j - BLOCKS / 2) * 64;
        const double w = weight_of<XT>(bits_of(min(order_of(b), order_of(scale.top_bits))), scale);
        i = first + apart * max(31 - __clz((int)__ballot_sync(0xffffffffu, w >= mp)), 0);
      }
    BlockView v;
    const int card = s.card_of[i];
    if (card < CARDS) {
      name_values(v, i);
      const BlockCard& k = s.card[card];
      v.w[0] = k.w[0][lane];
      v.w[1] = k.w[1][lane];
      v.before = k.before[lane];
      v.cnt[0] = k.cnt[0][lane];
      v.cnt[1] = k.cnt[1][lane];
    } else {
      view_block<XT>(v, s, i, ctas, scale);
    }
    uint32_t before_c[2];
    {
      uint32_t x = v.cnt[0] + v.cnt[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      before_c[1] = s.count[i] + x - v.cnt[1];
      before_c[0] = before_c[1] - v.cnt[0];
    }
    const double before_m[2] = {s.mass[i] + v.before, s.mass[i] + (v.before + v.cnt[0] * v.w[0])};
    // the first lane and value where the search ends: tokens up to there (c) and their mass (m)
    bool hit = false;
    uint32_t c = 0u, hb = 0u, ho = 0u;
    double m = 0.0, hw = 0.0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t cnt = v.cnt[e];
      const double we = v.w[e], b0 = before_m[e], b1 = b0 + cnt * we;
      if (!cnt || hit) continue;
      uint32_t q = 0u;  // how many of these equals are in
      if (nth) {
        hit = before_c[e] < nth && nth <= before_c[e] + cnt;
        q = nth - before_c[e];
      } else if (what == MIN_P) {
        if (we >= mp) {  // counted up: the last one that passes decides
          c = before_c[e] + cnt;
          m = b1;
        }
      } else {
        // the smallest q in 1 .. cnt with b0 + q we >= goal (> goal for the sample): a quotient in 32
        // bits is off by less than one, and the sums decide
        const bool reach = what == TOP_P;
        hit = reach ? goal <= b1 : goal < b1;
        if (hit) {
          const float f = we > 1e-30 ? (float)(goal - b0) / (float)we : (float)((goal - b0) / we);
          q = (uint32_t)fminf(fmaxf(ceilf(f), 1.0f), (float)cnt);
          const double less = b0 + (double)(q - 1u) * we, here = b0 + (double)q * we;
          if (q > 1u && (reach ? less >= goal : less > goal))
            --q;
          else if (q < cnt && (reach ? here < goal : here <= goal))
            ++q;
        }
      }
      if (hit) {
        c = before_c[e] + q;
        m = b0 + (double)q * we;
        hb = v.bits[e];
        ho = q - 1u;
        hw = we;
      }
    }
    if (what == MIN_P) {
      const uint32_t any = __ballot_sync(0xffffffffu, c != 0u);
      const int l = max(31 - __clz((int)any), 0);
      c = any ? __shfl_sync(0xffffffffu, c, l) : s.count[i];
      m = any ? __shfl_sync(0xffffffffu, m, l) : s.mass[i];
      if (c < n) {
        n = max(c, 1u);  // the first token always stays
        kept = c ? m : 1.0;
      }
      continue;
    }
    const uint32_t who = __ballot_sync(0xffffffffu, hit);
    if (!who) {
      // The goal lies between two roundings of one sum: at or past the block's own, before the scan's for
      // the next block.  The last token up to here (of some weight, if the block has one) is the one the
      // search ends at or its neighbour.
      const bool weighs[2] = {v.cnt[0] && v.w[0] > 0.0, v.cnt[1] && v.w[1] > 0.0};
      c = weighs[1] ? before_c[1] + v.cnt[1] : weighs[0] ? before_c[1] : 0u;
      c = max(max(__reduce_max_sync(0xffffffffu, c), s.count[i]), 1u);
      m = __shfl_sync(0xffffffffu, before_m[1] + v.cnt[1] * v.w[1], 31);
      if (what == SAMPLE) {
        at_most = c;
      } else if (what == TOP_P && c < n) {
        n = c;
        kept = m;
      }
      continue;
    }
    const int l = __ffs((int)who) - 1;
    c = __shfl_sync(0xffffffffu, c, l);
    m = __shfl_sync(0xffffffffu, m, l);
    if (what < MIN_P) {
      if (c < n) {
        n = c;
        kept = m;
      }
    } else {
      bits = __shfl_sync(0xffffffffu, hb, l);
      ord = __shfl_sync(0xffffffffu, ho, l);
      w = __shfl_sync(0xffffffffu, hw, l);
      done = c <= n;  // beyond the kept head only by rounding
    }
  }
  // the CTA whose slice holds it (slices are in index order): lane r has CTA r's count
  uint32_t mine = 0u;
  if (lane < ctas) {
    const SampleShared* o = cluster.map_shared_rank(&s, lane);
    mine = count_in(o->hist[bits & 0x7fffu], bits & 0x8000u) + spilled_of(o, bits);
  }
  uint32_t upto = mine;
#pragma unroll
  for (int o = 1; o < MAX_CTAS; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  const int owner = min(__ffs((int)__ballot_sync(0xffffffffu, lane < ctas && ord < upto)) - 1, ctas - 1);
  if (lane == max(owner, 0)) {
    SampleShared* o = cluster.map_shared_rank(&s, lane);
    o->bits = bits;
    o->ordinal = ord - (upto - mine);
    o->w = w;
    o->kept = kept;
    o->owner = lane;
  }
}

template <int XT>
__global__ void __launch_bounds__(sm::THREADS) sample_kernel(const tq_sample_args a, int row0) {
  using namespace sm;
  extern __shared__ __align__(16) uint8_t raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int row = row0 + blockIdx.x / ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < WORDS / 4; i += THREADS) reinterpret_cast<uint4*>(s.hist)[i] = make_uint4(0u, 0u, 0u, 0u);
  s.mass[tid] = 0.0;
  s.count[tid] = 0u;
  s.card_of[tid] = CARDS;
  if (tid < 64) s.masked[tid >> 5][lane] = 0u;
  if (tid < 32) s.occur[tid] = 0u;
  if (tid == 0) {
    s.top = 0u;
    s.owner = -1;
    s.spills = s.spilled = 0u;
  }
  cluster.barrier_arrive();  // awaited before the first CTA writes into another
  grid_dep_wait();
  grid_dep_launch();
  if (warp == WARPS - 1) {  // the row's parameters, on their way while it is counted
    if (lane == 0) s.temperature = a.temperature ? a.temperature[row] : 1.0f;
    if (lane == 1) s.top_k = a.top_k ? a.top_k[row] : 0;
    if (lane == 2) s.top_p = a.top_p ? a.top_p[row] : 1.0f;
    if (lane == 3) s.min_p = a.min_p ? a.min_p[row] : 0.0f;
    if (lane == 4) {
      const int64_t col = a.u_cols == 1 ? 0 : min(max(*a.position - a.prompt_tokens + 1, (int64_t)0), a.u_cols - 1);
      s.u = a.uniform[(int64_t)row * a.u_ld + col];
    }
  }

  // ---- the slice's histogram
  const uint16_t* x = reinterpret_cast<const uint16_t*>(a.logits) + (int64_t)row * a.ld;
  const int64_t slice = (a.vocab + ctas - 1) / ctas;
  const int64_t lo = min((int64_t)a.vocab, rank * slice), hi = min((int64_t)a.vocab, lo + slice);
  // lines of 16 bytes; the first may begin before lo
  const int64_t base = lo - (int64_t)(((reinterpret_cast<uintptr_t>(x + lo)) & 15) >> 1);
  const int lines = hi > lo ? (int)((hi - base + 7) / 8) : 0;
  constexpr uint32_t NONE = 0x8000u | Bits<XT>::INF;  // -inf: a mask, not counted
  uint32_t* words = reinterpret_cast<uint32_t*>(raw);
  auto at_byte = [&](uint32_t byte) { return reinterpret_cast<uint32_t*>(raw + byte); };
  static_assert(offsetof(SampleShared, hist) == 0, "a magnitude is a word's index");
  // Masks, -inf or the type's lowest value (neighbours as numbers), would meet in one counter: each
  // lane has its own for them.
  const uint32_t mine_at = (uint32_t)offsetof(SampleShared, masked) / 4 + lane;
  uint32_t seen = 0u;  // bit 15: a counter at half of its range or above
  auto add_one = [&](uint32_t b) {
    const uint32_t d = b - Bits<XT>::LOWEST;  // 0: the lowest value, 1: -inf
    const uint32_t at = d <= 1u ? mine_at + 32u * (d ^ 1u) : b & 0x7fffu;
    seen |= atomicAdd(words + at, ((b << 1) & 0x10000u) | 1u);
  };
  auto line = [&](int i) {
    if (i < lines) return load_line(x, base + 8 * (int64_t)i, lo, hi);
    return make_uint4(NONE * 0x10001u, NONE * 0x10001u, NONE * 0x10001u, NONE * 0x10001u);
  };
  auto count_line = [&](const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    const uint32_t high = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
    if (__any_sync(0xffffffffu, (high & 0xffffu) >= Bits<XT>::LOWEST || high >= Bits<XT>::LOWEST << 16)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        add_one(w[e] & 0xffffu);
        add_one(w[e] >> 16);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        seen |= atomicAdd(at_byte((w[e] << 2) & 0x1fffcu), ((w[e] << 1) & 0x10000u) | 1u);
        seen |= atomicAdd(at_byte((w[e] >> 14) & 0x1fffcu), ((w[e] >> 15) & 0x10000u) | 1u);
      }
    }
  };
  // lines in flight: four to be counted and the next four (a round has at most four a thread, or is
  // the only one)
  uint4 next[4];
  const int round = lines < ROUND ? 4 * THREADS : SHORT_ROUND;
  auto fetch = [&](int first) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = k * THREADS + tid;
      next[k] = line(i < round ? first + i : lines);
    }
  };
  fetch(0);
#pragma unroll 1
  for (int first = 0; first < lines; first += round) {
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = next[k];
    if (first + round < lines) fetch(first + round);
    if (first == 0) __syncthreads();  // the counters are zero
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (first + k * THREADS < lines && k * THREADS + warp * 32 < round) count_line(v[k]);
    // (a counter holds the 65528 logits at most of a single round)
    if (lines < ROUND || first + round >= lines || !__syncthreads_or((int)(seen & 0x8000u))) continue;
    seen = 0u;
#pragma unroll 2
    for (int m4 = tid; m4 < WORDS / 4; m4 += THREADS) {
      const uint4 w4 = reinterpret_cast<const uint4*>(s.hist)[m4];
      if (!((w4.x | w4.y | w4.z | w4.w) & (0x10000u - KEEP))) continue;
#pragma unroll 1
      for (uint32_t m = 4 * m4; m < 4 * m4 + 4; ++m) {
        if (m > Bits<XT>::INF) {  // NaN: never kept, and its block may be that of +inf
          s.hist[m] = 0u;
          continue;
        }
        const uint32_t w = s.hist[m], n[2] = {(w & 0xffffu) - (w >> 16), w >> 16};
#pragma unroll
        for (uint32_t neg = 0; neg < 2; ++neg) {
          if (n[neg] < (uint32_t)KEEP) continue;
          const uint32_t out = n[neg] - 1u;  // one stays: the value occurs
          const uint32_t at = min(atomicAdd(&s.spills, 1u), (uint32_t)SPILLS - 1u);
          s.spill_bits[at] = neg && m ? 0x8000u | m : m;  // (-0 is +0)
          s.spill_count[at] = out;
          s.hist[m] -= out * (neg ? 0x10001u : 1u);
        }
      }
    }
    __syncthreads();
  }
  if (lines == 0) __syncthreads();
  __syncthreads();
  // what is never kept leaves, -0 joins +0, and the lanes' counts of the lowest value come in
  for (int m = (int)Bits<XT>::INF + 1 + tid; m < WORDS; m += THREADS) s.hist[m] = 0u;
  if (warp == 0) {
    const uint32_t lowest = __reduce_add_sync(0xffffffffu, s.masked[1][lane] & 0xffffu);
    if (lane == 0) {
      s.hist[0] &= 0xffffu;
      uint32_t* w = &s.hist[Bits<XT>::LOWEST & 0x7fffu];
      const uint32_t most = min(lowest, 0xffffu - (*w & 0xffffu));  // (one at least: a round is shorter)
      *w += most * 0x10001u;
      if (most < lowest) {
        const uint32_t at = min(s.spills++, (uint32_t)SPILLS - 1u);
        s.spill_bits[at] = Bits<XT>::LOWEST;
        s.spill_count[at] = lowest - most;
      }
    }
  }
  __syncthreads();
  cluster.barrier_wait();

  // ---- which blocks occur, and the slice's largest logit: two threads a block of 64 magnitudes
  {
    constexpr int LAST = (int)Bits<XT>::INF / 64;  // +inf is this block's first; above are NaNs
    const int j = tid >> 1;
    uint32_t some = 0u, less = 0u;  // high half: negative ones; low half of `less`: all and negative ones differ
    if (j <= LAST) {
      const uint4* h = reinterpret_cast<const uint4*>(s.hist) + tid * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint4 v = h[(k + lane) & 7];
        some |= v.x | v.y | v.z | v.w;
        less |= (v.x ^ (v.x >> 16)) | (v.y ^ (v.y >> 16)) | (v.z ^ (v.z >> 16)) | (v.w ^ (v.w >> 16));
      }
    }
    uint32_t any = (some & 0xffff0000u) | (less & 0xffffu);
    any |= __shfl_xor_sync(0xffffffffu, any, 1);
    auto squeeze = [](uint32_t b) {  // the even bits
      b &= 0x55555555u;
      b = (b | (b >> 1)) & 0x33333333u;
      b = (b | (b >> 2)) & 0x0f0f0f0fu;
      b = (b | (b >> 4)) & 0x00ff00ffu;
      return (b | (b >> 8)) & 0xffffu;
    };
    const uint32_t pos = squeeze(__ballot_sync(0xffffffffu, (any & 0xffffu) != 0u));
    const uint32_t neg = squeeze(__ballot_sync(0xffffffffu, (any >> 16) != 0u));
    uint32_t top = 0u;
    if (pos | neg) {
      const uint32_t jb = (uint32_t)warp * 16 + (pos ? 31 - __clz((int)pos) : __ffs((int)neg) - 1);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t m = jb * 64 + lane + 32 * e;
        if (count_in(s.hist[m], !pos)) top = max(top, order_of(pos ? m : 0x8000u | m));
      }
      top = __reduce_max_sync(0xffffffffu, top);
    }
    if (lane < ctas && top) {  // into every CTA of the cluster
      SampleShared* o = cluster.map_shared_rank(&s, lane);
      atomicMax(&o->top, top);
      if (s.spills) atomicOr(&o->spilled, 1u);
      atomicOr(&o->occur[warp], pos | (neg << 16));
    }
  }
  cluster.sync();

  // ---- count and mass of each block that occurs, left with CTA 0
  const uint32_t top = s.top, both = s.occur[lane];
  const double T = (double)s.temperature;
  const bool greedy = !(T > 0.0);
  RowScale scale;
  scale.top_bits = bits_of(top);
  scale.vmax = top ? (double)h2f((uint16_t)scale.top_bits, XT) : 0.0;
  scale.inv_t = 1.0 / T;
  scale.spike = greedy || scale.vmax > 1e300;
  const bool only_first = greedy || s.top_k == 1;  // no sums are asked for
  if (!only_first) {
    const int mine = __popc(both);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const int total = __shfl_sync(0xffffffffu, upto, 31);
    SampleShared* zero = cluster.map_shared_rank(&s, 0);
#pragma unroll 1
    for (int n = warp * ctas + rank; n < total; n += WARPS * ctas) {  // the n-th block that occurs
      const int l = __ffs((int)__ballot_sync(0xffffffffu, n < upto)) - 1;
      uint32_t set = __shfl_sync(0xffffffffu, both, l);
      for (int skip = n - (__shfl_sync(0xffffffffu, upto, l) - __popc(set)); skip > 0; --skip) set &= set - 1u;
      const int bit = __ffs((int)set) - 1, j = l * 16 + (bit & 15);
      const int i = bit >= 16 ? BLOCKS / 2 + j : BLOCKS / 2 - 1 - j;
      BlockView v;
      const double d = view_block<XT>(v, s, i, ctas, scale);
      const uint32_t c = __reduce_add_sync(0xffffffffu, v.cnt[0] + v.cnt[1]);
      const int card = total - 1 - n;  // the largest magnitudes keep cards
      if (card < CARDS) {
        BlockCard& k = zero->card[card];
        k.w[0][lane] = v.w[0];
        k.w[1][lane] = v.w[1];
        k.before[lane] = v.before;
        k.cnt[0][lane] = v.cnt[0];
        k.cnt[1][lane] = v.cnt[1];
      }
      if (lane == 0) {
        zero->mass[i] = d;
        zero->count[i] = c;
        if (card < CARDS) zero->card_of[i] = (uint16_t)card;
      }
    }
  }
  cluster.sync();

  // ---- CTA 0: running sums over the blocks, then its first warp finds the cuts
  if (rank == 0 && top) {
    uint32_t cc = s.count[tid], all_c = 1u;
    double cm = s.mass[tid], all_m = 1.0;
    if (!only_first) {
      scan_pair(cc, cm, s, all_c, all_m);
      s.count[tid] = cc;  // from here on: before the block
      s.mass[tid] = cm;
      __syncthreads();
    }
    if (warp == 0) pick<XT>(cluster, s, ctas, scale, greedy, all_c, all_m);
  }
  cluster.sync();

  // ---- the token: the ordinal-th of the slice with these bits
  auto write = [&](int64_t id) {
    if (a.ids) a.ids[row] = id;
    if (a.keys) a.keys[row] = (unsigned long long)(0xFFFFFFFFu - (uint32_t)id);
  };
  if (!top) {  // nothing to keep
    if (rank == 0 && tid == 0) {
      write(0);
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  if (s.owner != rank) return;
  if (tid == THREADS - 1 && a.logprobs) a.logprobs[row] = (float)log(s.w / s.kept);
  const uint32_t want = s.bits, ord = s.ordinal;
  const uint32_t want2 = want * 0x10001u, care = want ? 0xffffffffu : 0x7fff7fffu;  // -0 equals +0
  auto equals = [&](const uint4& v) {  // bits 31 - k and 15 - k: the high and low logit of word k
    auto zero = [&](uint32_t w) {
      const uint32_t x = (w & care) ^ want2;
      return ~(((x & 0x7fff7fffu) + 0x7fff7fffu) | x) & 0x80008000u;
    };
    return zero(v.x) | (zero(v.y) >> 1) | (zero(v.z) >> 2) | (zero(v.w) >> 3);
  };
  uint32_t before_round = 0u;
#pragma unroll 1
  for (int start = 0; start < lines; start += ROUND) {
    const int n = min(ROUND, lines - start);
    const int per = ((n + WARPS - 1) / WARPS + 31) / 32;  // a warp has per * 32 lines in a row, 8 a lane at most
    uint32_t eq[8], total = 0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = (warp * per + k) * 32 + lane;
      eq[k] = equals(line(k < per && i < n ? start + i : lines));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) total += __popc(eq[k]);
    const uint32_t mine = __reduce_add_sync(0xffffffffu, total);
    if (lane == 0) s.red_c[warp] = mine;
    __syncthreads();
    const uint32_t wc = s.red_c[lane];
    uint32_t before = before_round + __reduce_add_sync(0xffffffffu, lane < warp ? wc : 0u);
    before_round += __reduce_add_sync(0xffffffffu, wc);
    if (ord >= before && ord < before + mine) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t upto = __popc(eq[k]);
        if (ord >= before && __any_sync(0xffffffffu, upto != 0u)) {
#pragma unroll 1
          for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
          }
          const uint32_t first = before + upto - __popc(eq[k]);
          if (first <= ord && ord < before + upto) {
            uint32_t nth = ord - first;
#pragma unroll 1
            for (int e = 0; e < 8; ++e)
              if ((eq[k] >> ((e & 1 ? 31 : 15) - (e >> 1))) & 1u) {
                if (nth-- == 0u) write(base + 8 * (int64_t)(start + (warp * per + k) * 32 + lane) + e);
              }
          }
          before += __shfl_sync(0xffffffffu, upto, 31);
        }
      }
    }
    if (before_round > ord) return;
    __syncthreads();  // red_c is read before the next round writes it
  }
}

}  // namespace tq

using namespace tq;

static void set_launch(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, int rows, int ctas, cudaStream_t st) {
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)(rows * ctas), 1, 1);
  cfg.blockDim = dim3(sm::THREADS, 1, 1);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = tq_pdl_enabled() ? 2 : 1;
}

// Clusters of each size that are resident at once on this device (one CTA fills an SM; how many
// clusters fit depends on how the SMs are grouped), asked once per device.
static int resident_clusters(int ctas) {
  static std::atomic<int> known[64][sm::MAX_CTAS + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return tq_sm_count() / ctas;
  int n = known[dev][ctas].load(std::memory_order_relaxed);
  if (n > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  set_launch(cfg, attr, 1, ctas, nullptr);
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, sample_kernel<TQ_DTYPE_BF16>, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = std::max(1, tq_sm_count() / ctas);
  }
  // larger clusters find all their places only on an empty device: 26 clusters of five, the most that
  // fit, took a second wave behind another kernel (26 against 18 us; the eighth that is kept free comes
  // from that case alone)
  if (ctas > 2) n = std::max(1, n * 7 / 8);
  known[dev][ctas].store(n, std::memory_order_relaxed);
  return n;
}

template <int XT>
static int launch_sample(const tq_sample_args& a, cudaStream_t st) {
  auto kern = sample_kernel<XT>;
  static std::atomic<uint64_t> done{0}, done_bf16{0};
  TQ_CUDA_TRY(tq_allow_smem(kern, (int)sizeof(SampleShared), done));
  TQ_CUDA_TRY(tq_allow_smem(sample_kernel<TQ_DTYPE_BF16>, (int)sizeof(SampleShared), done_bf16));  // resident_clusters asks of it
  // Cluster sizes by time: a wave of clusters takes the fixed chain of barriers and searches, the
  // passes over a slice (1.65e-4 us per token of it) and 1 us for each block of values that a warp
  // sums up, of which a row of bf16 logits has about 100 and one of f16 about 600, counted in rows of
  // normal logits with a few strong ones (18 us measured for
  // slices of 16k bf16 logits, 23 of 50k, 41 of 152k).  One size for all rows, or full waves of one size and then
  // the rest with a larger one in a second launch (192 rows of 152064, before later steps: 80 us, against
  // 85 in two waves of single CTAs and 98 in four of clusters of three).
  const int blocks = std::min(a.vocab, XT == TQ_DTYPE_BF16 ? 100 : 600);
  auto wave = [&](int c) {
    return 11.7 + 1.65e-4 * a.vocab / c + 1.0 * ((blocks + sm::WARPS * c - 1) / (sm::WARPS * c));
  };
  auto time_of = [&](int rows, int c) {
    const int fit = resident_clusters(c);
    return (rows + fit - 1) / fit * wave(c);
  };
  auto best_of = [&](int rows) {
    int best = 1;
    for (int c = 2; c <= sm::MAX_CTAS; ++c)
      if (time_of(rows, c) < time_of(rows, best)) best = c;
    return best;
  };
  int first = a.n_rows, c0 = best_of(a.n_rows), c1 = 0;
  double least = time_of(a.n_rows, c0);
  for (int c = 1; c <= sm::MAX_CTAS; ++c) {
    const int full = a.n_rows / resident_clusters(c) * resident_clusters(c);
    if (full == 0 || full == a.n_rows) continue;
    const int rest = best_of(a.n_rows - full);
    const double t = time_of(full, c) + time_of(a.n_rows - full, rest) + 2.0;
    if (t < least) {
      least = t;
      first = full;
      c0 = c;
      c1 = rest;
    }
  }
  for (int part = 0; part < (first < a.n_rows ? 2 : 1); ++part) {
    const int row0 = part ? first : 0;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    set_launch(cfg, attr, part ? a.n_rows - first : first, part ? c1 : c0, st);
    TQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, row0));
    tq_count_launch();
  }
  return TQ_OK;
}

extern "C" int tq_sample(const tq_sample_args* args, int dtype, void* stream) {
  if (!args) return tq_set_error(TQ_ERR_INVALID, "null arguments");
  const tq_sample_args a = *args;
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_F16) return tq_set_error(TQ_ERR_INVALID, "dtype must be bf16 or f16");
  if (a.n_rows < 0 || a.n_rows > 65536 || a.vocab < 1 || (a.n_rows > 1 && a.ld < a.vocab))
    return tq_set_error(TQ_ERR_INVALID, "sample: 0..65536 rows of vocab <= ld logits");
  if (a.vocab > sm::MAX_VOCAB) return tq_set_error(TQ_ERR_UNSUPPORTED, "sample: vocab above 1048576");
  if (a.n_rows == 0) return TQ_OK;
  if (!a.logits || !a.uniform || (!a.ids && !a.keys)) return tq_set_error(TQ_ERR_INVALID, "null pointer");
  if ((uintptr_t)a.logits & 1) return tq_set_error(TQ_ERR_INVALID, "sample: misaligned logits");
  if (a.u_cols < 1 || (a.u_cols > 1 && !a.position)) return tq_set_error(TQ_ERR_INVALID, "sample: bad random numbers");
  if (a.keys && !a.position) return tq_set_error(TQ_ERR_INVALID, "null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  const int rc = dtype == TQ_DTYPE_BF16 ? launch_sample<TQ_DTYPE_BF16>(a, st) : launch_sample<TQ_DTYPE_F16>(a, st);
  if (rc != TQ_OK || !a.keys) return rc;
  return tq_launch_pick_finish(a.keys, a.n_rows, a.next, a.token, a.generated, a.gen_ld, a.gen_cols, a.position,
                               a.prompt_tokens, st);
}
