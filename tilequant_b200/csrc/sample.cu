// Token sampling with temperature, top-k, top-p and min-p from given random numbers (sm_100a).
//
// The weights are w = exp((l - max) / T).  In the order (logit falling, index rising) each
// filter keeps a head, so the kept tokens are the first n of that order and the sampled one is
// the first whose running sum exceeds u times the sum of those n.  A decision of either kind
// compares long sums, and one token's weight may be 1e-7 of them, so sums and weights are f64.
//
// No sort: 16-bit logits take at most 65536 values, and equal logits have equal weights.  A row
// is counted into a histogram over the value's bits (made order-preserving), in integers, so
// nothing depends on the order of atomics; a weight is then computed once per value that occurs
// (a few thousand of 1e5 tokens), and every sum over tokens is a sum over values of
// count * weight.  The sampled value and its ordinal among equals known, one more pass over the
// row (from L2) finds the ordinal-th token with these bits.
//
// One cluster of up to eight CTAs per row.  A CTA holds a histogram of its slice of the row as
// 65536 16-bit counters (128 KB; a slice is at most 65535 tokens, so none overflows).  The
// values are cut into 1024 blocks of 64; the CTAs share out the blocks, add the cluster's
// counters up over distributed shared memory and leave (count, mass) of each block with CTA 0,
// which scans the 1024 blocks, looks into the (at most four) blocks where a filter or the
// sample falls, and tells the CTA whose slice holds the token.
//
// What bounds it: for few rows latency (three cluster barriers and the chain of searches); for
// many rows the shared-memory atomics, one per token.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "pick.cuh"
#include "tma.cuh"

namespace cg = cooperative_groups;

namespace tq {
namespace sm {
constexpr int THREADS = 1024;
constexpr int KEYS = 65536;
constexpr int BLOCKS = 1024;           // of 64 values
constexpr int WORDS = KEYS / 2;        // two counters per word
constexpr int MAX_SLICE = 65535;       // tokens per CTA: a counter holds no more
constexpr int MAX_CTAS = 8;
}  // namespace sm

struct SampleShared {
  uint32_t hist[sm::WORDS];
  double mass[sm::BLOCKS];   // CTA 0: of the whole row
  uint32_t count[sm::BLOCKS];
  double red_m[32];
  uint32_t red_c[32];
  uint32_t max_key;          // of this CTA's slice (0: nothing there)
  int owner;                 // rank of the CTA that holds the sampled token (-1: none)
  uint32_t key, ordinal;     // its value and its place among this CTA's equals
  float logprob;
};

// Order-preserving 16-bit key of a logit; 0 for what is never kept (NaN, -inf).
template <int XT>
__device__ __forceinline__ uint32_t key_of(uint32_t b) {
  constexpr uint32_t INF = XT == TQ_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  if ((b & 0x7fffu) > INF || b == (0x8000u | INF)) return 0u;
  if (b == 0x8000u) b = 0u;  // -0 equals +0
  return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
}
template <int XT>
__device__ __forceinline__ double value_of(uint32_t key) {
  const uint32_t b = (key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu);
  return (double)h2f((uint16_t)b, XT);
}

// exp((value - max) / T).  `spike`: only the largest value weighs (T <= 0, or the largest is +inf).
template <int XT>
__device__ __forceinline__ double weight_of(uint32_t key, uint32_t max_key, double vmax, double T, bool spike) {
  if (key == max_key) return 1.0;
  return spike ? 0.0 : exp((value_of<XT>(key) - vmax) / T);
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
  __syncthreads();
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

// 8 logits at the 16-byte line `line` of the row's memory, `first` their index; those outside
// [lo, hi) come as NaN.  Lines that cross an end are read value by value.
template <int XT>
__device__ __forceinline__ uint4 load_line(const uint16_t* row, int64_t first, int64_t lo, int64_t hi) {
  if (first >= lo && first + 8 <= hi) return *reinterpret_cast<const uint4*>(row + first);
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = 0x7fff7fffu;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t j = first + 2 * e + k;
      if (j >= lo && j < hi) w[e] = (w[e] & (k ? 0xffffu : 0xffff0000u)) | ((uint32_t)row[j] << (16 * k));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One warp's view of a block's 64 values, lane order falling (lane 0 has the largest two), with
// the counts of the whole row.
struct BlockView {
  uint32_t key[2], cnt[2];  // falling
  double w[2];
  uint32_t before_c[2];     // tokens of the block before this value
  double before_m[2];
};

template <int XT>
__device__ __forceinline__ BlockView view_block(cg::cluster_group& cluster, SampleShared& s, int block, int ctas,
                                                uint32_t max_key, double vmax, double T, bool spike) {
  const int lane = threadIdx.x & 31;
  BlockView v;
  const int word = block * 32 + 31 - lane;
  uint32_t lo = 0, hi = 0;
  for (int r = 0; r < ctas; ++r) {
    const uint32_t x = cluster.map_shared_rank(s.hist, r)[word];
    lo += x & 0xffffu;
    hi += x >> 16;
  }
  v.key[0] = 2 * word + 1;
  v.key[1] = 2 * word;
  v.cnt[0] = hi;
  v.cnt[1] = lo;
#pragma unroll
  for (int e = 0; e < 2; ++e) v.w[e] = v.cnt[e] ? weight_of<XT>(v.key[e], max_key, vmax, T, spike) : 0.0;
  const double m0 = v.cnt[0] * v.w[0], m1 = v.cnt[1] * v.w[1];
  uint32_t xc = hi + lo;
  double xm = m0 + m1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t yc = __shfl_up_sync(0xffffffffu, xc, o);
    const double ym = __shfl_up_sync(0xffffffffu, xm, o);
    if (lane >= o) {
      xc += yc;
      xm += ym;
    }
  }
  double em = __shfl_up_sync(0xffffffffu, xm, 1);
  if (lane == 0) em = 0.0;
  v.before_c[0] = xc - hi - lo;
  v.before_c[1] = v.before_c[0] + hi;
  v.before_m[0] = em;
  v.before_m[1] = em + m0;
  return v;
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
// s.count / s.mass hold the tokens and mass before the i-th block from the top.
template <int XT>
__device__ __forceinline__ void pick(cg::cluster_group& cluster, SampleShared& s, const tq_sample_args& a, int row,
                                     int ctas, uint32_t max_key, double vmax, double T, bool greedy, bool spike,
                                     uint32_t all_c, double all_m) {
  using namespace sm;
  const int lane = threadIdx.x & 31;
  auto view = [&](int i) {
    return view_block<XT>(cluster, s, BLOCKS - 1 - i, ctas, max_key, vmax, T, spike);
  };
  uint32_t n = all_c;  // the kept head and its mass
  double kept = all_m;
  const int k = a.top_k ? a.top_k[row] : 0;
  const uint32_t want = greedy ? 1u : k > 0 ? (uint32_t)k : 0u;
  if (want == 1u) {
    n = 1u;
    kept = 1.0;
  } else if (want && want < all_c) {
    const int i = last_block([&](int j) { return s.count[j] < want; });
    const BlockView v = view(i);
    double m = 0.0;
    bool hit = false;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t b0 = s.count[i] + v.before_c[e];
      if (v.cnt[e] && b0 < want && want <= b0 + v.cnt[e]) {
        hit = true;
        m = s.mass[i] + v.before_m[e] + (want - b0) * v.w[e];
      }
    }
    const uint32_t who = __ballot_sync(0xffffffffu, hit);
    n = want;
    kept = __shfl_sync(0xffffffffu, m, max(__ffs((int)who) - 1, 0));
  }
  const double p = a.top_p ? (double)a.top_p[row] : 1.0;
  uint32_t n2 = n;
  double kept2 = kept;
  if (p < 1.0 && n > 1u) {  // the shortest head with mass >= p of what is kept
    const double need = p * kept;
    if (need <= 1.0) {  // the first token, of weight 1, is enough
      n2 = 1u;
      kept2 = 1.0;
    } else {
      const int i = last_block([&](int j) { return s.mass[j] < need; });
      const BlockView v = view(i);
      double m = 0.0;
      uint32_t c = 0;
      bool hit = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const double b0 = s.mass[i] + v.before_m[e];
        if (v.cnt[e] && !hit && need <= b0 + v.cnt[e] * v.w[e]) {
          hit = true;
          double q = ceil((need - b0) / v.w[e]);
          q = fmin(fmax(q, 1.0), (double)v.cnt[e]);
          if (q > 1.0 && b0 + (q - 1.0) * v.w[e] >= need) q -= 1.0;  // the quotient was rounded
          if (q < (double)v.cnt[e] && b0 + q * v.w[e] < need) q += 1.0;
          c = s.count[i] + v.before_c[e] + (uint32_t)q;
          m = b0 + q * v.w[e];
        }
      }
      const uint32_t who = __ballot_sync(0xffffffffu, hit);
      if (who) {  // else the sums differ by a rounding and the head is everything
        c = __shfl_sync(0xffffffffu, c, __ffs((int)who) - 1);
        m = __shfl_sync(0xffffffffu, m, __ffs((int)who) - 1);
        if (c < n) {
          n2 = c;
          kept2 = m;
        }
      }
    }
  }
  const double mp = a.min_p ? (double)a.min_p[row] : 0.0;
  if (mp > 0.0 && n2 > 1u) {  // the tokens with weight >= min_p
    // the last block whose largest value has that weight; those above it hold no smaller ones
    const int i = last_block([&](int j) {
      const int key = min((BLOCKS - 1 - j) * 64 + 63, (int)max_key);
      return weight_of<XT>((uint32_t)key, max_key, vmax, T, spike) >= mp;
    });
    const BlockView v = view(i);
    uint32_t c = 0;
    double m = 0.0;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (v.cnt[e] && v.w[e] >= mp) {
        c += v.cnt[e];
        m = s.mass[i] + v.before_m[e] + v.cnt[e] * v.w[e];
      }
    const uint32_t any = __ballot_sync(0xffffffffu, c != 0u);
    m = any ? __shfl_sync(0xffffffffu, m, 31 - __clz((int)any)) : s.mass[i];
    c = __reduce_add_sync(0xffffffffu, c) + s.count[i];
    if (c < n2) {
      n2 = c;
      kept2 = m;
    }
  }
  n = max(n2, 1u);  // the first token always stays
  kept = n2 ? kept2 : 1.0;

  const int64_t col =
      a.u_cols == 1 ? 0 : min(max(*a.position - a.prompt_tokens + 1, (int64_t)0), a.u_cols - 1);
  double u = (double)a.uniform[(int64_t)row * a.u_ld + col];
  u = u > 0.0 ? fmin(u, 1.0) : 0.0;  // NaN: 0
  const double target = u * kept;
  uint32_t key = max_key, ord = 0u;
  double w = 1.0;
  bool done = n == 1u;
  if (!done) {
    const int i = last_block([&](int j) { return s.mass[j] <= target; });
    const BlockView v = view(i);
    uint32_t c = 0, kk = 0;
    double ww = 0.0;
    bool hit = false;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const double b0 = s.mass[i] + v.before_m[e];
      if (v.cnt[e] && kk == 0u && target < b0 + v.cnt[e] * v.w[e]) {
        double q = floor((target - b0) / v.w[e]);
        q = fmin(fmax(q, 0.0), (double)(v.cnt[e] - 1u));
        if (q > 0.0 && b0 + q * v.w[e] > target) q -= 1.0;
        if (q < (double)(v.cnt[e] - 1u) && b0 + (q + 1.0) * v.w[e] <= target) q += 1.0;
        c = (uint32_t)q;
        kk = v.key[e];
        ww = v.w[e];
        hit = s.count[i] + v.before_c[e] + c < n;  // beyond the kept head only by rounding
      }
    }
    // the first lane with such a value decides
    const uint32_t who = __ballot_sync(0xffffffffu, kk != 0u);
    if (who) {
      const int l = __ffs((int)who) - 1;
      ord = __shfl_sync(0xffffffffu, c, l);
      key = __shfl_sync(0xffffffffu, kk, l);
      w = __shfl_sync(0xffffffffu, ww, l);
      done = __shfl_sync(0xffffffffu, (int)hit, l) != 0;
    }
  }
  if (!done) {  // u times the sum reached the sum by rounding: the last kept token
    const int i = last_block([&](int j) { return s.count[j] < n; });
    const BlockView v = view(i);
    bool hit = false;
    uint32_t c = 0, kk = 0;
    double ww = 0.0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t b0 = s.count[i] + v.before_c[e];
      if (v.cnt[e] && b0 < n && n <= b0 + v.cnt[e]) {
        hit = true;
        c = n - 1u - b0;
        kk = v.key[e];
        ww = v.w[e];
      }
    }
    const int l = max(__ffs((int)__ballot_sync(0xffffffffu, hit)) - 1, 0);
    ord = __shfl_sync(0xffffffffu, c, l);
    key = __shfl_sync(0xffffffffu, kk, l);
    w = __shfl_sync(0xffffffffu, ww, l);
  }
  if (lane == 0) {  // the CTA whose slice holds it: slices are in index order
    int r = 0;
    for (; r < ctas - 1; ++r) {
      const uint32_t x = cluster.map_shared_rank(s.hist, r)[key >> 1];
      const uint32_t c = (key & 1u) ? x >> 16 : x & 0xffffu;
      if (ord < c) break;
      ord -= c;
    }
    SampleShared* o = cluster.map_shared_rank(&s, r);
    o->key = key;
    o->ordinal = ord;
    o->logprob = (float)log(w / kept);
    o->owner = r;
  }
}

template <int XT>
__global__ void __launch_bounds__(sm::THREADS) sample_kernel(const tq_sample_args a) {
  using namespace sm;
  extern __shared__ __align__(16) uint8_t raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int row = blockIdx.x / ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < WORDS / 4; i += THREADS) reinterpret_cast<uint4*>(s.hist)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (tid == 0) {
    s.max_key = 0u;
    s.owner = -1;
  }
  grid_dep_wait();
  grid_dep_launch();
  __syncthreads();

  // ---- the slice's histogram
  const uint16_t* x = reinterpret_cast<const uint16_t*>(a.logits) + (int64_t)row * a.ld;
  const int64_t slice = (a.vocab + ctas - 1) / ctas;
  const int64_t lo = min((int64_t)a.vocab, rank * slice), hi = min((int64_t)a.vocab, lo + slice);
  // lines of 16 bytes; the first may begin before lo
  const int64_t base = lo - (int64_t)(((reinterpret_cast<uintptr_t>(x + lo)) & 15) >> 1);
  const int lines = (int)((hi - base + 7) / 8) * (hi > lo);
  constexpr uint32_t LOWEST = XT == TQ_DTYPE_BF16 ? 0x0080u : 0x0400u;  // key of the type's lowest value
  uint32_t top = 0u, lowest = 0u;
  auto add = [&](uint32_t k) {
    top = max(top, k);
    if (k == LOWEST)
      ++lowest;  // a mask of the lowest value: the same counter for many lanes
    else if (k)
      atomicAdd(&s.hist[k >> 1], 1u << ((k & 1u) * 16));
  };
  for (int i = tid; i < lines; i += 2 * THREADS) {
    const int i1 = i + THREADS;
    const uint4 v0 = load_line<XT>(x, base + 8 * (int64_t)i, lo, hi);
    uint4 v1 = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
    if (i1 < lines) v1 = load_line<XT>(x, base + 8 * (int64_t)i1, lo, hi);
    const uint32_t w[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      add(key_of<XT>(w[e] & 0xffffu));
      add(key_of<XT>(w[e] >> 16));
    }
  }
  lowest = __reduce_add_sync(0xffffffffu, lowest);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) {
    if (lowest) atomicAdd(&s.hist[LOWEST >> 1], lowest << ((LOWEST & 1u) * 16));
    if (top) atomicMax(&s.max_key, top);
  }
  cluster.sync();

  // ---- count and mass of each block of 64 values, left with CTA 0
  uint32_t max_key = 0u;
  for (int r = 0; r < ctas; ++r) max_key = max(max_key, *cluster.map_shared_rank(&s.max_key, r));
  const double T = a.temperature ? (double)a.temperature[row] : 1.0;
  const double vmax = max_key ? value_of<XT>(max_key) : 0.0;
  const bool greedy = !(T > 0.0);
  const bool spike = greedy || vmax > 1e300;
  const int top_block = (int)(max_key >> 6);
  {
    double* mass0 = cluster.map_shared_rank(s.mass, 0);
    uint32_t* count0 = cluster.map_shared_rank(s.count, 0);
    for (int i = warp; i * ctas + rank < BLOCKS; i += THREADS / 32) {
      const int block = i * ctas + rank;
      uint32_t c0 = 0, c1 = 0;
      if (block <= top_block)
        for (int r = 0; r < ctas; ++r) {
          const uint32_t w = cluster.map_shared_rank(s.hist, r)[block * 32 + lane];
          c0 += w & 0xffffu;
          c1 += w >> 16;
        }
      uint32_t c = c0 + c1;
      double m = 0.0;
      if (__any_sync(0xffffffffu, c != 0u)) {
        const uint32_t k = (uint32_t)(block * 64 + 2 * lane);
        if (c0) m = c0 * weight_of<XT>(k, max_key, vmax, T, spike);
        if (c1) m += c1 * weight_of<XT>(k + 1, max_key, vmax, T, spike);
        c = __reduce_add_sync(0xffffffffu, c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      }
      if (lane == 0) {
        mass0[block] = m;
        count0[block] = c;
      }
    }
  }
  cluster.sync();

  // ---- CTA 0: running sums over the blocks in falling order, then its first warp finds the cuts
  if (rank == 0 && max_key) {
    uint32_t cc = s.count[BLOCKS - 1 - tid], all_c;
    double cm = s.mass[BLOCKS - 1 - tid], all_m;
    scan_pair(cc, cm, s, all_c, all_m);  // (its barriers separate these reads from the writes)
    s.count[tid] = cc;  // from here on: before the tid-th block from the top
    s.mass[tid] = cm;
    __syncthreads();
    if (warp == 0) pick<XT>(cluster, s, a, row, ctas, max_key, vmax, T, greedy, spike, all_c, all_m);
  }
  cluster.sync();

  // ---- the token: the ordinal-th of the slice with these bits
  auto write = [&](int64_t id, float lp) {
    if (a.ids) a.ids[row] = id;
    if (a.logprobs) a.logprobs[row] = lp;
    if (a.keys) a.keys[row] = (unsigned long long)(0xFFFFFFFFu - (uint32_t)id);
  };
  if (!max_key) {  // nothing to keep
    if (rank == 0 && tid == 0) write(0, -INFINITY);
    return;
  }
  if (s.owner != rank) return;
  const uint32_t key = s.key, ord = s.ordinal;
  const int per = (lines + THREADS - 1) / THREADS;  // consecutive lines of a thread
  uint32_t mine = 0;
  for (int i = tid * per; i < min(lines, (tid + 1) * per); ++i) {
    const uint4 v = load_line<XT>(x, base + 8 * (int64_t)i, lo, hi);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) mine += (key_of<XT>(w[e] & 0xffffu) == key) + (key_of<XT>(w[e] >> 16) == key);
  }
  uint32_t before = mine, total_c;
  double zero = 0.0, total_m;
  scan_pair(before, zero, s, total_c, total_m);
  if (before <= ord && ord < before + mine) {
    uint32_t at = before;
    for (int i = tid * per; i < min(lines, (tid + 1) * per); ++i) {
      const uint4 v = load_line<XT>(x, base + 8 * (int64_t)i, lo, hi);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (key_of<XT>((w[e >> 1] >> ((e & 1) * 16)) & 0xffffu) == key && at++ == ord)
          write(base + 8 * (int64_t)i + e, s.logprob);
    }
  }
}

}  // namespace tq

using namespace tq;

template <int XT>
static int launch_sample(const tq_sample_args& a, int ctas, cudaStream_t st) {
  auto kern = sample_kernel<XT>;
  const int smem = (int)sizeof(SampleShared);
  static std::atomic<uint64_t> done{0};
  TQ_CUDA_TRY(tq_allow_smem(kern, smem, done));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_rows * ctas), 1, 1);
  cfg.blockDim = dim3(sm::THREADS, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = tq_pdl_enabled() ? 2 : 1;
  TQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a));
  tq_count_launch();
  return TQ_OK;
}

extern "C" int tq_sample(const tq_sample_args* args, int dtype, void* stream) {
  if (!args) return tq_set_error(TQ_ERR_INVALID, "null arguments");
  const tq_sample_args a = *args;
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_F16) return tq_set_error(TQ_ERR_INVALID, "dtype must be bf16 or f16");
  if (a.n_rows < 0 || a.n_rows > 65536 || a.vocab < 1 || (a.n_rows > 1 && a.ld < a.vocab))
    return tq_set_error(TQ_ERR_INVALID, "sample: 0..65536 rows of vocab <= ld logits");
  if (a.vocab > sm::MAX_CTAS * sm::MAX_SLICE) return tq_set_error(TQ_ERR_UNSUPPORTED, "sample: vocab above 524280");
  if (a.n_rows == 0) return TQ_OK;
  if (!a.logits || !a.uniform || (!a.ids && !a.keys)) return tq_set_error(TQ_ERR_INVALID, "null pointer");
  if ((uintptr_t)a.logits & 1) return tq_set_error(TQ_ERR_INVALID, "sample: misaligned logits");
  if (a.u_cols < 1 || (a.u_cols > 1 && !a.position)) return tq_set_error(TQ_ERR_INVALID, "sample: bad random numbers");
  if (a.keys && !a.position) return tq_set_error(TQ_ERR_INVALID, "null pointer");
  // the slices' counters bound the cluster from below, one wave of CTAs (one per SM) from above
  const int least = (a.vocab + sm::MAX_SLICE - 1) / sm::MAX_SLICE;
  const int ctas = std::max(least, std::min(tq_sm_count() / a.n_rows, sm::MAX_CTAS));
  cudaStream_t st = (cudaStream_t)stream;
  const int rc = dtype == TQ_DTYPE_BF16 ? launch_sample<TQ_DTYPE_BF16>(a, ctas, st)
                                        : launch_sample<TQ_DTYPE_F16>(a, ctas, st);
  if (rc != TQ_OK || !a.keys) return rc;
  return tq_launch_pick_finish(a.keys, a.n_rows, a.next, a.token, a.generated, a.gen_ld, a.gen_cols, a.position,
                               a.prompt_tokens, st);
}
