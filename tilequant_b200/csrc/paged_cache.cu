// The 8-bit paged KV cache (sm_100a): pages planned on the device from request lengths, the
// new keys and values quantized into them, and pages read back.
//
// A pool has P pages of `page` tokens.  Request r holds lengths[r] tokens in the pages
// block_table[r][0 .. ceil(lengths[r] / page)); free_pages[0 .. free_count) is a stack of the
// pages nobody holds.  A layer's cache is k, v int8 [P][Hkv][page][D] and one f32 scale per
// (page, KV head) and side: value = code * scale.  A page and head is one contiguous block, so
// attention fetches it in whole TMA boxes and the writer owns it with one thread block.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "paged.cuh"
#include "tma.cuh"

namespace cg = cooperative_groups;

namespace tq {

// ------------------------------------------------------------------ page planning
// One step adds new_lens[r] tokens to request r.  With need_r = ceil((L_r + n_r) / page) -
// ceil(L_r / page) and running sums over the requests in order, the i-th fresh page of the
// step is free_pages[free_count - 1 - i], token i of request r is row cu_new[r] + i at
// position L_r + i, and everything else (write items, attention's work split) follows from
// further running sums.  So: three block-wide scans of at most four requests per thread, then the
// touched pages, which find their request by bisection in shared memory.  Nothing depends on the
// order of atomics.
//
// What bounds it is latency: about 2 KB are read for 64 requests.  The pages and token rows of a
// prefill (16 bytes per token) are spread over the CTAs of one cluster, each of which repeats the
// scans; the cluster barrier between reading the state and writing it lets a step update lengths
// and free_count in place.  Measured: 6.7 us for 64 decoding requests, 11.3 us for 256 requests
// with 65k new tokens (the three scans take 3 us of either; the rows and the cluster's barriers are
// the difference).  The scans are sized for 4096 requests: 64 fill two of their 32 warps.
//
// A request is admitted if its tokens fit its table row and the plan's token rows and its
// fresh pages are there; the pages go to the requests in order until the first that finds too
// few, and later requests then get none either.  A request that is not admitted keeps its
// length; its token rows have slot and position -1, and attention gives zeros for them.
namespace pl {
constexpr int THREADS = 1024;
constexpr int PER = TQ_MAX_REQUESTS / THREADS;  // requests per thread
constexpr int MARKS = 1 << 20;                  // pages that release_kernel marks at a time (128 KB of bits)
}  // namespace pl

// Exclusive running sums over the block (thread order) of K numbers at once; total gets the sums.
// `red` holds K * 32 numbers that no thread still reads.
template <int K>
__device__ __forceinline__ void block_scan(int64_t (&v)[K], int64_t* red, int64_t (&total)[K]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t x[K], w[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    x[k] = v[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x[k], o);
      if (lane >= o) x[k] += y;
    }
    if (lane == 31) red[k * 32 + warp] = x[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    w[k] = red[k * 32 + lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, w[k], o);
      if (lane >= o) w[k] += y;
    }
    const int64_t before = __shfl_sync(0xffffffffu, w[k], (warp + 31) & 31);
    total[k] = __shfl_sync(0xffffffffu, w[k], 31);
    v[k] = (warp ? before : 0) + x[k] - v[k];
  }
}

// The last r with cu[r] <= x, for cu[0] = 0 and x below cu[n].
__device__ __forceinline__ int owner_of(const int* cu, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(pl::THREADS) plan_kernel(const tq_plan_args a) {
  using namespace pl;
  extern __shared__ int sm[];
  const int R = a.requests, page = a.page, shift = 31 - __clz(page), tile_shift = 31 - __clz(a.row_tile);
  int* len = sm;                  // [R] tokens before the step
  int* cu_tok = len + R;          // [R + 1] token rows, clipped to max_tokens
  int* cu_fresh = cu_tok + R + 1;  // [R + 1] fresh pages
  int* cu_item = cu_fresh + R + 1;  // [R + 1] touched pages
  int* cu_work = cu_item + R + 1;  // [R + 1] attention chunks
  __shared__ int64_t red[5 * 32];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x;
  const int per = (R + THREADS - 1) / THREADS;
  const int r0 = tid * per;
  const int64_t room = (int64_t)a.table_width * page;
  const int avail = min(max(*a.free_count, 0), a.pages);
  int L[PER], n[PER];
  int64_t sum[1] = {0}, total[1];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (i >= per) break;
    const int r = r0 + i;
    L[i] = n[i] = 0;
    if (r < R) {
      L[i] = max(a.lengths[r], 0);
      n[i] = max(a.new_lens[r], 0);
    }
    sum[0] += n[i];
  }
  block_scan<1>(sum, red, total);
  int64_t at = sum[0];
  int64_t tok[PER];
  int need[PER];
  bool fits[PER];
  int bad = 0;
  sum[0] = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (i >= per) break;
    tok[i] = at;
    at += n[i];
    const int64_t end = (int64_t)L[i] + n[i];
    fits[i] = end <= room && at <= a.max_tokens;
    if (n[i] && end > room) bad |= TQ_PAGES_TABLE_FULL;
    if (n[i] && at > a.max_tokens) bad |= TQ_PAGES_ROWS_FULL;
    need[i] = fits[i] && n[i] ? (int)(((end + page - 1) >> shift) - ((L[i] + (int64_t)page - 1) >> shift)) : 0;
    sum[0] += need[i];
  }
  block_scan<1>(sum, red + 32, total);
  int64_t fresh = sum[0];
  int take[PER];
  int64_t run[3] = {0, 0, 0}, totals[3];  // fresh pages, touched pages, attention chunks
  int kv[PER], rows[PER], touched[PER];
  int64_t chunks[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (i >= per) break;
    fresh += need[i];
    const bool pool_short = need[i] && fresh > avail;
    if (pool_short) bad |= TQ_PAGES_POOL_EMPTY;
    const bool in = n[i] && fits[i] && !pool_short;
    take[i] = in ? need[i] : 0;
    kv[i] = in ? L[i] + n[i] : 0;
    touched[i] = in ? ((kv[i] - 1) >> shift) - (L[i] >> shift) + 1 : 0;
    rows[i] = (int)(min(tok[i] + n[i], (int64_t)a.max_tokens) - min(tok[i], (int64_t)a.max_tokens));
    const int64_t tiles = ((int64_t)rows[i] * a.group + a.row_tile - 1) >> tile_shift;
    chunks[i] = rows[i] ? tiles * a.kv_heads * (TQ_ATTN_LEAD + max(1, (kv[i] + TQ_ATTN_CHUNK - 1) / TQ_ATTN_CHUNK)) : 0;
    run[0] += take[i];
    run[1] += touched[i];
    run[2] += chunks[i];
  }
  block_scan<3>(run, red + 64, totals);
  const int64_t n_fresh = totals[0], n_items = totals[1], n_work = totals[2];
  int64_t f = run[0], it = run[1], wk = run[2];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (i >= per) break;
    const int r = r0 + i;
    if (r < R) {
      len[r] = kv[i] ? L[i] : -1;  // -1: not admitted
      cu_tok[r] = (int)min(tok[i], (int64_t)a.max_tokens);
      cu_fresh[r] = (int)f;
      cu_item[r] = (int)it;
      cu_work[r] = (int)wk;
      f += take[i];
      it += touched[i];
      wk += chunks[i];
      if (r == R - 1) {
        cu_tok[R] = (int)min(tok[i] + n[i], (int64_t)a.max_tokens);
        cu_fresh[R] = (int)n_fresh;
        cu_item[R] = (int)n_items;
        cu_work[R] = (int)n_work;
      }
    }
  }
  if (ctas > 1)
    cluster.sync();  // every CTA has read lengths and free_count before any is written
  else
    __syncthreads();

  if (rank == 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (i >= per) break;
      const int r = r0 + i;
      if (r < R) {
        // a length that was negative stays as it is when nothing is added
        if (kv[i] || a.lengths_out != a.lengths) a.lengths_out[r] = kv[i] ? kv[i] : a.lengths[r];
        a.kv_len[r] = kv[i];
        a.cu_new[r] = cu_tok[r];
        a.cu_work[r] = cu_work[r];
      }
    }
    if (tid == 0) {
      a.cu_new[R] = cu_tok[R];
      a.cu_work[R] = cu_work[R];
      *a.free_count_out = avail - (int)n_fresh;
      a.counts[0] = (int)n_items;
      a.counts[1] = (int)n_work;
      a.counts[2] = (int)min((int64_t)a.attn_ctas, n_work);
    }
    if (bad) atomicOr(a.status, bad);
  }
  // where each attention CTA starts: CTA i takes the chunks [i W / C, (i + 1) W / C)
  const int first = rank * THREADS + tid, step = ctas * THREADS;
  const int C = (int)min((int64_t)a.attn_ctas, n_work);
  for (int i = first; i < C; i += step) {
    const int r = owner_of(cu_work, R, (int)share(i, n_work, C)), n_rows = cu_tok[r + 1] - cu_tok[r];
    int4* out = reinterpret_cast<int4*>(a.attn_start) + 2 * i;
    out[0] = make_int4(r, cu_work[r], len[r] >= 0 ? len[r] + n_rows : 0, n_rows);
    out[1] = make_int4(cu_tok[r], 0, 0, 0);
  }
  // the p-th page of request r after the step: from the stack if it is fresh
  bad = 0;
  auto page_of = [&](int r, int p) {
    const int used = (len[r] + page - 1) >> shift;
    const int id = p >= used ? a.free_pages[avail - 1 - (cu_fresh[r] + p - used)]
                             : a.block_table[(int64_t)r * a.table_width + p];
    if (id >= 0 && id < a.pages) return id;
    bad = TQ_PAGES_BAD_PAGE;
    return -1;
  };
  // touched pages; the fresh ones among them are all there are, and go into the table
  int4* items_out = reinterpret_cast<int4*>(a.items);
  for (int i = first; i < (int)n_items; i += step) {
    const int r = owner_of(cu_item, R, i), L0 = len[r], end = L0 + cu_tok[r + 1] - cu_tok[r];
    const int p = (L0 >> shift) + i - cu_item[r], id = page_of(r, p);
    const int lo = max(L0, p << shift), hi = min(end, (p + 1) << shift);
    if (p >= (L0 + page - 1) >> shift) a.block_table[(int64_t)r * a.table_width + p] = id;
    items_out[i] = make_int4(cu_tok[r] + lo - L0, hi - lo, lo - (p << shift), id);
  }
  // token rows: a warp takes 128 in a row, a lane every 32nd of them, so that stores are whole lines
  // and the four page look-ups are in flight together
  const int last = cu_tok[R], lane = tid & 31;
  for (int64_t t0 = (int64_t)(first >> 5) * 128 + lane; t0 < a.max_tokens; t0 += (int64_t)step * 4) {
    int pos[4], id[4], r = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t t = t0 + 32 * k;
      pos[k] = -1;
      if (t >= last) continue;
      if (r < 0 || t >= cu_tok[r + 1]) r = owner_of(cu_tok, R, (int)t);
      if (len[r] < 0) continue;
      pos[k] = len[r] + (int)t - cu_tok[r];
      id[k] = page_of(r, pos[k] >> shift);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t t = t0 + 32 * k;
      if (t >= a.max_tokens) break;
      a.slots[t] = pos[k] >= 0 && id[k] >= 0 ? ((int64_t)id[k] << shift) + (pos[k] & (page - 1)) : -1;
      a.positions[t] = pos[k];
    }
  }
  if (bad) atomicOr(a.status, bad);
}

// Pages of the finished requests back onto the stack, in request and page order; their lengths
// become 0 and their table entries -1.  An entry that is -1 already gives nothing back (a page that
// another request goes on reading was taken out of the row), so the places on the stack come from
// a running count of the entries that do.
//
// A page that is on the stack already must not get there twice: two requests would be given it.  So
// the stack is first read into a bit per page in shared memory (a pool of more pages than fit: a
// part of them at a time), and an entry whose bit is set, by the stack or by an earlier entry, is
// struck out and reported.  That needs no state beside the stack, whoever wrote it.
//
// Measured, in a captured sequence: 1.7 us if nothing ends, 3.7 us for one request of 2000 tokens in
// pages of 64 beside 2k free pages (2.4 without the marks), 15 us for one of 8000 tokens in pages of
// 16 beside 134k free ones (3.4): a shared-memory atomic per free page.
__global__ void __launch_bounds__(pl::THREADS) release_kernel(const uint8_t* __restrict__ finished, int* lengths,
                                                              int* block_table, int* free_pages, int* free_count,
                                                              int* status, int R, int W, int page, int P) {
  using namespace pl;
  extern __shared__ int sm[];
  int* cu = sm;  // [R + 1] table entries of the finished requests
  uint32_t* marks = reinterpret_cast<uint32_t*>(sm + R + 1);  // [min(P, MARKS) / 32, rounded up]
  __shared__ int64_t red[32];
  __shared__ int given[2][THREADS / 32];
  __shared__ int turn_ids[THREADS];
  grid_dep_wait();
  grid_dep_launch();
  const int per = (R + THREADS - 1) / THREADS, r0 = threadIdx.x * per;
  const int count = min(max(*free_count, 0), P);
  int held[PER];
  int64_t sum[1] = {0}, totals[1];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = r0 + i;
    held[i] = 0;
    if (i < per && r < R && finished[r])
      held[i] = (int)min(((int64_t)max(lengths[r], 0) + page - 1) / page, (int64_t)W);
    sum[0] += held[i];
  }
  block_scan<1>(sum, red, totals);
  int64_t at = sum[0];
  const int64_t total = totals[0];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = r0 + i;
    if (i < per && r < R) {
      cu[r] = (int)at;
      at += held[i];
      if (finished[r]) lengths[r] = 0;
      if (r == R - 1) cu[R] = (int)total;
    }
  }
  __syncthreads();
  for (int low = 0; low < P && total > 0; low += MARKS) {
    const int span = min(P - low, MARKS);
    for (int i = threadIdx.x; i < (span + 31) / 32; i += THREADS) marks[i] = 0u;
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += THREADS) {
      const uint32_t at = (uint32_t)free_pages[i] - (uint32_t)low;
      if (at < (uint32_t)span) atomicOr(&marks[at >> 5], 1u << (at & 31));
    }
    __syncthreads();
    for (int64_t i0 = 0; i0 < total; i0 += THREADS) {
      const int64_t i = i0 + threadIdx.x;
      int* e = nullptr;
      uint32_t at = (uint32_t)span;
      if (i < total) {
        const int r = owner_of(cu, R, (int)i);
        e = block_table + (int64_t)r * W + (i - cu[r]);
        at = (uint32_t)*e - (uint32_t)low;
      }
      const uint32_t bit = 1u << (at & 31);
      bool twice = at < (uint32_t)span && (marks[at >> 5] & bit);
      const bool mine = at < (uint32_t)span && !twice;
      __syncthreads();  // all have looked
      const bool met = mine && (atomicOr(&marks[at >> 5], bit) & bit);  // another of this turn has it too
      turn_ids[threadIdx.x] = mine ? (int)at : -1;
      if (__syncthreads_or(met)) {  // the first in order stays
        for (int j = 0; mine && !twice && j < (int)threadIdx.x; ++j) twice = turn_ids[j] == (int)at;
        __syncthreads();
      }
      if (twice) {
        *e = -1;
        atomicOr(status, TQ_PAGES_BAD_PAGE);
      }
    }
  }
  const int room = P - count, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t kept = 0;  // given back so far, the same in every thread
  int turn = 0;
  for (int64_t i0 = 0; i0 < total; i0 += THREADS, turn ^= 1) {
    const int64_t i = i0 + threadIdx.x;
    int id = -1;
    if (i < total) {
      const int r = owner_of(cu, R, (int)i);
      int* e = block_table + (int64_t)r * W + (i - cu[r]);
      id = *e;
      *e = -1;
      if (id < -1 || id >= P) {
        atomicOr(status, TQ_PAGES_BAD_PAGE);
        id = -1;
      }
    }
    const unsigned gives = __ballot_sync(0xffffffffu, id >= 0);
    if (lane == 0) given[turn][warp] = __popc(gives);
    __syncthreads();  // (two buffers: a warp that is a turn ahead writes the other one)
    int n = given[turn][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += y;
    }
    const int before = __shfl_sync(0xffffffffu, n, (warp + 31) & 31), all = __shfl_sync(0xffffffffu, n, 31);
    const int64_t place = kept + (warp ? before : 0) + __popc(gives & ((1u << lane) - 1u));
    if (id >= 0 && place < room) free_pages[count + place] = id;
    kept += all;
  }
  if (threadIdx.x == 0) {
    *free_count = count + (int)min((int64_t)room, kept);
    if (kept > room) atomicOr(status, TQ_PAGES_BAD_PAGE);  // (the stack itself held a page twice)
  }
}

// ------------------------------------------------------------------ cache write
// One unit is the new tokens of one touched page for one KV head, K and V each by itself.  With A
// the largest finite |x| among them, s_old the page's scale (0 if the page held nothing):
//   s = max(s_old, A / 127),  held codes q -> rint(q * (s_old / s)) if s > s_old,
//   new codes clamp(rint(x / s), -127, 127)
// with every operation a rounded f32 one, so the codes follow exactly.  NaN becomes 0 and an
// infinity the largest code of its sign.  A unit is one thread block: its rows stay in
// registers between the maximum and the codes, so x is read once, and nothing else writes that
// page and head.  A page of zeros has scale 0, which later tokens raise.
//
// With cos/sin, K is rotated first and the query heads are rotated by further blocks of the
// same launch (to q_out), with the decoder's roundings (decode_ops.cu's rope8).  A thread takes
// the values d and d + D/2 of a rotation pair together, so q_out may be q.
//
// Measured: 16.4k tokens of 8 KV heads of 128 (67 MB in, 34 MB out) 26 us, 3.9 TB/s or 0.59 of the
// measured copy rate; with the conversion to codes left out 18 us.  A block loads, meets a barrier,
// converts and stores, and nothing of the next unit is in flight meanwhile: the most frequent stall is
// the wait for loads, and the integer pipe is active for 47 % of the time.  64 decoding requests, 4 KV
// heads, with RoPE: 4.9 us, 0.3 of them since a call with too few rows is told (whichever block looks).
// Blocks of 128 or 512 threads 32 and 33 us.
namespace cw {
constexpr int THREADS = 256;
}

__device__ __forceinline__ int cache_code(float v, float s) {
  const float k = fminf(fmaxf(rintf(__fdiv_rn(v, s)), -127.0f), 127.0f);
  return v == v ? (int)k : 0;
}

// One rotation pair of 8-value pieces: lo holds x[d0 .. d0+8), hi x[d0+D/2 ..).
template <int XT>
__device__ __forceinline__ void rope_pair(uint4& lo, uint4& hi, const uint4 cl, const uint4 ch, const uint4 sl,
                                          const uint4 sh) {
  uint32_t* l = reinterpret_cast<uint32_t*>(&lo);
  uint32_t* h = reinterpret_cast<uint32_t*>(&hi);
  const uint32_t c0[4] = {cl.x, cl.y, cl.z, cl.w}, c1[4] = {ch.x, ch.y, ch.z, ch.w};
  const uint32_t s0[4] = {sl.x, sl.y, sl.z, sl.w}, s1[4] = {sh.x, sh.y, sh.z, sh.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t a = 0, b = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int sft = 16 * k;
      const float xl = h2f((uint16_t)(l[e] >> sft), XT), xh = h2f((uint16_t)(h[e] >> sft), XT);
      const float pl0 = round16(__fmul_rn(xl, h2f((uint16_t)(c0[e] >> sft), XT)), XT);
      const float pl1 = round16(__fmul_rn(-xh, h2f((uint16_t)(s0[e] >> sft), XT)), XT);
      const float ph0 = round16(__fmul_rn(xh, h2f((uint16_t)(c1[e] >> sft), XT)), XT);
      const float ph1 = round16(__fmul_rn(xl, h2f((uint16_t)(s1[e] >> sft), XT)), XT);
      a |= (uint32_t)f2h(__fadd_rn(pl0, pl1), XT) << sft;
      b |= (uint32_t)f2h(__fadd_rn(ph0, ph1), XT) << sft;
    }
    l[e] = a;
    h[e] = b;
  }
}

__device__ __forceinline__ uint4 ld16(const void* base, int64_t elem) {
  return *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + elem);
}

// The larger of m and the magnitudes' bits (magnitudes order like their bits), both halves apart.
__device__ __forceinline__ uint32_t max_bits(const uint4 v, uint32_t m) {
  constexpr uint32_t M = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(__vmaxu2(v.x & M, v.y & M), __vmaxu2(v.z & M, v.w & M)), m);
}

template <int XT>
__device__ __noinline__ float finite_absmax(const uint4 v, float m) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = fabsf(h2f((uint16_t)(w[e >> 1] >> ((e & 1) * 16)), XT));
    m = x < INFINITY ? fmaxf(m, x) : m;
  }
  return m;
}

// 8 codes by division (a call: it is rare, and its registers are not the caller's).
template <int XT>
__device__ __noinline__ uint2 codes8_divided(const uint4 v, float s) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    o[e >> 2] |= ((uint32_t)cache_code(h2f((uint16_t)(w[e >> 1] >> ((e & 1) * 16)), XT), s) & 255u) << ((e & 3) * 8);
  return make_uint2(o[0], o[1]);
}

// Two f32 at once.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 8 codes.  x * (1/s) is within 2^-15 of the rounded quotient where that is below 256, so its
// nearest integer is the quotient's unless it lies within 2^-14 of a tie; then, and for `odd` rows
// (values or a 1/s that are no finite numbers), the quotient itself decides.  Adding 1.5 * 2^23
// rounds to the nearest integer (ties to even) and leaves it in the low bits: nothing here runs on
// the conversion unit, which has a quarter of the rate.
template <int XT>
__device__ __forceinline__ uint2 codes8(const uint4 v, float s, float rs, bool odd) {
  constexpr float MAGIC = 12582912.0f, TIE = 0.5f - 6.103515625e-05f;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  const uint64_t rs2 = pair_of(rs, rs), up = pair_of(MAGIC, MAGIC), down = pair_of(-MAGIC, -MAGIC), neg = pair_of(-1.0f, -1.0f);
  uint32_t k[8];
  float off = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x0, x1;
    if constexpr (XT == TQ_DTYPE_BF16) {
      x0 = __uint_as_float(w[e] << 16);
      x1 = __uint_as_float(w[e] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      x0 = f.x;
      x1 = f.y;
    }
    const uint64_t t = mul2(pair_of(x0, x1), rs2), r = add2(t, up);
    const uint64_t d = fma2(add2(r, down), neg, t);  // t less the integer
    float d0, d1, r0, r1;
    split(d, d0, d1);
    split(r, r0, r1);
    off = fmaxf(off, fmaxf(fabsf(d0), fabsf(d1)));
    k[2 * e] = __float_as_uint(r0);
    k[2 * e + 1] = __float_as_uint(r1);
  }
  if (odd || off > TIE) return codes8_divided<XT>(v, s);
  return make_uint2(__byte_perm(__byte_perm(k[0], k[1], 0x0040), __byte_perm(k[2], k[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(k[4], k[5], 0x0040), __byte_perm(k[6], k[7], 0x0040), 0x5410));
}

// NP: rotation pairs of 8-value pieces a thread holds at most of each side (page * D / 16 / THREADS,
// 1 at least).  A block takes both sides of a page and head, all their rows in flight at once: with
// one side it waited most of its life on half the bytes.
template <int XT, int D, int NP>
__global__ void __launch_bounds__(cw::THREADS) cache_write_kernel(const tq_cache_write_args a, int unit_blocks) {
  using namespace cw;
  __shared__ float red[2][THREADS / 32];
  grid_dep_wait();
  grid_dep_launch();
  constexpr int H = D / 2, ppr = D / 16;  // pairs of pieces per row and head
  if ((int)blockIdx.x >= unit_blocks) {  // the query heads' rotation
    if (blockIdx.x == gridDim.x - 1) {  // one more block, which tells if the step has more tokens than rows
      if (threadIdx.x == 0 && a.cu_new[a.requests] > a.rows) atomicOr(a.status, TQ_PAGES_ROWS_FULL);
      return;
    }
    const uint32_t i = (blockIdx.x - unit_blocks) * (uint32_t)THREADS + threadIdx.x;  // (below 2^31: checked)
    const uint32_t rh = i / ppr, row = rh / (uint32_t)a.q_heads, head = rh - row * (uint32_t)a.q_heads;
    const bool there = (int)row < a.cu_new[a.requests];  // else behind the last token
    if ((int)row >= a.rows || !(there || (a.flags & TQ_CLEAR_REST))) return;
    const int d0 = i % ppr * 8;
    const int64_t src = (int64_t)row * a.ld_q + (int64_t)head * D + d0, cs = (int64_t)row * a.ld_cs + d0;
    uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
    if (there) {
      lo = ld16(a.q, src), hi = ld16(a.q, src + H);
      rope_pair<XT>(lo, hi, ld16(a.cos, cs), ld16(a.cos, cs + H), ld16(a.sin, cs), ld16(a.sin, cs + H));
    }
    uint16_t* dst = reinterpret_cast<uint16_t*>(a.q_out) + (int64_t)row * a.ld_qo + (int64_t)head * D + d0;
    *reinterpret_cast<uint4*>(dst) = lo;
    *reinterpret_cast<uint4*>(dst + H) = hi;
    return;
  }
  const int item = blockIdx.x / a.kv_heads, head = blockIdx.x - item * a.kv_heads;
  const int4 it = reinterpret_cast<const int4*>(a.items)[item];  // (the grid is not longer than the list)
  if (item >= a.counts[0]) return;
  const int row0 = it.x, n = it.y, off = it.z, pg = it.w;
  if (pg < 0 || pg >= a.pages || row0 < 0 || n < 1 || off < 0 || off + n > a.page || row0 + n > a.rows) {
    // (rows that are not there: the last block tells, and the page stays as it is)
    if (threadIdx.x == 0 && row0 + n <= a.rows) atomicOr(a.status, TQ_PAGES_BAD_PAGE);
    return;
  }
  uint4 lo[2][NP], hi[2][NP];
  bool odd[2];
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int i = threadIdx.x + j * THREADS;
      lo[side][j] = hi[side][j] = make_uint4(0u, 0u, 0u, 0u);
      if (i < n * ppr) {
        const int64_t src = (int64_t)(row0 + i / ppr) * (side ? a.ld_v : a.ld_k) + (int64_t)head * D + i % ppr * 8;
        lo[side][j] = ld16(side ? a.v : a.k, src);
        hi[side][j] = ld16(side ? a.v : a.k, src + H);
      }
    }
  const int64_t blk = (int64_t)pg * a.kv_heads + head;
  const float old_k = off ? a.k_scale[blk] : 0.0f, old_v = off ? a.v_scale[blk] : 0.0f;
  if (a.cos) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int i = threadIdx.x + j * THREADS;
      if (i < n * ppr) {
        const int64_t cs = (int64_t)(row0 + i / ppr) * a.ld_cs + i % ppr * 8;
        rope_pair<XT>(lo[0][j], hi[0][j], ld16(a.cos, cs), ld16(a.cos, cs + H), ld16(a.sin, cs), ld16(a.sin, cs + H));
      }
    }
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    uint32_t mb = 0u;
#pragma unroll
    for (int j = 0; j < NP; ++j) mb = max_bits(lo[side][j], max_bits(hi[side][j], mb));
    float m = h2f((uint16_t)max(mb & 0xffffu, mb >> 16), XT);
    odd[side] = !(m < INFINITY);
    if (odd[side]) {  // an infinity or a NaN among them: they do not set the scale
      m = 0.0f;
#pragma unroll
      for (int j = 0; j < NP; ++j) m = finite_absmax<XT>(lo[side][j], finite_absmax<XT>(hi[side][j], m));
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(m));  // (floats above 0 order like their bits)
    if ((threadIdx.x & 31) == 0) red[side][threadIdx.x >> 5] = __uint_as_float(top);
  }
  __syncthreads();  // also orders every thread's read of the scales before the writes below
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    float m = red[side][0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) m = fmaxf(m, red[side][w]);
    int8_t* codes = (side ? a.v_codes : a.k_codes) + blk * a.page * D;
    const float old = side ? old_v : old_k, mine = __fdiv_rn(m, 127.0f), s = fmaxf(old, mine);
    if (mine > old && off) {  // the scale grows: the codes the page holds follow
      const float ratio = __fdiv_rn(old, s);
      for (int i = threadIdx.x; i < off * D / 16; i += THREADS) {
        uint4 w = reinterpret_cast<uint4*>(codes)[i];
        uint32_t* p = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t o = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const float q = (float)(int8_t)(p[e] >> (8 * b));
            o |= ((uint32_t)(int)rintf(__fmul_rn(q, ratio)) & 255u) << (8 * b);
          }
          p[e] = o;
        }
        reinterpret_cast<uint4*>(codes)[i] = w;
      }
    }
    if (threadIdx.x == 0) (side ? a.v_scale : a.k_scale)[blk] = s;
    const float rs = __frcp_rn(s);
    if (!(rs < INFINITY)) odd[side] = true;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int i = threadIdx.x + j * THREADS;
      if (i < n * ppr) {
        int8_t* dst = codes + (off + i / ppr) * D + i % ppr * 8;
        uint2 cl = make_uint2(0u, 0u), ch = cl;
        if (s > 0.0f) {
          cl = codes8<XT>(lo[side][j], s, rs, odd[side]);
          ch = codes8<XT>(hi[side][j], s, rs, odd[side]);
        }
        *reinterpret_cast<uint2*>(dst) = cl;
        *reinterpret_cast<uint2*>(dst + H) = ch;
      }
    }
  }
}

// ------------------------------------------------------------------ pages read back
// code * scale in f32, rounded once to the 16-bit type; pages in the order of `ids`, an id
// outside the pool (-1 marks an unused table entry) gives zeros.  16 codes per thread.  Memory
// bound: 34 MB of codes to 67 MB in 18.5 us, 0.83 of the measured copy rate.
template <int XT>
__global__ void __launch_bounds__(256) read_pages_kernel(const int8_t* __restrict__ k, const int8_t* __restrict__ v,
                                                         const float* __restrict__ ks, const float* __restrict__ vs,
                                                         const int* __restrict__ ids, int64_t pieces, int block_shift,
                                                         uint32_t Hkv, int P, void* __restrict__ ko, void* __restrict__ vo) {
  grid_dep_wait();
  grid_dep_launch();
  const bool side = blockIdx.y;
  const int8_t* src = side ? v : k;
  const float* sc = side ? vs : ks;
  uint16_t* dst = reinterpret_cast<uint16_t*>(side ? vo : ko);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * blockDim.x) {
    const uint32_t unit = (uint32_t)(i >> block_shift), entry = unit / Hkv, head = unit - entry * Hkv;
    const int id = ids[entry];
    uint32_t o[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
    if (id >= 0 && id < P) {
      const int64_t blk = (int64_t)id * Hkv + head;
      const float s = sc[blk];
      const uint4 w = *reinterpret_cast<const uint4*>(src + ((blk << block_shift) + (i & ((1 << block_shift) - 1))) * 16);
      const uint32_t p[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // byte u = code + 128 under the bits of 2^23: the float 2^23 + u
        const float a = __uint_as_float(__byte_perm(p[e >> 1], 0x4b000000u, e & 1 ? 0x7652 : 0x7650)) - 8388736.0f;
        const float b = __uint_as_float(__byte_perm(p[e >> 1], 0x4b000000u, e & 1 ? 0x7653 : 0x7651)) - 8388736.0f;
        if constexpr (XT == TQ_DTYPE_BF16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(__fmul_rn(a, s), __fmul_rn(b, s));
          o[e] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(__fmul_rn(a, s), __fmul_rn(b, s));
          o[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
    }
    uint4* d = reinterpret_cast<uint4*>(dst + i * 16);
    d[0] = make_uint4(o[0], o[1], o[2], o[3]);
    d[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

}  // namespace tq

using namespace tq;

static bool good_page(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }

// A request with n >= 1 new tokens touches at most (n + page - 2) / page + 1 pages.
static int64_t most_items(int64_t tokens, int requests, int page) {
  const int64_t active = tokens < requests ? tokens : requests;
  return active + (tokens + active * (page - 2)) / page;
}

extern "C" int64_t tq_plan_items(int64_t max_tokens, int requests, int page) {
  if (max_tokens < 1 || max_tokens > INT32_MAX || requests < 1 || requests > TQ_MAX_REQUESTS || !good_page(page)) return 0;
  return most_items(max_tokens, requests, page);
}

extern "C" int tq_plan_step(const tq_plan_args* args, void* stream) {
  if (!args) return tq_set_error(TQ_ERR_INVALID, "null arguments");
  const tq_plan_args a = *args;
  if (a.requests < 1 || a.requests > TQ_MAX_REQUESTS)
    return tq_set_error(TQ_ERR_INVALID, "plan_step: 1..4096 requests");
  if (!good_page(a.page)) return tq_set_error(TQ_ERR_INVALID, "page size must be 16, 32, 64 or 128");
  if (a.table_width < 1 || a.pages < 1 || a.max_tokens < 1 || a.kv_heads < 1 || a.group < 1 || a.attn_ctas < 1 || a.attn_ctas > 4095)
    return tq_set_error(TQ_ERR_INVALID, "plan_step: sizes must be positive (and attn_ctas below 4096)");
  if (a.row_tile != 8 && a.row_tile != 16)
    return tq_set_error(TQ_ERR_INVALID, "plan_step: row_tile must be 8 or 16");
  if (!a.new_lens || !a.lengths || !a.lengths_out || !a.block_table || !a.free_pages || !a.free_count ||
      !a.free_count_out || !a.cu_new || !a.slots || !a.positions || !a.kv_len || !a.items || !a.counts || !a.cu_work ||
      !a.attn_start || !a.status)
    return tq_set_error(TQ_ERR_INVALID, "null pointer");
  if (((uintptr_t)a.items | (uintptr_t)a.attn_start) & 15)
    return tq_set_error(TQ_ERR_INVALID, "plan_step: items and attn_start must be 16-byte aligned");
  const int64_t room = (int64_t)a.table_width * a.page;
  // (keys are counted in 32 bits up to the end of a chunk, query rows up to the end of a tile)
  if (room > INT32_MAX - TQ_ATTN_CHUNK || (int64_t)a.pages * a.page > INT32_MAX)
    return tq_set_error(TQ_ERR_INVALID, "plan_step: more than 2^31 - 129 tokens in a request or 2^31 - 1 in the pool");
  if ((int64_t)a.max_tokens * a.group > INT32_MAX - a.row_tile)
    return tq_set_error(TQ_ERR_INVALID, "plan_step: too many query rows for one step (split the batch)");
  // the most attention chunks a step can have: rows are shared out over the requests
  const double tiles = (double)a.max_tokens * a.group / a.row_tile + a.requests;
  if (tiles * a.kv_heads * ((double)room / TQ_ATTN_CHUNK + 1 + TQ_ATTN_LEAD) > 2147483647.0)
    return tq_set_error(TQ_ERR_INVALID, "plan_step: too much attention work for one step (split the batch)");
  // a prefill's pages and rows are shared by up to eight CTAs (a cluster barrier costs about 1 us)
  int ctas = 1;
  while (ctas < 8 && ctas * 4096 < a.max_tokens) ctas *= 2;
  const int smem = (a.requests * 5 + 4) * 4;
  static std::atomic<uint64_t> done{0};
  TQ_CUDA_TRY(tq_allow_smem(plan_kernel, (TQ_MAX_REQUESTS * 5 + 4) * 4, done));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, 1, 1);
  cfg.blockDim = dim3(pl::THREADS, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = (cudaStream_t)stream;
  cfg.attrs = attr;
  cfg.numAttrs = tq_pdl_enabled() ? 2 : 1;
  TQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, plan_kernel, a));
  tq_count_launch();
  return TQ_OK;
}

extern "C" int tq_release_requests(const uint8_t* finished, int32_t* lengths, int32_t* block_table, int32_t* free_pages,
                                   int32_t* free_count, int32_t* status, int requests, int table_width, int page,
                                   int pages, void* stream) {
  if (requests < 1 || requests > TQ_MAX_REQUESTS)
    return tq_set_error(TQ_ERR_INVALID, "release_requests: 1..4096 requests");
  if (!good_page(page)) return tq_set_error(TQ_ERR_INVALID, "page size must be 16, 32, 64 or 128");
  if (table_width < 1 || pages < 1 || (int64_t)requests * table_width > INT32_MAX)
    return tq_set_error(TQ_ERR_INVALID, "release_requests: bad table width or page count");
  if (!finished || !lengths || !block_table || !free_pages || !free_count || !status)
    return tq_set_error(TQ_ERR_INVALID, "null pointer");
  static std::atomic<uint64_t> done{0};
  TQ_CUDA_TRY(tq_allow_smem(release_kernel, (TQ_MAX_REQUESTS + 1) * 4 + pl::MARKS / 8, done));
  const int smem = (requests + 1) * 4 + (std::min(pages, pl::MARKS) + 31) / 32 * 4;
  release_kernel<<<1, pl::THREADS, smem, (cudaStream_t)stream>>>(
      finished, lengths, block_table, free_pages, free_count, status, requests, table_width, page, pages);
  TQ_LAUNCHED();
  return TQ_OK;
}

template <int XT, int D>
static int launch_write(const tq_cache_write_args& a, cudaStream_t st) {
  const int64_t units = most_items(a.rows, a.requests, a.page) * a.kv_heads;
  const int64_t qb = a.cos ? ((int64_t)a.rows * a.q_heads * (D / 16) + cw::THREADS - 1) / cw::THREADS : 0;
  if (units > INT32_MAX / 2 || qb > INT32_MAX / cw::THREADS) return tq_set_error(TQ_ERR_INVALID, "cache_write: too many rows in one call");
  const int most = std::min(a.rows, a.page) * (D / 16);
  auto kern = most <= 256 ? cache_write_kernel<XT, D, 1>
                          : most <= 512 ? cache_write_kernel<XT, D, 2> : cache_write_kernel<XT, D, 4>;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units + qb + 1), 1, 1);
  cfg.blockDim = dim3(cw::THREADS, 1, 1);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = tq_pdl_enabled() ? 1 : 0;
  TQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, (int)units));
  tq_count_launch();
  return TQ_OK;
}

extern "C" int tq_cache_write(const tq_cache_write_args* args, int dtype, void* stream) {
  if (!args) return tq_set_error(TQ_ERR_INVALID, "null arguments");
  const tq_cache_write_args a = *args;
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_F16) return tq_set_error(TQ_ERR_INVALID, "dtype must be bf16 or f16");
  if (a.head_dim != 64 && a.head_dim != 128) return tq_set_error(TQ_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (!good_page(a.page)) return tq_set_error(TQ_ERR_INVALID, "page size must be 16, 32, 64 or 128");
  if (a.rows < 0 || a.requests < 1 || a.requests > TQ_MAX_REQUESTS || a.pages < 1 || a.kv_heads < 1)
    return tq_set_error(TQ_ERR_INVALID, "cache_write: bad sizes");
  if (a.flags & ~TQ_CLEAR_REST) return tq_set_error(TQ_ERR_INVALID, "cache_write: unknown flags");
  if (a.rows == 0) return TQ_OK;
  if (!a.k || !a.v || !a.k_codes || !a.v_codes || !a.k_scale || !a.v_scale || !a.items || !a.counts || !a.cu_new ||
      !a.status)
    return tq_set_error(TQ_ERR_INVALID, "null pointer");
  if (!a.cos != !a.sin || !a.cos != !a.q || !a.q != !a.q_out)
    return tq_set_error(TQ_ERR_INVALID, "cache_write: cos, sin, q and its output come together");
  const int64_t wk = (int64_t)a.kv_heads * a.head_dim;
  uintptr_t al = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.k_codes | (uintptr_t)a.v_codes | (uintptr_t)a.items;
  int64_t ls = a.ld_k | a.ld_v;
  if ((a.ld_k < wk || a.ld_v < wk) && a.rows > 1) return tq_set_error(TQ_ERR_INVALID, "cache_write: row stride too small");
  if (a.cos) {
    const int64_t wq = (int64_t)a.q_heads * a.head_dim;
    if (a.q_heads < 1) return tq_set_error(TQ_ERR_INVALID, "cache_write: bad sizes");
    if ((a.ld_q < wq || a.ld_qo < wq || (a.ld_cs < a.head_dim && a.ld_cs != 0)) && a.rows > 1)
      return tq_set_error(TQ_ERR_INVALID, "cache_write: row stride too small");
    al |= (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.cos | (uintptr_t)a.sin;
    ls |= a.ld_q | a.ld_qo | a.ld_cs;
  }
  if ((al & 15) || (ls & 7)) return tq_set_error(TQ_ERR_INVALID, "cache_write: rows must start on 16-byte boundaries");
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TQ_DTYPE_BF16)
    return a.head_dim == 128 ? launch_write<TQ_DTYPE_BF16, 128>(a, st) : launch_write<TQ_DTYPE_BF16, 64>(a, st);
  return a.head_dim == 128 ? launch_write<TQ_DTYPE_F16, 128>(a, st) : launch_write<TQ_DTYPE_F16, 64>(a, st);
}

extern "C" int tq_read_pages(const int8_t* k_codes, const int8_t* v_codes, const float* k_scale, const float* v_scale,
                             const int32_t* ids, int64_t n, int pages, int kv_heads, int page, int head_dim, void* k_out,
                             void* v_out, int dtype, void* stream) {
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_F16) return tq_set_error(TQ_ERR_INVALID, "dtype must be bf16 or f16");
  if (head_dim != 64 && head_dim != 128) return tq_set_error(TQ_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (!good_page(page)) return tq_set_error(TQ_ERR_INVALID, "page size must be 16, 32, 64 or 128");
  if (n < 0 || pages < 1 || kv_heads < 1) return tq_set_error(TQ_ERR_INVALID, "read_pages: bad sizes");
  if (n == 0) return TQ_OK;
  if (!k_codes || !v_codes || !k_scale || !v_scale || !ids || !k_out || !v_out)
    return tq_set_error(TQ_ERR_INVALID, "null pointer");
  if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_out | (uintptr_t)v_out) & 15)
    return tq_set_error(TQ_ERR_INVALID, "read_pages: pages and outputs must be 16-byte aligned");
  if (n * kv_heads > INT32_MAX) return tq_set_error(TQ_ERR_INVALID, "read_pages: too many pages in one call");
  const int per_block = page * head_dim / 16;  // a power of two
  const int64_t pieces = n * kv_heads * per_block;
  const int64_t want = (pieces + 255) / 256, most = (int64_t)tq_sm_count() * 8;
  const dim3 grid((unsigned)(want < most ? want : most), 2, 1);
  auto kern = dtype == TQ_DTYPE_BF16 ? read_pages_kernel<TQ_DTYPE_BF16> : read_pages_kernel<TQ_DTYPE_F16>;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = (cudaStream_t)stream;
  cfg.attrs = attr;
  cfg.numAttrs = tq_pdl_enabled() ? 1 : 0;
  TQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, k_codes, v_codes, k_scale, v_scale, ids, pieces, __builtin_ctz(per_block),
                                 (uint32_t)kv_heads, pages, k_out, v_out));
  tq_count_launch();
  return TQ_OK;
}
