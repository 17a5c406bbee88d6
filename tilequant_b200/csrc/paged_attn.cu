// Attention of a step's new tokens over the 8-bit paged cache (sm_100a).
//
// Request b has n_b new query tokens (rows cu_new[b] ..) and kv_b = kv_len[b] cached tokens, its
// new ones included; new token i sees the keys [0, kv_b - n_b + i].  With the page's scales
// a, c for K and V and codes k, v:
//   s = scale * a * (q . k),  p = 2^(s log2 e - m),  o = sum p * c * v / sum p
// in one pass over the keys with running m, sum and o (online softmax).  What bounds a step of
// few new tokens is the codes' bytes: 2 * kv_b * Hkv * D, read once for all query heads of a
// KV head and all new tokens that fit a row tile.
//
// Work split.  A chunk is 128 keys of one (request, KV head, row tile); the plan counted them
// (cu_work).  The grid is the blocks that fit the GPU at once, and block i takes the chunks
// [i W / C, (i + 1) W / C) of all W in a row, so every block has the same number whatever the
// requests' lengths.  A (request, head, row tile) inside one block goes straight to the output;
// one that spans blocks leaves partial (m, sum, o) in the workspace and the block that arrives
// last merges them in block order (so the result does not depend on who that is).  The arrival
// counter wraps to zero by itself.
//
// Within a block, warp w takes keys [32 w, 32 w + 32) of every chunk through a ring of its own:
// TMA boxes of K and V (128-byte swizzle), completion on the warp's mbarriers, three units in
// flight, no block barrier until a group of chunks ends.
//
// Tensor cores.  The *codes* are the 16-row operand of both products,
//   S^T [16 keys x 8 rows] = K q^T,   O^T [16 d x 8 rows] += V^T P^T
// so up to 8 query rows cost no padding (as the 16-row operand they would cost half).
// For bf16, S is exact integer arithmetic on the codes as they are: a query row, scaled by a power of
// two that brings its largest value to [2^14, 2^15), is rounded to 16-bit integers 256 hi + lo and
// multiplied as two int8 operands.  That keeps values down to 1/128 of the row's largest exactly,
// smaller ones to 2^-15 of the largest, and needs no conversion of K, which would be a quarter of the
// instructions.  For O the codes become exact f16 (a byte u under the pattern 0x64uu is 1024 + u) and
// P is rounded to f16, relative 2^-11: an eighth of a bf16 output's step (its sum takes P unrounded;
// with the rounded one the errors measure the same).  An f16 output's step is as
// small as those roundings, which cost up to 1.6 times the error of its own; so for f16 q is the f16
// operand as it is, over K's codes as f16, and P is two f16 numbers, the second what rounding the first
// left (64 requests 35.4 us against 32.9 with the bf16 form, drafts 46.6 against 41.5; error against
// 64 bits 2.07e-4 against 2.25e-4, for single requests 2.17e-4 against up to 3.3e-4: now the output's
// rounding alone).  The running maximum is lazy: it moves only when a score passes it by 2^5, so
// most units need no reduction across lanes and no rescaling; P is held as 2^10 p (at most 2^15),
// normal down to p = 2^-24.
// The reduction index of a product may be numbered freely as long as both operands agree, and so
// may the rows of O^T: thread t of a quad reads 32 consecutive bytes of its K row and thread
// group g 16 consecutive bytes of its V rows, each 16-byte shared load free of bank conflicts
// under the swizzle; pairs of keys for V^T are interleaved bytewise in registers.  P goes from
// the accumulator layout to the operand layout by an 8x8 transpose per 8 keys.
//
// Measured on one B200, per call of a captured sequence: 64 requests of 61 to 4096 keys (28 query /
// 4 KV heads of 128) 33.0 us for 137 MB, 4.2 TB/s or 0.63 of the measured copy rate; two requests
// of 98303 and 131071 keys (24 / 8 heads) 82.4 us for 470 MB, 0.87; 16 requests of up to 8190 keys
// with up to four new tokens (40 / 8 heads) 41.8 us for 143 MB, 0.52; one request of 513 keys 6.5
// us.  In the first, 2 us pass until the first load is issued (start record, table, page), 20 us at
// the memory's rate, and the rest with the ends of groups (a warp's join 0.6 us, an arrival 1.5 us,
// a merge 1.4 us) and blocks that have more of them.  With 16 query rows the instructions' latency
// at two warps per scheduler bounds it.  Tried and not kept: the row tile of 32 rows (spills, one
// block per SM: 122 us for the drafts), skipping idle halves of a 16-row tile (branches: 48 against
// 45 us), block barriers at the ends of groups (+5 us), the codes of K as f16 (no faster, a quarter
// more instructions), query rows prefetched into L1 and spinning waits (no gain).
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"
#include "tma.cuh"

namespace tq {
namespace pa {
constexpr int WARPS = 4;
constexpr int UNIT = 32;  // keys per warp and chunk
template <int NT>
constexpr int STAGES = NT == 1 ? 3 : 2;  // units in flight per warp: what lets two blocks share an SM
static_assert(WARPS * UNIT == TQ_ATTN_CHUNK, "the plan counts chunks of this size");
constexpr float P_BITS = 10.0f;  // P is held as 2^P_BITS p
constexpr float SLACK = 5.0f;    // by which a score may pass the running maximum
}  // namespace pa

struct PagedMaps {
  CUtensorMap k, v;  // [codes / 128][128] bytes, boxes of one page part, 128-byte swizzle
};

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
// Bytes (b0, b1) resp. (b2, b3) of a word of biased codes (code + 128) as two f16 codes.
__device__ __forceinline__ uint32_t sub1152(uint32_t h) {
  uint32_t r;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) { return sub1152(prmt(w, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) { return sub1152(prmt(w, 0x64646464u, 0x4342)); }

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// d += a (int8) * b (int8 or, LO, uint8)
template <bool LO>
__device__ __forceinline__ void mma_digit(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (LO)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    mma_s8_16832(d, a0, a1, a2, a3, b0, b1);
}

// Running softmax state of a warp: rows 8 j + 2 t + {0, 1}, for which this lane holds the D/8
// outputs d0 .. d0 + D/8 (d0 = lane / 4 * D / 8) as o[j][i][.] = (d0+2i, row 0), (d0+2i, row 1),
// (d0+2i+1, row 0), (d0+2i+1, row 1).
template <int D, int NT>
struct AttnState {
  static constexpr int MT = D / 16;
  static constexpr int WORDS = NT * (MT * 4 + 4);  // floats a lane parks in shared memory
  float o[NT][MT][4];
  float m[NT][2], l[NT][2];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      m[j][0] = m[j][1] = -INFINITY;
      l[j][0] = l[j][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.0f;
    }
  }
  // lane-major: conflict-free, and the reader has the writer's layout
  __device__ __forceinline__ void park(float* slot, int lane) const {
    float4* s = reinterpret_cast<float4*>(slot) + lane;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
        s[(j * (MT + 1) + i) * 32] = make_float4(o[j][i][0], o[j][i][1], o[j][i][2], o[j][i][3]);
      s[(j * (MT + 1) + MT) * 32] = make_float4(m[j][0], m[j][1], l[j][0], l[j][1]);
    }
  }
  __device__ __forceinline__ void join(const float* slot, int lane) {
    const float4* s = reinterpret_cast<const float4*>(slot) + lane;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float4 ml = s[(j * (MT + 1) + MT) * 32];
      const float om[2] = {ml.x, ml.y}, ol[2] = {ml.z, ml.w};
      float fa[2], fb[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float mn = fmaxf(m[j][q], om[q]);
        const float base = mn == -INFINITY ? 0.0f : mn;
        fa[q] = ex2(m[j][q] - base);
        fb[q] = ex2(om[q] - base);
        l[j][q] = l[j][q] * fa[q] + ol[q] * fb[q];
        m[j][q] = mn;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float4 v = s[(j * (MT + 1) + i) * 32];
        o[j][i][0] = o[j][i][0] * fa[0] + v.x * fb[0];
        o[j][i][1] = o[j][i][1] * fa[1] + v.y * fb[1];
        o[j][i][2] = o[j][i][2] * fa[0] + v.z * fb[0];
        o[j][i][3] = o[j][i][3] * fa[1] + v.w * fb[1];
      }
    }
  }
};

// A group whose partials this block merges, being the last to arrive.
struct Pending {
  int first, parts;              // the blocks that left partials
  int h, rq0, row0, tile_rows;   // KV head, first row of the tile, first token row, rows
};

// Merges a group's partials: a warp per row, lanes over D.  K rows (r, r + WARPS) and B parts of
// each are read at a time, so that one or two round trips to L2 serve a usual merge; the running
// maximum needs no pass of its own.  Small on purpose: a block runs it once, from a cold
// instruction cache.
template <int XT, int D, int ROWS, int K, int B>
__device__ __forceinline__ void merge_rows(const tq_paged_attn_args& a, const Pending& m, int G) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31;
  const float2* ws_ml = reinterpret_cast<const float2*>(a.ws_ml);
#pragma unroll 1
  for (int r = threadIdx.x >> 5; r < m.tile_rows; r += K * pa::WARPS) {
    float mx[K], sum[K], acc[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      mx[k] = -INFINITY;
      sum[k] = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[k][e] = 0.0f;
    }
#pragma unroll 1
    for (int p0 = 0; p0 < m.parts; p0 += B) {
      float o[K][B][V];
      float2 ml[K][B];
#pragma unroll
      for (int q = 0; q < B; ++q) {
        const int p = min(p0 + q, m.parts - 1);
        const int64_t slot = (2 * (int64_t)(m.first + p) + (p == 0 ? 1 : 0)) * ROWS;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int64_t at = slot + min(r + k * pa::WARPS, m.tile_rows - 1);
          ml[k][q] = __ldcg(&ws_ml[at]);
          const float* src = a.ws_o + at * D + lane * V;
          if constexpr (D == 128) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
            o[k][q][0] = v.x;
            o[k][q][1] = v.y;
            o[k][q][2] = v.z;
            o[k][q][3] = v.w;
          } else {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
            o[k][q][0] = v.x;
            o[k][q][1] = v.y;
          }
          if (p0 + q >= m.parts) ml[k][q] = make_float2(-INFINITY, 0.0f);
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float top = mx[k];
#pragma unroll
        for (int q = 0; q < B; ++q) top = fmaxf(top, ml[k][q].x);
        const float base = top == -INFINITY ? 0.0f : top, keep = ex2(mx[k] - base);
        mx[k] = top;
        sum[k] *= keep;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[k][e] *= keep;
#pragma unroll
        for (int q = 0; q < B; ++q) {
          const float f = ex2(ml[k][q].x - base);
          sum[k] = fmaf(ml[k][q].y, f, sum[k]);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[k][e] = fmaf(o[k][q][e], f, acc[k][e]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int row = r + k * pa::WARPS, rq = m.rq0 + row, tok = m.row0 + rq / G;
      if (row >= m.tile_rows || tok >= a.rows) continue;
      const float inv = sum[k] > 0.0f ? 1.0f / sum[k] : (sum[k] == 0.0f ? 0.0f : sum[k]);
      uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + (int64_t)tok * a.ld_out +
                                                  (int64_t)(m.h * G + rq % G) * D + lane * V);
#pragma unroll
      for (int e = 0; e < V / 2; ++e)
        dst[e] = (uint32_t)f2h(acc[k][2 * e] * inv, XT) | ((uint32_t)f2h(acc[k][2 * e + 1] * inv, XT) << 16);
    }
  }
}

// The block whose share [i W / C, (i + 1) W / C) holds chunk x: floor(((x + 1) C - 1) / W), in f64 for
// the reason given at share() (the quotient is below 2^12 and a fraction at least 2^-31).
__device__ __forceinline__ int64_t block_of(int64_t x, int64_t W, int64_t C) {
  return (int64_t)((double)((x + 1) * C - 1) / (double)W);
}

// Counts an arrival of `n`; true for the last.  Orders the warp's writes before it (they are the
// arriving lane's by the barrier) and its reads after it.
__device__ __forceinline__ bool arrive_last(uint32_t* count, int n) {
  __syncwarp();
  uint32_t old = 0;
  if ((threadIdx.x & 31) == 0)
    asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;" : "=r"(old) : "l"(count), "r"(n - 1) : "memory");
  old = __shfl_sync(0xffffffffu, old, 0);
  return old == (uint32_t)(n - 1);
}

// XT: the 16-bit type of q and out.  NT: tiles of 8 query rows.  PT: keys per page part (16 for
// 16-token pages, else 32): one scale pair each.
template <int XT, int D, int NT, int PT>
__global__ void __launch_bounds__(pa::WARPS * 32, 2)
    paged_attn_kernel(const tq_paged_attn_args a, const __grid_constant__ PagedMaps maps) {
  using namespace pa;
  using State = AttnState<D, NT>;
  constexpr int STG = STAGES<NT>, PARTS = UNIT / PT, KS = D / 32, MT = D / 16, ROWS = 8 * NT;
  constexpr int UB = UNIT * D;  // bytes of a unit's K (or V)
  constexpr int PB = PT * D;
  constexpr int SLOT = State::WORDS * 32;  // floats of a parked state
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[WARPS][STG];
  __shared__ __align__(8) uint64_t parked, taken;  // a group's three parked states written, read
  __shared__ int4 unit_i[WARPS][STG];    // KV head, row tile, 2 (chunk + lead) + (last of its group here), keys
  __shared__ int2 unit_r[WARPS][STG];    // first token row, token rows
  __shared__ float4 unit_f[WARPS][STG];  // K scales and V scales of the parts
  // groups to merge at the end: a block shares its first group with earlier blocks and its last with
  // later ones, and any other group is its own
  __shared__ Pending pending[2];  // the first, the last; parts 0: nothing to do
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (STG * 2 * UB);
  float* park = reinterpret_cast<float*>(smem + WARPS * STG * 2 * UB);  // 3 slots
  float2* ws_ml = reinterpret_cast<float2*>(a.ws_ml);

  if (lane == 0)
    for (int i = 0; i < STG; ++i) mbar_init(&full[warp][i], 1);
  if (threadIdx.x == 0) {
    mbar_init(&parked, WARPS - 1);
    mbar_init(&taken, 1);
    pending[0].parts = pending[1].parts = 0;
    prefetch_tensormap(&maps.k);
    prefetch_tensormap(&maps.v);
  }
  if (lane == 0) fence_mbar_init();
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();
  const int cta = blockIdx.x;
  // the request of the block's first chunk: its index, first chunk, keys, token rows, first row
  const int4 start = reinterpret_cast<const int4*>(a.attn_start)[2 * cta];
  const int start_row = a.attn_start[8 * cta + 4];
  const int64_t W = a.counts[1], C = a.counts[2];
  auto clear_rest = [&]() {  // rows behind the last token, a row per block and turn
    if (a.flags & TQ_CLEAR_REST)
      for (int row = a.cu_new[a.requests] + cta; row < a.rows; row += gridDim.x)
        for (int i = threadIdx.x; i < a.q_heads * (D / 8); i += WARPS * 32)
          reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + (int64_t)row * a.ld_out)[i] =
              make_uint4(0u, 0u, 0u, 0u);
  };
  if (cta >= C) {
    clear_rest();
    return;
  }
  const int64_t X0 = share(cta, W, C);
  const int steps = (int)(share(cta + 1, W, C) - X0);
  const int G = a.q_heads / a.kv_heads, R = a.requests;
  const int page_shift = 31 - __clz(a.page);

  // ---- the warp's units, 32 chunks at a time: lane i has chunk i of the batch
  int from = start.x;
  int my_h = 0, my_rt = 0, my_c = 0, my_kv = 0, my_row0 = 0, my_nv = 0;
  int my_y[PARTS];
  float my_ks[PARTS], my_vs[PARTS];
  auto load_batch = [&](int base) {
    const int64_t x = min(X0 + base + lane, X0 + steps - 1);
    int b = start.x, begin = start.y, kv = start.z, nv = start.w, row0 = start_row;
    int tiles = max(1, (nv * G + ROWS - 1) / ROWS), chunks = max(1, (kv + TQ_ATTN_CHUNK - 1) / TQ_ATTN_CHUNK);
    if (!__all_sync(0xffffffffu, x < begin + (int64_t)(chunks + TQ_ATTN_LEAD) * tiles * a.kv_heads)) {
      b = -1;  // the request of x: the last b with cu_work[b] <= x
      while (__any_sync(0xffffffffu, b < 0)) {
        const int e = from + 1 + lane;
        const int v = e <= R ? a.cu_work[e] : INT32_MAX;
        int n = 0;  // how many of the 32 ends are <= x
#pragma unroll
        for (int s = 16; s > 0; s >>= 1)
          if (__shfl_sync(0xffffffffu, v, n + s - 1) <= x) n += s;
        if (__shfl_sync(0xffffffffu, v, n) <= x) ++n;
        if (b < 0 && n < 32) b = from + n;
        if (from + 32 > R) {  // the plan's sums cover every chunk: not reached with an intact plan
          if (b < 0) b = R - 1;
          break;
        }
        if (__all_sync(0xffffffffu, b >= 0)) break;
        from += 32;
      }
      from = __shfl_sync(0xffffffffu, b, 31);
      begin = a.cu_work[b];
      kv = a.kv_len[b];
      row0 = a.cu_new[b];
      nv = a.cu_new[b + 1] - row0;
      tiles = max(1, (nv * G + ROWS - 1) / ROWS);
      chunks = max(1, (kv + TQ_ATTN_CHUNK - 1) / TQ_ATTN_CHUNK);
    }
    const int rel = (int)(x - begin), hr = rel / (chunks + TQ_ATTN_LEAD);
    const int c = rel - hr * (chunks + TQ_ATTN_LEAD) - TQ_ATTN_LEAD;  // negative: an empty one before the first
    my_h = hr / tiles;
    my_rt = hr - my_h * tiles;
    my_kv = kv;
    my_row0 = row0;
    my_nv = nv;
    int id[PARTS];
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      const int key = c * TQ_ATTN_CHUNK + warp * UNIT + j * PT;
      const bool there = c >= 0 && key < kv;
      id[j] = there ? a.block_table[(int64_t)b * a.table_width + (key >> page_shift)] : -1;
      if (there && (id[j] < 0 || id[j] >= a.pages || my_h >= a.kv_heads)) {
        atomicOr(a.status, TQ_PAGES_BAD_PAGE);  // its keys count as masked
        id[j] = -1;
      }
      my_y[j] = id[j] < 0 ? -1 : (int)((((int64_t)id[j] * a.kv_heads + my_h) * a.page + (key & (a.page - 1))) * D / 128);
    }
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      const int64_t blk = (int64_t)id[j] * a.kv_heads + my_h;
      my_ks[j] = id[j] >= 0 ? a.k_scale[blk] : 0.0f;
      my_vs[j] = id[j] >= 0 ? a.v_scale[blk] : -1.0f;  // -1: not loaded
    }
    my_c = 2 * (c + TQ_ATTN_LEAD) + (c >= 0 && (c == chunks - 1 || x == X0 + steps - 1));
  };
  bool ok = true;  // cleared when a load never lands: no further load is issued or awaited
  auto issue = [&](int i) {  // the loads of unit i
    const int st = i % STG;
    int y[PARTS];
    uint32_t bytes = 0;
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      y[j] = __shfl_sync(0xffffffffu, my_y[j], i & 31);
      bytes += y[j] >= 0 ? 2 * PB : 0;
    }
    if (lane == 0 && ok) {
      uint8_t* dst = ring + st * 2 * UB;
      mbar_expect_tx(&full[warp][st], bytes);
#pragma unroll
      for (int j = 0; j < PARTS; ++j)
        if (y[j] >= 0) {
          tma_load_2d(dst + j * PB, &maps.k, 0, y[j], &full[warp][st]);
          tma_load_2d(dst + UB + j * PB, &maps.v, 0, y[j], &full[warp][st]);
        }
    }
  };
  auto note = [&](int i) {  // what the reader of unit i needs (after issue: the scales may still be on their way)
    const int st = i % STG;
    if (lane == (i & 31)) {
      unit_i[warp][st] = make_int4(my_h, my_rt, my_c, my_kv);
      unit_r[warp][st] = make_int2(my_row0, my_nv);
      unit_f[warp][st] = make_float4(my_ks[0], my_ks[PARTS - 1], my_vs[0], my_vs[PARTS - 1]);
    }
    __syncwarp();
  };

  State S;
  // bf16: the digits of 4 values a word, step e has words 2 e, 2 e + 1; f16: the values, step e has ql[e], qh[e]
  uint32_t qh[NT][2 * KS], ql[NT][2 * KS];
  float qs[NT][2];   // score factor of the lane's two rows of each tile
  int lim[NT][2];    // keys the row sees
  int h = 0, rt = 0, kv = 0, nv = 0, row0 = 0, all_see = 0, group = 0;
  bool fresh = true;

  load_batch(0);
  for (int i = 0; i < min(STG, steps); ++i) issue(i);
  for (int i = 0; i < min(STG, steps); ++i) note(i);
  clear_rest();  // (while the first loads are on their way)
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    const int st = i % STG;
    const int4 ui = unit_i[warp][st];
    const int c = (ui.z >> 1) - TQ_ATTN_LEAD;
    const bool last = ui.z & 1;
    if (fresh && c >= 0) {  // a new (request, KV head, row tile): its query rows into operand registers
      fresh = false;
      h = ui.x;
      rt = ui.y;
      kv = ui.w;
      const int2 ur = unit_r[warp][st];
      row0 = ur.x;
      nv = ur.y;
      all_see = kv - nv + rt * ROWS / G + 1;
      S.clear();
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int r = rt * ROWS + 8 * j + g, tok = row0 + r / G;
        uint32_t w[D / 8];
        uint32_t amax = 0u;  // the largest magnitude's 16 bits (they order like the values)
        const bool there = r < nv * G && tok < a.rows;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)tok * a.ld_q +
                              (int64_t)(h * G + r % G) * D + t * (D / 4);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (there) v = *reinterpret_cast<const uint4*>(src + 8 * e);
          w[4 * e] = v.x;
          w[4 * e + 1] = v.y;
          w[4 * e + 2] = v.z;
          w[4 * e + 3] = v.w;
        }
#pragma unroll
        for (int e = 0; e < D / 8; ++e) amax = max(amax, max(w[e] & 0x7fffu, (w[e] >> 16) & 0x7fffu));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int ex = (int)(__float_as_uint(h2f((uint16_t)amax, XT)) >> 23);
        const int fe = min(268 - ex, 253);
        const float f = __uint_as_float((uint32_t)fe << 23);
        // a row with an infinity or a NaN gives NaN
        const float back = ex == 255 ? __uint_as_float(0x7fc00000u)
                                     : XT == TQ_DTYPE_F16 ? a.scale_log2
                                                          : __uint_as_float((uint32_t)(254 - fe) << 23) * a.scale_log2;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) {
          if constexpr (XT == TQ_DTYPE_F16) {  // as they are
            ql[j][e] = w[2 * e];
            qh[j][e] = w[2 * e + 1];
            continue;
          }
          int v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] = min(__float2int_rn(h2f((uint16_t)(w[2 * e + (k >> 1)] >> (16 * (k & 1))), XT) * f), 32767);
          const uint32_t x = prmt((uint32_t)v[0], (uint32_t)v[1], 0x5410), y = prmt((uint32_t)v[2], (uint32_t)v[3], 0x5410);
          ql[j][e] = prmt(x, y, 0x6420);
          qh[j][e] = prmt(x, y, 0x7531);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          qs[j][q] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * q);
          const int rq = rt * ROWS + 8 * j + 2 * t + q;
          lim[j][q] = rq < nv * G && kv > 0 ? kv - nv + rq / G + 1 : 0;
        }
      }
    }
    if (ok) {
      ok = __all_sync(0xffffffffu, mbar_wait_sleep(&full[warp][st], (uint32_t)((i / STG) & 1), a.err));
      if (!ok)  // the other loads in flight land (or give up) before the block may end
        for (int k = i + 1; k < min(i + STG, steps); ++k)
          mbar_wait_sleep(&full[warp][k % STG], (uint32_t)((k / STG) & 1), a.err);
    }
    const int k0 = c * TQ_ATTN_CHUNK + warp * UNIT;
    if (ok && c >= 0 && k0 < kv) {
      const float4 uf = unit_f[warp][st];
      const float ks[2] = {uf.x, uf.y}, vs[2] = {fmaxf(uf.z, 0.0f), fmaxf(uf.w, 0.0f)};
      const uint8_t* kb = ring + st * 2 * UB;
      const uint8_t* vb = kb + UB;
      // S^T = K q^T
      float s[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t w[2][D / 16];  // the lane's codes of keys g and g + 8
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const int key = mt * 16 + rr * 8 + g;
#pragma unroll
          for (int e = 0; e < D / 64; ++e) {
            uint32_t off;
            if constexpr (D == 128)
              off = (uint32_t)(key * 128 + (((2 * t + e) ^ (key & 7)) << 4));
            else
              off = (uint32_t)((key >> 1) * 128 + ((((key & 1) * 4 + t) ^ ((key >> 1) & 7)) << 4));
            const uint4 v = *reinterpret_cast<const uint4*>(kb + off);
            w[rr][4 * e] = v.x;
            w[rr][4 * e + 1] = v.y;
            w[rr][4 * e + 2] = v.z;
            w[rr][4 * e + 3] = v.w;
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float f[2] = {qs[j][0] * ks[PARTS == 2 ? mt : 0], qs[j][1] * ks[PARTS == 2 ? mt : 0]};
          if constexpr (XT == TQ_DTYPE_F16) {
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < D / 16; ++e) {
              const uint32_t x = w[0][e] ^ 0x80808080u, y = w[1][e] ^ 0x80808080u;
              mma_16816<TQ_DTYPE_F16>(acc, codes_lo(x), codes_lo(y), codes_hi(x), codes_hi(y), ql[j][e], qh[j][e]);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) s[mt][j][x] = acc[x] * f[x & 1];
          } else {
            int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < KS; ++e) {
              mma_digit<false>(hi, w[0][2 * e], w[1][2 * e], w[0][2 * e + 1], w[1][2 * e + 1], qh[j][2 * e], qh[j][2 * e + 1]);
              mma_digit<true>(lo, w[0][2 * e], w[1][2 * e], w[0][2 * e + 1], w[1][2 * e + 1], ql[j][2 * e], ql[j][2 * e + 1]);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) s[mt][j][x] = (float)(hi[x] * 256 + lo[x]) * f[x & 1];  // below 2^30: exact sums
          }
        }
      }
      // keys a row does not see, and keys of unloaded parts, are masked
      if (k0 + UNIT > all_see || uf.z < 0.0f || uf.w < 0.0f) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const bool gone = (mt && PARTS == 2 ? uf.w : uf.z) < 0.0f;
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (gone || k0 + mt * 16 + (x >> 1) * 8 + g >= lim[j][x & 1]) s[mt][j][x] = -INFINITY;
        }
      }
      bool past = false;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int q = 0; q < 2; ++q)
          past = past || fmaxf(fmaxf(s[0][j][q], s[0][j][2 + q]), fmaxf(s[1][j][q], s[1][j][2 + q])) > S.m[j][q] + SLACK;
      if (__any_sync(0xffffffffu, past)) {  // the maximum moves: what was summed follows
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float corr[2];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float mx = fmaxf(fmaxf(s[0][j][q], s[0][j][2 + q]), fmaxf(s[1][j][q], s[1][j][2 + q]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            mx = fmaxf(mx, S.m[j][q]);
            corr[q] = mx == S.m[j][q] ? 1.0f : ex2(S.m[j][q] - mx);
            S.m[j][q] = mx;
            S.l[j][q] *= corr[q];
          }
#pragma unroll
          for (int e = 0; e < MT; ++e) {
            S.o[j][e][0] *= corr[0];
            S.o[j][e][1] *= corr[1];
            S.o[j][e][2] *= corr[0];
            S.o[j][e][3] *= corr[1];
          }
        }
      }
      uint32_t pb[2][NT][2], pl[2][NT][2];  // P and, for f16 outputs, what its rounding left
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float base[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) base[q] = (S.m[j][q] == -INFINITY ? 0.0f : S.m[j][q]) - P_BITS;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int rr = 0; rr < 2; ++rr) {
            const float p0 = ex2(s[mt][j][2 * rr] - base[0]), p1 = ex2(s[mt][j][2 * rr + 1] - base[1]);
            S.l[j][0] += p0;
            S.l[j][1] += p1;
            const uint32_t p = half2_of(p0, p1);
            pb[mt][j][rr] = transpose8(p);
            if constexpr (XT == TQ_DTYPE_F16) {
              const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&p));
              pl[mt][j][rr] = transpose8(half2_of(p0 - r.x, p1 - r.y));
            }
          }
      }
      // O^T += V^T P^T, the scale on the part's product
      uint32_t w[2][4][D / 32];  // [16 keys][keys 2t, 2t + 1, 2t + 8, 2t + 9][the lane's D/8 codes]
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = mt * 16 + 2 * t + (e & 1) + (e >> 1) * 8;
          if constexpr (D == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(vb + key * 128 + ((g ^ (key & 7)) << 4));
            w[mt][e][0] = v.x;
            w[mt][e][1] = v.y;
            w[mt][e][2] = v.z;
            w[mt][e][3] = v.w;
          } else {
            const int r2 = key >> 1;
            const uint2 v = *reinterpret_cast<const uint2*>(
                vb + r2 * 128 + ((((key & 1) * 4 + (g >> 1)) ^ (r2 & 7)) << 4) + (g & 1) * 8);
            w[mt][e][0] = v.x;
            w[mt][e][1] = v.y;
          }
        }
#pragma unroll
      for (int e = 0; e < MT; ++e) {  // word e / 2 of the lane's codes, its bytes 2 (e & 1) and + 1
        const uint32_t sel = e & 1 ? 0x7362 : 0x5140;
        float acc[NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const uint32_t x = prmt(w[mt][0][e >> 1], w[mt][1][e >> 1], sel) ^ 0x80808080u;
          const uint32_t y = prmt(w[mt][2][e >> 1], w[mt][3][e >> 1], sel) ^ 0x80808080u;
          const uint32_t a0 = codes_lo(x), a1 = codes_hi(x), a2 = codes_lo(y), a3 = codes_hi(y);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (mt == 0 || PARTS == 2) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
            mma_16816<TQ_DTYPE_F16>(acc[j], a0, a1, a2, a3, pb[mt][j][0], pb[mt][j][1]);
            if constexpr (XT == TQ_DTYPE_F16)
              mma_16816<TQ_DTYPE_F16>(acc[j], a0, a1, a2, a3, pl[mt][j][0], pl[mt][j][1]);
            if (mt == 1 || PARTS == 2) {
              const float f = vs[PARTS == 2 ? mt : 0];
#pragma unroll
              for (int q = 0; q < 4; ++q) S.o[j][e][q] = fmaf(f, acc[j][q], S.o[j][e][q]);
            }
          }
        }
      }
    }
    __syncwarp();
    if (i + STG < steps) {
      if (((i + STG) & 31) == 0) load_batch(i + STG);
      issue(i + STG);
      note(i + STG);
    }
    if (!last) continue;

    // ---- the group ends here: one warp (another for each group) joins the other three's states,
    // which go on with the next group meanwhile
    fresh = true;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) S.l[j][q] += __shfl_xor_sync(0xffffffffu, S.l[j][q], x);
    const int chunks = max(1, (kv + TQ_ATTN_CHUNK - 1) / TQ_ATTN_CHUNK);
    const int64_t xf = X0 + i - c;  // the group's first chunk, in an earlier block if before X0
    const int first = (int)block_of(xf, W, C), parts = (int)block_of(xf + chunks - 1, W, C) - first + 1;
    const int joiner = group & 3, slot_id = (warp - joiner - 1) & 3;
    const uint32_t phase = (uint32_t)(group & 1);
    ++group;
    // the slots of the group before are read (the joiner waits too: a parity tells a phase only from
    // the next, so nobody may be two groups ahead of anybody)
    if (group > 1) mbar_wait_sleep(&taken, phase ^ 1, a.err);
    if (warp != joiner) {
      S.park(park + slot_id * SLOT, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(&parked);
      continue;
    }
    mbar_wait_sleep(&parked, phase, a.err);
    for (int k = 0; k < 3; ++k) S.join(park + k * SLOT, lane);
    __syncwarp();
    if (lane == 0) mbar_arrive(&taken);
    const int tile_rows = min(ROWS, nv * G - rt * ROWS);
    const int d0 = g * (D / 8);
    if (parts == 1) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int r = 8 * j + 2 * t + q, rq = rt * ROWS + r, tok = row0 + rq / G;
          if (r >= tile_rows || tok >= a.rows) continue;
          const float inv = S.l[j][q] > 0.0f ? 1.0f / S.l[j][q] : (S.l[j][q] == 0.0f ? 0.0f : S.l[j][q]);
          uint32_t w[MT];
#pragma unroll
          for (int e = 0; e < MT; ++e)
            w[e] = (uint32_t)f2h(S.o[j][e][q] * inv, XT) | ((uint32_t)f2h(S.o[j][e][2 + q] * inv, XT) << 16);
          uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + (int64_t)tok * a.ld_out +
                          (int64_t)(h * G + rq % G) * D + d0;
#pragma unroll
          for (int e = 0; e < MT / 4; ++e)
            reinterpret_cast<uint4*>(dst)[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
        }
      continue;
    }
    const int64_t slot = 2 * cta + (cta == first ? 1 : 0);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = 8 * j + 2 * t + q;
        if (r >= tile_rows) continue;
        float4* dst = reinterpret_cast<float4*>(a.ws_o + (slot * ROWS + r) * D + d0);
#pragma unroll
        for (int e = 0; e < MT / 2; ++e)
          dst[e] = make_float4(S.o[j][2 * e][q], S.o[j][2 * e][2 + q], S.o[j][2 * e + 1][q], S.o[j][2 * e + 1][2 + q]);
        if (g == 0) ws_ml[slot * ROWS + r] = make_float2(S.m[j][q], S.l[j][q]);
      }
    if (arrive_last(a.arrivals + first, parts) && lane == 0)
      pending[cta == first] = Pending{first, parts, h, rt * ROWS, row0, tile_rows};
  }
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const Pending m = pending[k];
    if (m.parts == 0) continue;
    if (m.tile_rows <= WARPS)
      merge_rows<XT, D, ROWS, 1, 16>(a, m, G);
    else
      merge_rows<XT, D, ROWS, 2, 4>(a, m, G);
  }
}

template <int D, int NT>
constexpr int paged_smem() {
  return pa::WARPS * pa::STAGES<NT> * 2 * pa::UNIT * D + 3 * AttnState<D, NT>::WORDS * 32 * 4;
}

}  // namespace tq

using namespace tq;

// Two blocks per SM are resident for every row tile and head size (the kernel's launch bounds; shared
// memory and registers of the head size 64 with 8 rows would hold three, which is not measured).
extern "C" int tq_paged_attn_ctas(int row_tile) {
  (void)row_tile;
  return 2 * tq_sm_count();
}

template <int XT, int D, int NT, int PT>
static int launch_paged(const tq_paged_attn_args& a, const PagedMaps& maps, cudaStream_t st) {
  auto kern = paged_attn_kernel<XT, D, NT, PT>;
  constexpr int smem = paged_smem<D, NT>();
  static std::atomic<uint64_t> done{0};
  TQ_CUDA_TRY(tq_allow_smem(kern, smem, done));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.attn_ctas, 1, 1);
  cfg.blockDim = dim3(pa::WARPS * 32, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = tq_pdl_enabled() ? 1 : 0;
  TQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, maps));
  tq_count_launch();
  return TQ_OK;
}

template <int XT, int D, int NT>
static int launch_paged_pt(const tq_paged_attn_args& a, const PagedMaps& maps, cudaStream_t st) {
  return a.page == 16 ? launch_paged<XT, D, NT, 16>(a, maps, st) : launch_paged<XT, D, NT, 32>(a, maps, st);
}

template <int XT, int D>
static int launch_paged_nt(const tq_paged_attn_args& a, const PagedMaps& maps, cudaStream_t st) {
  return a.row_tile == 8 ? launch_paged_pt<XT, D, 1>(a, maps, st) : launch_paged_pt<XT, D, 2>(a, maps, st);
}

extern "C" int tq_attn_paged(const tq_paged_attn_args* args, int dtype, void* stream) {
  if (!args) return tq_set_error(TQ_ERR_INVALID, "null arguments");
  const tq_paged_attn_args a = *args;
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_F16) return tq_set_error(TQ_ERR_INVALID, "dtype must be bf16 or f16");
  if (a.head_dim != 64 && a.head_dim != 128) return tq_set_error(TQ_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (a.page != 16 && a.page != 32 && a.page != 64 && a.page != 128)
    return tq_set_error(TQ_ERR_INVALID, "page size must be 16, 32, 64 or 128");
  if (a.row_tile != 8 && a.row_tile != 16)
    return tq_set_error(TQ_ERR_INVALID, "attn_paged: row_tile must be 8 or 16");
  if (a.rows < 0 || a.requests < 1 || a.requests > TQ_MAX_REQUESTS || a.pages < 1 || a.table_width < 1 ||
      a.kv_heads < 1 || a.q_heads < 1 || a.q_heads % a.kv_heads || a.attn_ctas < 1 || a.attn_ctas > 4095)
    return tq_set_error(TQ_ERR_INVALID, "attn_paged: bad sizes");
  if (a.flags & ~TQ_CLEAR_REST) return tq_set_error(TQ_ERR_INVALID, "attn_paged: unknown flags");
  if (a.rows == 0) return TQ_OK;
  if (!a.q || !a.out || !a.k_codes || !a.v_codes || !a.k_scale || !a.v_scale || !a.block_table || !a.cu_new ||
      !a.kv_len || !a.cu_work || !a.attn_start || !a.counts || !a.ws_o || !a.ws_ml || !a.arrivals || !a.status)
    return tq_set_error(TQ_ERR_INVALID, "null pointer");
  const int64_t width = (int64_t)a.q_heads * a.head_dim;
  if ((a.ld_q < width || a.ld_out < width) && a.rows > 1)
    return tq_set_error(TQ_ERR_INVALID, "attn_paged: row stride too small");
  if (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k_codes | (uintptr_t)a.v_codes | (uintptr_t)a.ws_o) & 15 ||
      ((a.ld_q | a.ld_out) & 7) || ((uintptr_t)a.ws_ml & 7) || ((uintptr_t)a.attn_start & 15))
    return tq_set_error(TQ_ERR_INVALID, "attn_paged: q, out, pages and workspace must start on 16-byte boundaries");
  const uint64_t lines = (uint64_t)a.pages * a.kv_heads * a.page * a.head_dim / 128;
  if (lines > INT32_MAX) return tq_set_error(TQ_ERR_UNSUPPORTED, "attn_paged: the pool is too large");
  const uint32_t box = (uint32_t)(std::min(a.page, pa::UNIT) * a.head_dim / 128);
  PagedMaps maps;
  int rc = tq_encode_2d(&maps.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.k_codes, 128, lines, 128, 128, box,
                        CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == TQ_OK)
    rc = tq_encode_2d(&maps.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.v_codes, 128, lines, 128, 128, box,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != TQ_OK) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TQ_DTYPE_BF16)
    return a.head_dim == 128 ? launch_paged_nt<TQ_DTYPE_BF16, 128>(a, maps, st)
                             : launch_paged_nt<TQ_DTYPE_BF16, 64>(a, maps, st);
  return a.head_dim == 128 ? launch_paged_nt<TQ_DTYPE_F16, 128>(a, maps, st)
                           : launch_paged_nt<TQ_DTYPE_F16, 64>(a, maps, st);
}
