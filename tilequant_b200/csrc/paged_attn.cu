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
// Tensor cores.  The codes become exact f16 (a byte u under the pattern 0x64uu is 1024 + u), the
// query rows are scaled by a power of two each so that f16's 11 bits hold bf16's 8 over 2^28 of
// range, and both products are f16 x f16 -> f32 with the *codes* as the 16-row operand:
//   S^T [16 keys x 8 rows] = K q^T,   O^T [16 d x 8 rows] += V^T P^T
// so up to 8 query rows cost no padding (as the 16-row operand they would cost half).  The
// reduction index of a product may be numbered freely as long as both operands agree, and so
// may the rows of O^T: thread t of a quad reads 32 consecutive bytes of its K row and thread
// group g 16 consecutive bytes of its V rows, each 16-byte shared load free of bank conflicts
// under the swizzle; pairs of keys for V^T are interleaved bytewise in registers.  P goes from
// the accumulator layout to the operand layout by an 8x8 transpose per 8 keys.  P is held as
// 2^14 p: the f16 rounding is relative (2^-11) down to p = 2^-28.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"
#include "tma.cuh"

namespace tq {
namespace pa {
constexpr int WARPS = 4;
constexpr int UNIT = 32;  // keys per warp and chunk
constexpr int STG = 3;    // units in flight per warp
static_assert(WARPS * UNIT == TQ_ATTN_CHUNK, "the plan counts chunks of this size");
constexpr float P_BITS = 14.0f;
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

// XT: the 16-bit type of q and out.  NT: tiles of 8 query rows.  PT: keys per page part (16 for
// 16-token pages, else 32): one scale pair each.
template <int XT, int D, int NT, int PT>
__global__ void __launch_bounds__(pa::WARPS * 32, NT <= 2 ? 2 : 1)
    paged_attn_kernel(const tq_paged_attn_args a, const __grid_constant__ PagedMaps maps) {
  using namespace pa;
  using State = AttnState<D, NT>;
  constexpr int PARTS = UNIT / PT, KC = D / 16, MT = D / 16, ROWS = 8 * NT;
  constexpr int UB = UNIT * D;  // bytes of a unit's K (or V)
  constexpr int PB = PT * D;
  constexpr int SLOT = State::WORDS * 32;  // floats of a parked state
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[WARPS][STG];
  __shared__ int4 unit_i[WARPS][STG];    // request, KV head, row tile, chunk (bit 31: last of its group here)
  __shared__ float4 unit_f[WARPS][STG];  // K scales and V scales of the parts
  __shared__ int is_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (STG * 2 * UB);
  float* park = reinterpret_cast<float*>(smem + WARPS * STG * 2 * UB);  // 3 slots
  float2* ws_ml = reinterpret_cast<float2*>(a.ws_ml);

  if (lane == 0) {
    for (int i = 0; i < STG; ++i) mbar_init(&full[warp][i], 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) {
    prefetch_tensormap(&maps.k);
    prefetch_tensormap(&maps.v);
  }
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();
  const int64_t W = a.counts[1], C = a.counts[2];
  const int cta = blockIdx.x;
  if (cta >= C) return;
  const int64_t X0 = cta * W / C;
  const int steps = (int)((cta + 1) * W / C - X0);
  const int G = a.q_heads / a.kv_heads, R = a.requests;

  // ---- the warp's units, 32 chunks at a time: lane i has chunk i of the batch
  int from = a.attn_start[cta];
  int my_b = 0, my_h = 0, my_rt = 0, my_c = 0;
  int my_y[PARTS];
  float my_ks[PARTS], my_vs[PARTS];
  auto load_batch = [&](int base) {
    const int64_t x = min(X0 + base + lane, X0 + steps - 1);
    my_b = -1;
    while (__any_sync(0xffffffffu, my_b < 0)) {  // the request of x: the last b with cu_work[b] <= x
      const int e = from + 1 + lane;
      const int v = e <= R ? a.cu_work[e] : INT32_MAX;
      int n = 0;  // how many of the 32 ends are <= x
#pragma unroll
      for (int s = 16; s > 0; s >>= 1)
        if (__shfl_sync(0xffffffffu, v, n + s - 1) <= x) n += s;
      if (__shfl_sync(0xffffffffu, v, n) <= x) ++n;
      if (my_b < 0 && n < 32) my_b = from + n;
      if (from + 32 > R) {  // the plan's sums cover every chunk: not reached with an intact plan
        if (my_b < 0) my_b = R - 1;
        break;
      }
      if (__all_sync(0xffffffffu, my_b >= 0)) break;
      from += 32;
    }
    from = __shfl_sync(0xffffffffu, my_b, 31);
    const int kv = a.kv_len[my_b];
    const int rows = (a.cu_new[my_b + 1] - a.cu_new[my_b]) * G;
    const int chunks = max(1, (kv + TQ_ATTN_CHUNK - 1) / TQ_ATTN_CHUNK);
    const int rel = (int)(x - a.cu_work[my_b]), hr = rel / chunks, tiles = max(1, (rows + ROWS - 1) / ROWS);
    my_c = rel - hr * chunks;
    my_h = hr / tiles;
    my_rt = hr - my_h * tiles;
    const bool last = my_c == chunks - 1 || x == X0 + steps - 1;
    int id[PARTS];
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      const int key = my_c * TQ_ATTN_CHUNK + warp * UNIT + j * PT;
      id[j] = -1;
      my_y[j] = -1;
      if (key < kv) {
        id[j] = a.block_table[(int64_t)my_b * a.table_width + key / a.page];
        if (id[j] < 0 || id[j] >= a.pages || my_h >= a.kv_heads) {
          atomicOr(a.status, TQ_PAGES_BAD_PAGE);  // its keys count as masked
          id[j] = -1;
        } else {
          my_y[j] = (int)((((int64_t)id[j] * a.kv_heads + my_h) * a.page + key % a.page) * D / 128);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      const int64_t blk = (int64_t)id[j] * a.kv_heads + my_h;
      my_ks[j] = id[j] >= 0 ? a.k_scale[blk] : 0.0f;
      my_vs[j] = id[j] >= 0 ? a.v_scale[blk] : 0.0f;
    }
    my_c |= last ? (int)0x80000000 : 0;
  };
  bool ok = true;  // cleared when a load never lands: no further load is issued or awaited
  auto produce = [&](int i) {
    const int st = i % STG, src = i & 31;
    if (src == 0) load_batch(i);
    if (lane == src) {
      unit_i[warp][st] = make_int4(my_b, my_h, my_rt, my_c);
      // a part that is not loaded is told by a V scale of -1
      unit_f[warp][st] = make_float4(my_ks[0], my_ks[PARTS - 1], my_y[0] < 0 ? -1.0f : my_vs[0],
                                     my_y[PARTS - 1] < 0 ? -1.0f : my_vs[PARTS - 1]);
    }
    int y[PARTS];
    uint32_t bytes = 0;
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      y[j] = __shfl_sync(0xffffffffu, my_y[j], src);
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
    __syncwarp();
  };

  State S;
  uint32_t qf[NT][KC][2];
  float qs[NT][2];   // score factor of the lane's two rows of each tile
  int lim[NT][2];    // keys the row sees
  int b = 0, h = 0, rt = 0, kv = 0, nv = 0, row0 = 0, all_see = 0;
  bool fresh = true;

  for (int i = 0; i < min(STG, steps); ++i) produce(i);
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    const int st = i % STG;
    if (ok) {
      ok = __all_sync(0xffffffffu, mbar_wait_sleep(&full[warp][st], (uint32_t)((i / STG) & 1), a.err));
      if (!ok)  // the other loads in flight land (or give up) before the block may end
        for (int k = i + 1; k < min(i + STG, steps); ++k)
          mbar_wait_sleep(&full[warp][k % STG], (uint32_t)((k / STG) & 1), a.err);
    }
    __syncwarp();
    const int4 ui = unit_i[warp][st];
    const int c = ui.w & 0x7fffffff;
    const bool last = ui.w < 0;
    if (fresh) {  // a new (request, KV head, row tile): its query rows into operand registers
      fresh = false;
      b = ui.x;
      h = ui.y;
      rt = ui.z;
      row0 = a.cu_new[b];
      nv = a.cu_new[b + 1] - row0;
      kv = a.kv_len[b];
      all_see = kv - nv + rt * ROWS / G + 1;
      S.clear();
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int r = rt * ROWS + 8 * j + g, tok = row0 + r / G;
        uint32_t w[D / 8];
        float amax = 0.0f;
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
        for (int e = 0; e < D / 8; ++e)
          amax = fmaxf(amax, fmaxf(fabsf(h2f((uint16_t)(w[e] & 0xffffu), XT)), fabsf(h2f((uint16_t)(w[e] >> 16), XT))));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // the power of two that brings the row's largest value to [2^13, 2^14); an infinity stays one
        const int ex = (int)(__float_as_uint(amax) >> 23);
        const int fe = ex == 255 ? 127 : min(267 - ex, 253);
        const float f = __uint_as_float((uint32_t)fe << 23);
        const float back = __uint_as_float((uint32_t)(254 - fe) << 23) * a.scale_log2;
#pragma unroll
        for (int e = 0; e < D / 8; ++e)
          qf[j][e >> 1][e & 1] =
              half2_of(h2f((uint16_t)(w[e] & 0xffffu), XT) * f, h2f((uint16_t)(w[e] >> 16), XT) * f);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          qs[j][q] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * q);
          const int rq = rt * ROWS + 8 * j + 2 * t + q;
          lim[j][q] = rq < nv * G && kv > 0 ? kv - nv + rq / G + 1 : 0;
        }
      }
    }
    const int k0 = c * TQ_ATTN_CHUNK + warp * UNIT;
    if (ok && k0 < kv) {
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
            w[rr][4 * e] = v.x ^ 0x80808080u;
            w[rr][4 * e + 1] = v.y ^ 0x80808080u;
            w[rr][4 * e + 2] = v.z ^ 0x80808080u;
            w[rr][4 * e + 3] = v.w ^ 0x80808080u;
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) s[mt][j][0] = s[mt][j][1] = s[mt][j][2] = s[mt][j][3] = 0.0f;
#pragma unroll
        for (int e = 0; e < KC; ++e) {
          const uint32_t a0 = codes_lo(w[0][e]), a1 = codes_lo(w[1][e]), a2 = codes_hi(w[0][e]), a3 = codes_hi(w[1][e]);
#pragma unroll
          for (int j = 0; j < NT; ++j)
            mma_16816<TQ_DTYPE_F16>(s[mt][j], a0, a1, a2, a3, qf[j][e][0], qf[j][e][1]);
        }
      }
      // scores in the log2 domain; keys a row does not see, and keys of unloaded parts, are masked
      const bool masked = k0 + UNIT > all_see || uf.z < 0.0f || uf.w < 0.0f;
      uint32_t pb[2][NT][2];
      bool grew = false;
      float corr[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float mx[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          mx[q] = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const float f = qs[j][q] * ks[PARTS == 2 ? mt : 0];
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
              float v = s[mt][j][2 * rr + q] * f;
              if (masked) {
                const int key = k0 + mt * 16 + rr * 8 + g;
                if (key >= lim[j][q] || (mt && PARTS == 2 ? uf.w : uf.z) < 0.0f) v = -INFINITY;
              }
              s[mt][j][2 * rr + q] = v;
              mx[q] = fmaxf(mx[q], v);
            }
          }
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], x));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], x));
        }
        float base[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float mn = fmaxf(S.m[j][q], mx[q]);
          grew = grew || mn > S.m[j][q];
          base[q] = (mn == -INFINITY ? 0.0f : mn) - P_BITS;
          corr[j][q] = ex2(S.m[j][q] - P_BITS - base[q]);  // 1 where the maximum stays
          S.m[j][q] = mn;
          S.l[j][q] *= corr[j][q];
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int rr = 0; rr < 2; ++rr) {
            const float p0 = ex2(s[mt][j][2 * rr] - base[0]), p1 = ex2(s[mt][j][2 * rr + 1] - base[1]);
            S.l[j][0] += p0;
            S.l[j][1] += p1;
            pb[mt][j][rr] = transpose8(half2_of(p0, p1));
          }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < MT; ++e) {
            S.o[j][e][0] *= corr[j][0];
            S.o[j][e][1] *= corr[j][1];
            S.o[j][e][2] *= corr[j][0];
            S.o[j][e][3] *= corr[j][1];
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
    if (i + STG < steps) produce(i + STG);
    if (!last) continue;

    // ---- the group ends here: the four warps' states into warp 0's
    fresh = true;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) S.l[j][q] += __shfl_xor_sync(0xffffffffu, S.l[j][q], x);
    if (warp >= 2) S.park(park + (warp - 2) * SLOT, lane);
    __syncthreads();
    if (warp < 2) S.join(park + warp * SLOT, lane);
    if (warp == 1) S.park(park + 2 * SLOT, lane);  // its own slot: warp 3 may already refill slot 1
    __syncthreads();
    const int chunks = max(1, (kv + TQ_ATTN_CHUNK - 1) / TQ_ATTN_CHUNK);
    const int64_t xf = X0 + i - c;  // the group's first chunk, in an earlier block if before X0
    const int first = (int)(((xf + 1) * C - 1) / W), end = (int)(((xf + chunks) * C - 1) / W);
    const int parts = end - first + 1;
    const int tile_rows = min(ROWS, nv * G - rt * ROWS);
    const int d0 = g * (D / 8);
    if (warp == 0) {
      S.join(park + 2 * SLOT, lane);
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
      } else {
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
        __threadfence();
        __syncwarp();
        if (lane == 0) is_last = atomicInc(a.arrivals + first, (unsigned)parts - 1) == (unsigned)parts - 1;
      }
    }
    if (parts == 1) continue;
    __syncthreads();
    const bool mine = is_last;
    __syncthreads();  // read before the next group's arrival may write it
    if (!mine) continue;
    __threadfence();
    // merge the blocks' partials: a warp per row, lanes over D
    for (int r = warp; r < tile_rows; r += WARPS) {
      float mx = -INFINITY;
      for (int p = lane; p < parts; p += 32) {
        const int64_t slot = 2 * (int64_t)(first + p) + (p == 0 ? 1 : 0);
        mx = fmaxf(mx, __ldcg(&ws_ml[slot * ROWS + r]).x);
      }
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float base = mx == -INFINITY ? 0.0f : mx;
      float acc[D / 32], sum = 0.0f;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] = 0.0f;
#pragma unroll 8
      for (int p = 0; p < parts; ++p) {
        const int64_t slot = 2 * (int64_t)(first + p) + (p == 0 ? 1 : 0);
        const float2 ml = __ldcg(&ws_ml[slot * ROWS + r]);
        const float f = ex2(ml.x - base);
        sum = fmaf(ml.y, f, sum);
        const float* src = a.ws_o + (slot * ROWS + r) * D + lane * (D / 32);
        if constexpr (D == 128) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
          acc[0] = fmaf(v.x, f, acc[0]);
          acc[1] = fmaf(v.y, f, acc[1]);
          acc[2] = fmaf(v.z, f, acc[2]);
          acc[3] = fmaf(v.w, f, acc[3]);
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          acc[0] = fmaf(v.x, f, acc[0]);
          acc[1] = fmaf(v.y, f, acc[1]);
        }
      }
      const int rq = rt * ROWS + r, tok = row0 + rq / G;
      if (tok >= a.rows) continue;
      const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
      uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + (int64_t)tok * a.ld_out +
                                                  (int64_t)(h * G + rq % G) * D + lane * (D / 32));
#pragma unroll
      for (int e = 0; e < D / 64; ++e)
        dst[e] = (uint32_t)f2h(acc[2 * e] * inv, XT) | ((uint32_t)f2h(acc[2 * e + 1] * inv, XT) << 16);
    }
  }
}

template <int D, int NT>
constexpr int paged_smem() {
  return pa::WARPS * pa::STG * 2 * pa::UNIT * D + 3 * AttnState<D, NT>::WORDS * 32 * 4;
}

}  // namespace tq

using namespace tq;

extern "C" int tq_paged_attn_ctas(int row_tile) {
  // the blocks resident at once: two per SM, one for the widest row tile (registers)
  return tq_sm_count() * (row_tile <= 16 ? 2 : 1);
}

template <int XT, int D, int NT, int PT>
static int launch_paged(const tq_paged_attn_args& a, const PagedMaps& maps, cudaStream_t st) {
  auto kern = paged_attn_kernel<XT, D, NT, PT>;
  constexpr int smem = paged_smem<D, NT>();
  TQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
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
  return a.row_tile == 8    ? launch_paged_pt<XT, D, 1>(a, maps, st)
         : a.row_tile == 16 ? launch_paged_pt<XT, D, 2>(a, maps, st)
                            : launch_paged_pt<XT, D, 4>(a, maps, st);
}

extern "C" int tq_attn_paged(const tq_paged_attn_args* args, int dtype, void* stream) {
  if (!args) return tq_set_error(TQ_ERR_INVALID, "null arguments");
  const tq_paged_attn_args a = *args;
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_F16) return tq_set_error(TQ_ERR_INVALID, "dtype must be bf16 or f16");
  if (a.head_dim != 64 && a.head_dim != 128) return tq_set_error(TQ_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (a.page != 16 && a.page != 32 && a.page != 64 && a.page != 128)
    return tq_set_error(TQ_ERR_INVALID, "page size must be 16, 32, 64 or 128");
  if (a.row_tile != 8 && a.row_tile != 16 && a.row_tile != 32)
    return tq_set_error(TQ_ERR_INVALID, "attn_paged: row_tile must be 8, 16 or 32");
  if (a.rows < 0 || a.requests < 1 || a.requests > TQ_MAX_REQUESTS || a.pages < 1 || a.table_width < 1 ||
      a.kv_heads < 1 || a.q_heads < 1 || a.q_heads % a.kv_heads || a.attn_ctas < 1)
    return tq_set_error(TQ_ERR_INVALID, "attn_paged: bad sizes");
  if (a.rows == 0) return TQ_OK;
  if (!a.q || !a.out || !a.k_codes || !a.v_codes || !a.k_scale || !a.v_scale || !a.block_table || !a.cu_new ||
      !a.kv_len || !a.cu_work || !a.attn_start || !a.counts || !a.ws_o || !a.ws_ml || !a.arrivals || !a.status)
    return tq_set_error(TQ_ERR_INVALID, "null pointer");
  const int64_t width = (int64_t)a.q_heads * a.head_dim;
  if ((a.ld_q < width || a.ld_out < width) && a.rows > 1)
    return tq_set_error(TQ_ERR_INVALID, "attn_paged: row stride too small");
  if (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k_codes | (uintptr_t)a.v_codes | (uintptr_t)a.ws_o) & 15 ||
      ((a.ld_q | a.ld_out) & 7) || ((uintptr_t)a.ws_ml & 7))
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
