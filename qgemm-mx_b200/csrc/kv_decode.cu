// kv_decode.cu -- attention over the paged 8-bit cache for few query rows per
// KV head (decoding, speculative tokens); no counterpart in
// titoatwork/qgemm-mx.  Arithmetic: kv_attention.cuh.
//
// What bounds it: HBM.  Every K and V code is read once, one byte for 2 to
// 2 x rows multiply-adds, so the kernel is built around the copy: each warp
// streams its own tiles of 16 tokens through a private ring that one lane
// fills by TMA (2 copies a tile, swizzled), and meets no barrier of the CTA
// until its tokens are done.
//
// Split.  A pair is (request, KV head, group of 8 NT rows); its tokens are
// tiles of 16.  All pairs' tiles form one line that is cut into equal shares,
// one per warp of the grid, wherever the cuts fall, so ragged batches and a
// single long request load the GPU alike.  A share that holds a whole pair
// writes its output; the others leave (O, m, l) partials that the CTA
// joins in shared memory, and pairs that cross CTAs are joined by the
// last CTA to arrive at a ticket, in CTA order, so results do not depend on
// timing.
//
// Tile arithmetic (transposed, so that 8 query rows fill an MMA's N side):
//   S^T[16 tokens x 8 rows] = K . q^T     A = K codes widened to f16
//   O^T[dims x 8 rows]     += V^T . W^T   A = V codes, pairs of tokens by prmt
// mma.sync m16n8k16 with 32-bit accumulators.  The token order inside a tile
// and the dims inside an MMA are permuted so that every shared-memory read is
// a conflict-free 128-bit (64-bit for V at 64 dims) load of the swizzled
// bytes.  With 2 x 8 rows per byte the tensor work is an eighth of what the
// legacy MMA path sustains beside the copy, so tcgen05's TMEM round trips
// would buy nothing here.
//
// Every mbarrier wait is bounded; on a timeout the kernel sets
// g_kv_decode_fault, finishes its joins without waiting and returns
// (qgemm_umma_status reports it).
#include "gemv_core.cuh"
#include "kv_attention.cuh"
#include "tc.cuh"

namespace qg {

__device__ unsigned g_kv_decode_fault = 0;

constexpr int kDecRequests = 1024;  // of a launch: they are kept in shared memory
// Shares end with whole pairs where those have at most so many places and the
// fullest share then gets at most so many more than the mean.
constexpr int kDecSnapLongest = 40, kDecSnapOver = 13;
constexpr float kDecLow = -1e30f;  // m before a row has seen a token

template <int HD, int NT>
struct DecCfg {
  static constexpr int kStage = 2 * 16 * HD;  // K and V of 16 tokens
  static constexpr int kWarps = NT == 1 ? 12 : 8;
  static constexpr int kStages = HD == 128 ? (NT == 1 ? 3 : 4) : (NT == 1 ? 6 : 8);
  static constexpr int kSlot = 8 * NT * (HD + 2);  // floats of a partial: O, m, l
  static constexpr int kRing = kStages * kStage;
  // alignment | rings (a warp's last partial reuses its own) | first partials
  static constexpr int kSmem = 1024 + kWarps * (kRing + kSlot * 4);
};

// Byte of 16-byte chunk `ch` of token row `row` in a tile, as TMA's 128-byte
// (64-byte) swizzle leaves it.
template <int HD>
__device__ __forceinline__ int tile_off(int row, int ch) {
  return HD == 128 ? row * 128 + ((ch ^ (row & 7)) << 4) : row * 64 + ((ch ^ ((row >> 1) & 3)) << 4);
}
// Token row of MMA row (and k index) i < 8; 8 + i is 8 rows on.  K's reads take
// rows tau(2i), tau(2i + 1) and chunks 0-3 (4-7) together, V's rows tau(2t) of
// four t and two chunks: these orders give them 8 bank groups each.
template <int HD>
__device__ __forceinline__ int tau(int i) {
  const int r = HD == 128 ? (i & 6) : ((i >> 1) & 1) | (i & 4);  // tau(2t): 0 2 4 6, or 0 1 4 5
  return (i & 1) ? (HD == 128 ? r ^ 5 : r ^ 3) : r;
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint4 lds16(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
  return v;
}

template <int TYPE, int HD, int NT>
__global__ void __launch_bounds__(DecCfg<HD, NT>::kWarps * 32, 1)
k_kv_decode(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const KvAttnArgs a) {
  using Cfg = DecCfg<HD, NT>;
  constexpr int RG = 8 * NT, KJ = HD / 64, MT = HD / 16, ST = Cfg::kStages, W = Cfg::kWarps;
  extern __shared__ uint8_t smem_raw[];
  __shared__ KvBatch<kDecRequests> s_batch;
  __shared__ int s_scan[2 * W];
  __shared__ __align__(1024) uint64_t s_bars[W * ST];
  __shared__ int s_cell[W * ST];   // a stage's (block, head)
  __shared__ int2 s_part[2 * W];   // the pair each partial belongs to: its range on the line
  __shared__ int4 s_rows[2 * W];   // and its rows: first token row, first row, rows, head
  __shared__ int4 s_cross[2];              // pairs that cross CTAs: begun before this CTA, begun in it
  __shared__ int2 s_joins[2];              // the CTAs of those that this CTA joins
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t raw = su32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);

  if (tid < 2 * W) s_part[tid] = make_int2(-1, -1);
  if (tid < 2) s_cross[tid] = make_int4(-1, -1, 0, 0);
  if (lane == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(su32(&s_bars[warp * ST + i]), 1);
      s_cell[warp * ST + i] = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  kv_tell(a);
  pdl_launch_dependents();
  int longest;
  const int V = kv_line<RG, 4, W>(a, s_batch, s_scan, longest);
  const int E = max(1, min((int)gridDim.x * W, V));  // shares
  const int k0 = blockIdx.x * W;
  if (V == 0 || k0 >= E) return;
  // Short pairs are not cut where that keeps the shares even: a share takes the
  // pairs that begin in it, which costs the fullest one some tiles and saves
  // joining nearly every pair.  Requests x tokens, 8 KV heads of 128: 200 x 100
  // 14.7 us instead of 27.3, 200 x 500 41 instead of 52, 64 x 200 18.4 and 18.2;
  // uneven and so cut: 64 x 300 20.5 instead of 24.2, 64 x 500 24 instead of 31.
  const int mean = V / E;
  const bool snap = longest <= kDecSnapLongest && (mean + longest - 1) / longest * longest - mean <= kDecSnapOver;
  const KvCuts cuts(V, E);

  const uint32_t ring = base + warp * Cfg::kRing;
  float* const last_part = reinterpret_cast<float*>(smem + warp * Cfg::kRing);
  float* const first_part = reinterpret_cast<float*>(smem + W * Cfg::kRing) + warp * Cfg::kSlot;
  const float inv_group = 1.0f / (float)a.group;
  // row / group for the few rows of this kernel (exact below 2^21)
  auto token_of = [&](int row) { return (int)(((float)row + 0.5f) * inv_group); };
  bool ok = true;

  if (k0 + warp < E) {
    const int v0 = cuts.at(k0 + warp), v1 = cuts.at(k0 + warp + 1);
    // ---- producer state: runs ST tiles ahead of the arithmetic --------------
    int p_v = v0, p_r = kv_find(s_batch, a.requests, v0);
    int c_r = p_r;  // the arithmetic's place
    KvSeg s;
    kv_seg<RG, 4>(a, s_batch, c_r, v0, snap ? INT32_MAX : v1, s);
    const bool skip = snap && s.pair_v < v0;  // begun in the share before
    if (skip) p_v = s.pair_end;
    KvSeg ps = s;
    ps.tile = 0; ps.tile_end = 0;
    int win = 0, win_end = 0, win_id = -1;  // 32 block ids from `win` on, one per lane
    uint32_t outside = 0;  // stages whose block is outside the pool, one bit each
    const int lg = a.block_log2;
    auto issue = [&](int stage) {
      while (ps.tile >= ps.tile_end) {
        if (p_v >= v1) return;
        kv_seg<RG, 4>(a, s_batch, p_r, p_v, snap ? INT32_MAX : v1, ps);
        p_v = snap ? ps.pair_end : min(ps.pair_end, v1);
        win_end = 0;
      }
      const int tok = ps.tile * 16, page = tok >> lg;
      if (page >= win_end) {
        win = page;
        win_end = page + 32;
        const int p = page + lane;
        win_id = ((long long)p << lg) < ps.len ? a.table[(size_t)ps.r * a.width + p] : -1;
        if (win_id < 0 || win_id >= a.blocks) win_id = -1;  // before it is multiplied
      }
      const int id = __shfl_sync(0xFFFFFFFFu, win_id, page - win);
      outside = (outside & ~(1u << stage)) | ((uint32_t)(id < 0) << stage);
      if (lane == 0) {
        const uint32_t bar = su32(&s_bars[warp * ST + stage]), dst = ring + stage * Cfg::kStage;
        const int cell = id * a.heads + ps.h;
        // a block outside the pool: rows in front of it, which TMA fills with zeros
        const int y = id < 0 ? -16 : (cell << lg) + (tok & ((1 << lg) - 1));
        s_cell[warp * ST + stage] = max(cell, 0);
        mbar_expect_tx(bar, Cfg::kStage);
        tma_load_2d(dst, &map_k, 0, y, bar);
        tma_load_2d(dst + 16 * HD, &map_v, 0, y, bar);
      }
      ++ps.tile;
    };
    // queries of a stretch: this lane's part of row g of each tile of 8
    auto load_q = [&](const KvSeg& s, uint4 (&w)[NT][KJ][2]) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int row = s.row0 + nt * 8 + g, i = token_of(row), gh = row - i * a.group;
        const uint16_t* qp = a.q + (int64_t)(s.start + i) * a.q_stride + (int64_t)(s.h * a.group + gh) * a.q_head_stride;
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            w[nt][j][x] = row < s.rows ? ld16(reinterpret_cast<const uint4*>(qp + (t + 4 * j) * 16) + x)
                                       : make_uint4(0, 0, 0, 0);
      }
    };
    uint4 qw[NT][KJ][2];
    if (!skip) load_q(s, qw);  // in flight while the ring fills
#pragma unroll 1
    for (int i = 0; i < ST; ++i) issue(i);

    // ---- fixed shared-memory offsets of this lane ---------------------------
    const int tg = tau<HD>(g);  // token row of MMA row g
    uint32_t k_off[2][KJ], v_off[4];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int j = 0; j < KJ; ++j) k_off[hh][j] = tile_off<HD>(tg + 8 * hh, t + 4 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = tau<HD>(2 * t + (i & 1)) + (i >> 1) * 8;
      v_off[i] = 16 * HD + (HD == 128 ? tile_off<HD>(row, g) : tile_off<HD>(row, g >> 1) + (g & 1) * 8);
    }

    int stage = 0;
    uint32_t parity = 0;
    bool first = true;
    // exponents of a stage's blocks, K's | V's << 8: loaded a tile ahead
    auto load_exp = [&](int stage) {
      const int cell = s_cell[warp * ST + stage];
      return (uint32_t)a.ks[cell] | ((uint32_t)a.vs[cell] << 8);
    };
    __syncwarp();
    uint32_t mt_next = load_exp(0);
    for (int v = skip ? s.pair_end : v0; v < v1;) {
      const int seg_v0 = v;
      if (v > v0) {
        kv_seg<RG, 4>(a, s_batch, c_r, v, snap ? INT32_MAX : v1, s);
        load_q(s, qw);
      }
      v = snap ? s.pair_end : min(s.pair_end, v1);
      // ---- queries: f16 fragments and score factors --------------------------
      uint32_t qf[NT][KJ][8];
      float fac[NT][2], m[NT][2], l[NT][2];
      int lo_t[NT][2], hi_t[NT][2];
      float o[NT][MT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t mx = 0;
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t u[4] = {qw[nt][j][x].x, qw[nt][j][x].y, qw[nt][j][x].z, qw[nt][j][x].w};
#pragma unroll
            for (int y = 0; y < 4; ++y) mx = max(mx, max(u[y] & 0x7FFFu, (u[y] >> 16) & 0x7FFFu));
          }
        mx = max(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
        // exponent of the row's largest value; rows with inf or NaN keep theirs
        const int e = mx >= 0x7F80u || mx < 0x0080u ? 0 : min((int)(mx >> 7) - 127, 126);
        const float down = pow2f(-e);
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t u[4] = {qw[nt][j][x].x, qw[nt][j][x].y, qw[nt][j][x].z, qw[nt][j][x].w};
#pragma unroll
            for (int y = 0; y < 4; ++y)
              qf[nt][j][x * 4 + y] = pack_f16(u2f(u[y] << 16) * down, u2f(u[y] & 0xFFFF0000u) * down);
          }
        const float fq = a.scale_log2 * pow2f(e);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = 2 * t + c;
          fac[nt][c] = __shfl_sync(0xFFFFFFFFu, fq, col * 4);
          const int ci = token_of(min(s.row0 + nt * 8 + col, s.rows - 1));
          lo_t[nt][c] = row_lo(a, s.len, s.n_all, ci);
          hi_t[nt][c] = row_hi(a, s.len, s.n_all, ci);
          m[nt][c] = kDecLow;
          l[nt][c] = 0.0f;
        }
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) o[nt][x][y] = 0.0f;
      }
      // tiles every row of the group sees whole need no mask
      const int full_lo = row_lo(a, s.len, s.n_all, token_of(min(s.row0 + RG, s.rows) - 1));
      const int full_hi = row_hi(a, s.len, s.n_all, token_of(s.row0));

      // ---- tiles ----------------------------------------------------------------
#pragma unroll 1
      for (int tile = s.tile; tile < s.tile_end && ok; ++tile) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_flag(su32(&s_bars[warp * ST + stage]), parity, &g_kv_decode_fault));
        if (!ok) break;
        const uint32_t sb = ring + stage * Cfg::kStage;
        const uint32_t mt = outside >> stage & 1u ? 0x7F7Fu : mt_next;  // 2^0 beside the zeros outside the pool
        float sc[NT][2][4];
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const uint4 k0v = lds16(sb + k_off[0][j]), k1v = lds16(sb + k_off[1][j]);
          const uint32_t kw[2][4] = {{k0v.x, k0v.y, k0v.z, k0v.w}, {k1v.x, k1v.y, k1v.z, k1v.w}};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            codes4_to_f16<TYPE>(kw[0][i], a0, a2);
            codes4_to_f16<TYPE>(kw[1][i], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (j == 0 && i < 2) mma_f16_z(sc[nt][i], a0, a1, a2, a3, qf[nt][j][2 * i], qf[nt][j][2 * i + 1]);
              else mma_f16(sc[nt][i & 1], a0, a1, a2, a3, qf[nt][j][2 * i], qf[nt][j][2 * i + 1]);
            }
          }
        }
        uint32_t vw[4][HD / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (HD == 128) {
            const uint4 x = lds16(sb + v_off[i]);
            vw[i][0] = x.x; vw[i][1] = x.y; vw[i][HD / 32 - 2] = x.z; vw[i][HD / 32 - 1] = x.w;
          } else {
            const uint2 x = lds8(sb + v_off[i]);
            vw[i][0] = x.x; vw[i][1] = x.y;
          }
        }
        const float ksc = u2f((mt & 0xFFu) << 23);
        const int vexp = (int)((mt >> 8) & 0xFFu) - 127;
        const float ev = (float)vexp, inv = pow2f(-vexp);
        float f[NT][2], p[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 2; ++c) f[nt][c] = fac[nt][c] * ksc;
#pragma unroll
          for (int y = 0; y < 4; ++y) sc[nt][0][y] += sc[nt][1][y];
        }
        const int tok = tile * 16;
        const bool mask = tok < full_lo || tok + 16 > full_hi;
        bool hide[NT][4];
        if (mask) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int at = tok + tg + (y >> 1) * 8;
              hide[nt][y] = at < lo_t[nt][y & 1] || at >= hi_t[nt][y & 1];
            }
          // what lies behind the last token is not the request's: its codes may be NaN
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (tok + tau<HD>(2 * t + (i & 1)) + (i >> 1) * 8 >= s.len) {
#pragma unroll
              for (int w = 0; w < HD / 32; ++w) vw[i][w] = 0u;
            }
        }
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            p[nt][y] = fmaf(sc[nt][0][y], f[nt][y & 1], ev - m[nt][y & 1]);
            if (mask && hide[nt][y]) p[nt][y] = -INFINITY;
            grow |= p[nt][y] > kKvGrow;
          }
        if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x0 = fmaf(sc[nt][0][c], f[nt][c], ev), x1 = fmaf(sc[nt][0][2 + c], f[nt][c], ev);
              if (mask && hide[nt][c]) x0 = -INFINITY;
              if (mask && hide[nt][2 + c]) x1 = -INFINITY;
              float x = fmaxf(x0, x1);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
              if (x > m[nt][c] + kKvGrow) {
                const float mn = x - kKvTop, al = ex2(m[nt][c] - mn);
                l[nt][c] *= al;
#pragma unroll
                for (int z = 0; z < MT; ++z) {
                  o[nt][z][c] *= al;
                  o[nt][z][2 + c] *= al;
                }
                m[nt][c] = mn;
              }
              p[nt][c] = x0 - m[nt][c];
              p[nt][2 + c] = x1 - m[nt][c];
            }
        }
        uint32_t bw[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int y = 0; y < 4; ++y) p[nt][y] = ex2(p[nt][y]);
#pragma unroll
          for (int c = 0; c < 2; ++c) l[nt][c] = fmaf(p[nt][c] + p[nt][2 + c], inv, l[nt][c]);
#pragma unroll
          for (int x = 0; x < 2; ++x) bw[nt][x] = movmatrix(pack_f16(p[nt][2 * x], p[nt][2 * x + 1]));
        }
        __syncwarp();
        issue(stage);  // the stage's bytes are in registers: refill it
        mt_next = load_exp(stage + 1 == ST ? 0 : stage + 1);
        // ---- O^T += V^T . W^T
#pragma unroll
        for (int w = 0; w < HD / 32; ++w)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t sel = x ? 0x7362u : 0x5140u;
            uint32_t a0, a1, a2, a3;
            codes4_to_f16<TYPE>(__byte_perm(vw[0][w], vw[1][w], sel), a0, a1);
            codes4_to_f16<TYPE>(__byte_perm(vw[2][w], vw[3][w], sel), a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][2 * w + x], a0, a1, a2, a3, bw[nt][0], bw[nt][1]);
          }
        if (++stage == ST) { stage = 0; parity ^= 1u; }
      }

      // ---- the stretch's end -------------------------------------------------------
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nt][c] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][c], d);
          if (m[nt][c] == kDecLow) m[nt][c] = 0.0f;  // l is 0, or NaN for a NaN score
        }
      if (seg_v0 == s.pair_v && v == s.pair_end) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int row = s.row0 + nt * 8 + 2 * t + c;
            if (row >= s.rows) continue;
            const int i = token_of(row), gh = row - i * a.group;
            const int64_t at = (int64_t)(s.start + i) * a.heads * a.group + s.h * a.group + gh;
            const float f = kv_inv(l[nt][c]);
            uint32_t w[MT];
#pragma unroll
            for (int z = 0; z < MT; ++z) w[z] = pack_bf16(o[nt][z][c] * f, o[nt][z][2 + c] * f);
            uint4* dst = reinterpret_cast<uint4*>(a.out + at * HD + g * MT * 2);
#pragma unroll
            for (int z = 0; z < MT / 4; ++z) dst[z] = make_uint4(w[4 * z], w[4 * z + 1], w[4 * z + 2], w[4 * z + 3]);
            if (a.lse && g == 0) a.lse[at] = kv_lse(m[nt][c], l[nt][c]);
          }
      } else {
        // a warp has at most two: its first pair's end and its last pair's
        // beginning, when all its tiles have been read
        float* slot = first ? first_part : last_part;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int qr = nt * 8 + 2 * t + c;
#pragma unroll
            for (int z = 0; z < MT / 2; ++z)
              *reinterpret_cast<float4*>(slot + qr * HD + g * MT * 2 + 4 * z) =
                  make_float4(o[nt][2 * z][c], o[nt][2 * z][2 + c], o[nt][2 * z + 1][c], o[nt][2 * z + 1][2 + c]);
            if (g == 0) {
              slot[RG * HD + qr] = m[nt][c];
              slot[RG * HD + RG + qr] = l[nt][c];
            }
          }
        if (lane == 0) {
          s_part[2 * warp + (first ? 0 : 1)] = make_int2(s.pair_v, s.pair_end);
          s_rows[2 * warp + (first ? 0 : 1)] = make_int4(s.start, s.row0, s.rows, s.h);
        }
        first = false;
      }
    }
    if (!ok && lane == 0) fault_drain();
  }
  __syncthreads();

  // ---- join the partials: a warp takes row `warp` (and 8 on) of every pair --------
  const int cta0 = cuts.at(k0), cta1 = cuts.at(min(k0 + W, E));
  constexpr int N = HD / 32;
  const int pair_of = lane < 2 * W ? s_part[lane].x : -1;
  unsigned left = __ballot_sync(0xFFFFFFFFu, pair_of >= 0);
#pragma unroll 1
  while (left) {
    const int k = __ffs(left) - 1;
    const int2 pr = s_part[k];
    const unsigned members = __ballot_sync(0xFFFFFFFFu, pair_of == pr.x);
    left &= ~members;
    const int4 rw = s_rows[k];
    const bool whole = pr.x >= cta0 && pr.y <= cta1, begun = pr.x >= cta0;
#pragma unroll 1
    for (int qr = warp; qr < RG; qr += W) {
      // lane x takes slot x's m and l; then all slots' values are loaded at once
      const float* const firsts = reinterpret_cast<const float*>(smem + W * Cfg::kRing);
      float m = -INFINITY, l = 0.0f;
      if (members >> lane & 1u) {
        const float* p = (lane & 1 ? reinterpret_cast<const float*>(smem + (lane >> 1) * Cfg::kRing)
                                   : firsts + (lane >> 1) * Cfg::kSlot) + RG * HD + qr;
        l = p[RG];
        if (l != 0.0f) m = p[0];  // 0: a share that saw no token
      }
      KvJoined<RG, HD> j;
      j.M = m;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) j.M = fmaxf(j.M, __shfl_xor_sync(0xFFFFFFFFu, j.M, d));
      if (j.M == -INFINITY) j.M = 0.0f;
      const float f = l != 0.0f ? ex2(m - j.M) : 0.0f;
      j.L = l * f;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) j.L += __shfl_xor_sync(0xFFFFFFFFu, j.L, d);
#pragma unroll
      for (int i = 0; i < N; ++i) j.acc[i] = 0.0f;
#pragma unroll
      for (int x = 0; x < 2 * W; ++x) {
        const float fx = __shfl_sync(0xFFFFFFFFu, f, x);
        const float* p = (x & 1 ? reinterpret_cast<const float*>(smem + (x >> 1) * Cfg::kRing)
                                : firsts + (x >> 1) * Cfg::kSlot) + qr * HD + lane * N;
        if (fx != 0.0f) {
#pragma unroll
          for (int i = 0; i < N; ++i) j.acc[i] = fmaf(p[i], fx, j.acc[i]);
        }
      }
      const int row = rw.y + qr;
      if (whole) {
        if (row < rw.z) {
          const int tk = token_of(row);
          kv_store<RG, HD>(a, rw.x + tk, rw.w * a.group + row - tk * a.group, j);
        }
      } else {
        float* gp = a.partials + (size_t)(blockIdx.x * 2 + (begun ? 1 : 0)) * Cfg::kSlot;
#pragma unroll
        for (int i = 0; i < N; ++i) __stcg(gp + qr * HD + lane * N + i, j.acc[i]);
        if (lane == 0) {
          __stcg(gp + RG * HD + qr, j.M);
          __stcg(gp + RG * HD + RG + qr, j.L);
        }
      }
    }
    if (!whole && tid == 0) s_cross[begun ? 1 : 0] = make_int4(pr.x, pr.y, k, 0);
  }
  __syncthreads();
  // ---- pairs that cross CTAs: the last of their CTAs to arrive joins them ----------
  if (tid < 2) {
    const int4 pr = s_cross[tid];
    int c_first = 0, c_last = -1;
    if (pr.x >= 0) {
      const int first = cuts.share_of(pr.x) / W, last = cuts.share_of(pr.y - 1) / W;
      if (ticket_acq_rel(a.tickets + first) == (unsigned)(last - first)) { c_first = first; c_last = last; }
    }
    s_joins[tid] = make_int2(c_first, c_last);
  }
  __syncthreads();
#pragma unroll 1
  for (int x = 0; x < 2; ++x) {
    const int c_first = s_joins[x].x, c_last = s_joins[x].y;
    if (c_last < 0) continue;
    const int4 pr = s_cross[x];
    const int4 rw = s_rows[pr.z];
#pragma unroll 1
    for (int qr = warp; qr < min(RG, rw.z - rw.y); qr += W) {
      const int row = rw.y + qr, tk = token_of(row);
      kv_store<RG, HD>(a, rw.x + tk, rw.w * a.group + row - tk * a.group,
                       kv_join<RG, HD>(a.partials, Cfg::kSlot, c_first, c_last, qr));
    }
    if (tid == 0) a.tickets[c_first] = 0u;
  }
}

bool make_tma_map_2d(CUtensorMap* map, CUtensorMapDataType dt, const void* ptr, uint64_t inner, uint64_t outer,
                     uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle sw);

template <int TYPE, int HD, int NT>
static cudaError_t launch_decode(const CUtensorMap& mk, const CUtensorMap& mv, const KvAttnArgs& a, int grid,
                                 cudaStream_t s) {
  constexpr int BYTES = DecCfg<HD, NT>::kSmem;
  static bool attr[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !attr[dev]) {
    e = cudaFuncSetAttribute(k_kv_decode<TYPE, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr[dev] = true;
  }
  return pdl_launch(k_kv_decode<TYPE, HD, NT>, dim3((unsigned)grid), dim3(DecCfg<HD, NT>::kWarps * 32), BYTES, s, mk, mv, a);
}

// Row tiles of 8 that share a pair's codes: two when a request brings more than 8
// rows per KV head and the pairs are enough to fill the GPU.  Measured with 2
// tokens x 8 heads x 8 grouped, 128 dims, 4000 tokens: 1, 8 and 16 requests 20.0,
// 29.9 and 44.7 us with two tiles, 14.4, 29.3 and 46.7 with one, whose second
// reading of the codes mostly hits L2.
static int dec_nt(long long rows, long long pairs) { return rows > 8 && pairs * rows > 1024 ? 2 : 1; }

static cudaError_t kv_decode_launch(int type, int head_dim, int nt, const CUtensorMap& mk, const CUtensorMap& mv,
                                    const KvAttnArgs& a, int grid, cudaStream_t s) {
#define QG_DEC(T_, H_) \
  nt == 1 ? launch_decode<T_, H_, 1>(mk, mv, a, grid, s) : launch_decode<T_, H_, 2>(mk, mv, a, grid, s)
  if (type == QGEMM_KV_E4M3) return head_dim == 64 ? QG_DEC(QGEMM_KV_E4M3, 64) : QG_DEC(QGEMM_KV_E4M3, 128);
  return head_dim == 64 ? QG_DEC(QGEMM_KV_INT8, 64) : QG_DEC(QGEMM_KV_INT8, 128);
#undef QG_DEC
}

extern const int kKvPrefillRequests;  // of a launch
size_t kv_prefill_workspace(int head_dim, int sm_count);
cudaError_t kv_prefill_launch(int type, int head_dim, const KvAttnArgs& a, int grid, cudaStream_t s);

unsigned kv_decode_fault() {
  unsigned f = 0;
  return cudaMemcpyFromSymbol(&f, g_kv_decode_fault, sizeof(f)) == cudaSuccess ? f : 0xFFFFFFFFu;
}
cudaError_t kv_decode_fault_clear() {
  const unsigned z = 0;
  return cudaMemcpyToSymbol(g_kv_decode_fault, &z, sizeof(z));
}

// Requests with more rows per KV head than this run on the tcgen05 kernel.
// Measured there and here: 8 requests x 8 heads of 128 over 4096 tokens, 48 rows
// 65 and 57 us, 64 rows 65 and 71 us; 64 requests x 8 heads of 64 over 1000 to 3000,
// 32 rows 147 and 113 us, 40 rows 148 and 158 us.
static int kv_prefill_rows(int head_dim) { return head_dim == 128 ? 48 : 32; }

// Workspace: 4 KiB of the decode kernel's tickets and, as their last word, the call's
// `ready`; then both kernels' partials.
struct KvWorkspace {
  size_t decode, prefill, total;  // byte offsets of the partials
  KvWorkspace(int head_dim, long long rows, int sm_count) {
    const size_t slot = (size_t)8 * dec_nt(rows, INT32_MAX) * (head_dim + 2) * sizeof(float);
    decode = 4096;
    prefill = decode + (size_t)sm_count * 2 * slot;
    total = prefill + (rows > kv_prefill_rows(head_dim) ? kv_prefill_workspace(head_dim, sm_count) : 0);
  }
};

static qgemm_status_t kv_attention_run(const qgemm_kv_cache_t* c, KvAttnArgs a, void* ws, int sm_count, cudaStream_t s) {
  const long long rows = (long long)a.max_new * a.group;
  const KvWorkspace w(c->head_dim, rows, sm_count);
  // K and V as rows of head_dim codes, which the decode kernel copies 16 at a time
  const uint64_t code_rows = (uint64_t)c->blocks * c->heads * c->block;
  if (code_rows > INT32_MAX)
    return fail(QGEMM_ERR_UNSUPPORTED_SHAPE, "kv_attention: blocks x heads x block of the pool exceed 2^31 - 1");
  CUtensorMap mk, mv;
  const CUtensorMapSwizzle sw = c->head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (!make_tma_map_2d(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, c->k, c->head_dim, code_rows, c->head_dim, c->head_dim, 16, sw) ||
      !make_tma_map_2d(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, c->v, c->head_dim, code_rows, c->head_dim, c->head_dim, 16, sw))
    return fail(QGEMM_ERR_CUDA, "kv_attention: cuTensorMapEncodeTiled failed");
  const int all = a.requests;
  const int32_t *starts = a.starts, *lens = a.lens, *table = a.table;
  // rows enough for max_new of every request: all bring as many, and one kernel
  // takes whatever they bring.  Otherwise the decode kernel goes first and the
  // prefill kernel's CTAs take the SMs as it leaves them.
  const int few = kv_prefill_rows(c->head_dim);
  const bool many = rows > few, even = (long long)a.requests * a.max_new <= a.tokens;
  for (int kernel = many && even ? 1 : 0; kernel <= (many ? 1 : 0); ++kernel) {
    a.rows_min = kernel && !even ? few : 0;
    a.rows_max = kernel ? INT32_MAX : few;
    a.tickets = static_cast<unsigned*>(ws);
    a.ready = many ? a.tickets + 1023 : nullptr;
    a.partials = reinterpret_cast<float*>(static_cast<char*>(ws) + (kernel ? w.prefill : w.decode));
    // beside prompt chunks the few rows are as a rule one token's
    const int nt = dec_nt(many ? a.group : rows, (long long)all * a.heads);
    // requests per launch: the prefix sums fit shared memory and the line 31 bits
    const long long per = kernel ? kv_line_most(a, 256, 7) : kv_line_most(a, 8 * nt, 4);
    if (per > INT32_MAX)
      return fail(QGEMM_ERR_UNSUPPORTED_SHAPE, "kv_attention: a request's rows x heads x tokens exceed 2^31 tiles");
    long long most = INT32_MAX / per;
    if (most > (kernel ? kKvPrefillRequests : kDecRequests)) most = kernel ? kKvPrefillRequests : kDecRequests;
    for (int r0 = 0; r0 < all; r0 += (int)most) {
      a.requests = all - r0 < most ? all - r0 : (int)most;
      a.beside = kernel && !even && r0 == 0;
      a.starts = starts + r0;
      a.lens = lens + r0;
      a.table = table + (size_t)r0 * a.width;
      const cudaError_t e = kernel ? kv_prefill_launch(c->type, c->head_dim, a, sm_count, s)
                                   : kv_decode_launch(c->type, c->head_dim, nt, mk, mv, a, sm_count, s);
      if (e != cudaSuccess) return fail(QGEMM_ERR_CUDA, "kv_attention: launch: %s", cudaGetErrorString(e));
    }
  }
  return QGEMM_OK;
}

}  // namespace qg

using namespace qg;

extern "C" {

size_t qgemm_kv_attention_workspace(const qgemm_kv_cache_t* c, int32_t q_heads, int32_t requests, int32_t tokens,
                                    int32_t max_new) {
  if (kv_cache_error(c) || q_heads < 1 || q_heads % c->heads || max_new < 1) return 0;
  DevProps dp;
  if (device_props(&dp) != QGEMM_OK) return 0;
  return KvWorkspace(c->head_dim, (long long)max_new * (q_heads / c->heads), dp.sm_count).total;
}

qgemm_status_t qgemm_kv_attention(const qgemm_kv_cache_t* c, const uint16_t* q, int64_t q_stride,
                                  int64_t q_head_stride, int32_t q_heads, int32_t requests, const int32_t* starts, const int32_t* lens, const int32_t* table,
                                  int32_t table_width, int32_t tokens, int32_t max_new, float scale, int32_t window,
                                  int32_t causal, uint16_t* out, float* lse, void* workspace, size_t ws_bytes,
                                  void* stream) {
  if (const char* e = kv_cache_error(c)) return fail(QGEMM_ERR_INVALID_ARG, "kv_attention: %s", e);
  if (q_heads < 1 || q_heads % c->heads)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_attention: q_heads must be a positive multiple of the cache's heads");
  if (requests < 0 || tokens < 0 || table_width < 0 || max_new < 0 || window < 0 || tokens >= kKvMaxTokens)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_attention: bad size");
  if (((long long)table_width * c->block) > INT32_MAX)
    return fail(QGEMM_ERR_UNSUPPORTED_SHAPE, "kv_attention: table rows of more than 2^31 - 1 tokens");
  if (!(scale == scale) || scale - scale != 0.0f)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_attention: scale must be finite");
  if (requests == 0 || tokens == 0 || max_new == 0) return QGEMM_OK;
  if (!q || !starts || !lens || (table_width && !table) || !out)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_attention: null pointer");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_attention: q and out must be 16-byte aligned");
  if (q_stride % 8 || q_head_stride % 8)
    return fail(QGEMM_ERR_INVALID_ARG, "kv_attention: q's strides must be multiples of 8");
  if (reinterpret_cast<uintptr_t>(workspace) & 15u)
    return fail(QGEMM_ERR_WORKSPACE, "kv_attention: workspace must be 16-byte aligned");
  DevProps dp;
  qgemm_status_t st = device_props(&dp);
  if (st != QGEMM_OK) return st;
  const int group = q_heads / c->heads;
  if ((long long)max_new * group > INT32_MAX - 256)
    return fail(QGEMM_ERR_UNSUPPORTED_SHAPE, "kv_attention: a request's rows x grouped heads exceed 2^31");
  const size_t need = KvWorkspace(c->head_dim, (long long)max_new * group, dp.sm_count).total;
  if (!workspace || ws_bytes < need)
    return fail(QGEMM_ERR_WORKSPACE, "kv_attention: workspace of %zu bytes needed, %zu given", need, workspace ? ws_bytes : 0);
  KvAttnArgs a;
  a.k = c->k; a.v = c->v; a.ks = c->k_scales; a.vs = c->v_scales; a.blocks = c->blocks;
  a.q = q; a.q_stride = q_stride; a.q_head_stride = q_head_stride; a.starts = starts; a.lens = lens; a.table = table; a.width = table_width;
  a.block_log2 = c->block == 16 ? 4 : c->block == 32 ? 5 : c->block == 64 ? 6 : 7;
  a.requests = requests; a.tokens = tokens; a.heads = c->heads; a.group = group;
  a.max_new = max_new < tokens ? max_new : tokens;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.window = window; a.causal = causal != 0; a.out = out; a.lse = lse;
  return kv_attention_run(c, a, workspace, dp.sm_count, as_stream(stream));
}

}  // extern "C"
