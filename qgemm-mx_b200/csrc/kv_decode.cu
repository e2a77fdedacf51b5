// kv_decode.cu -- attention over the paged 8-bit cache for few query rows per
// KV head (decoding, speculative tokens); no counterpart in
// titoatwork/qgemm-mx.  Arithmetic: kv_attention.cuh.
//
// What bounds it: HBM.  Every K and V code is read once, one byte for 2 to
// 2 x rows multiply-adds, so the kernel is built around the copy: each warp
// streams its own tiles of 16 tokens through a private ring of cp.async stages
// and never meets a barrier until its work is done.
//
// Split.  A pair is (request, group of 8 NT rows, KV head); its tokens are
// tiles of 16.  All pairs' tiles form one line that is cut into equal shares,
// one per warp of the grid, wherever the cuts fall, so ragged batches and a
// single long request load the GPU alike.  A share that holds a whole pair
// writes its output; the others leave (m, l, O) partials that the CTA joins in
// shared memory, and pairs that cross CTAs are joined by the last CTA to
// arrive at a ticket, in CTA order, so results do not depend on timing.
//
// Tile arithmetic (transposed, so that 8 query rows fill an MMA's N side):
//   S^T[16 tokens x 8 rows] = K . q^T     A = K codes widened to f16
//   O^T[dims x 8 rows]     += V^T . W^T   A = V codes, pairs of tokens by prmt
// mma.sync m16n8k16 with 32-bit accumulators.  The token order inside a tile
// and the dims inside an MMA are permuted so that every shared-memory read is
// a conflict-free 128-bit (64-bit for V at 64 dims) load of bytes as they lie
// in the cache.  With 2 x 8 rows per byte the tensor work is an eighth of what
// the legacy MMA path sustains beside the copy, so tcgen05's TMEM round trips
// would buy nothing here.
#include "gemv_core.cuh"
#include "kv_attention.cuh"

namespace qg {

constexpr int kDecWarps = 8;
constexpr int kDecMinTiles = 2;        // tiles per warp below which the grid shrinks

template <int HD, int NT>
struct DecCfg {
  static constexpr int kStage = 2 * 16 * HD;             // K and V of 16 tokens
  static constexpr int kStages = HD == 128 ? (NT == 1 ? 5 : 4) : 8;
  static constexpr int kSlot = 8 * NT * (HD + 2);        // floats of a partial: O, m, l
  static constexpr int kRing = kStages * kStage;
  // ring (a warp's last partial reuses it) | first partials | block exponents
  static constexpr int kSmem = kDecWarps * (kRing + kSlot * 4 + kStages * 4);
};

// Byte of 16-byte chunk `ch` of token row `row` in a tile: chunks are permuted
// so that both the K reads (rows tau(g), chunks t) and the V reads (rows
// t-dependent, chunk by g) of 8 or 16 lanes cover all banks once.
template <int HD>
__device__ __forceinline__ int tile_off(int row, int ch) {
  if (HD == 128) return row * 128 + ((ch ^ ((((row ^ (row >> 1)) & 1) << 2) | (((row >> 2) & 1) << 1))) << 4);
  return ((row & ~1) | ((row ^ (row >> 1)) & 1)) * 64 + ((ch ^ (((row >> 2) & 1) << 1)) << 4);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
__global__ void __launch_bounds__(kDecWarps * 32, 1) k_kv_decode(const KvAttnArgs a) {
  using Cfg = DecCfg<HD, NT>;
  constexpr int RG = 8 * NT, CPR = HD / 16, KJ = HD / 64, MT = HD / 16, ST = Cfg::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ KvBatch s_batch;
  __shared__ int s_scan[kDecWarps];
  __shared__ int4 s_part[kDecWarps][2];  // the pair each partial belongs to: its range on the line, its request
  __shared__ float s_wt[2 * kDecWarps + 2][RG];  // the partials' factors, then the joined m and l
  __shared__ unsigned s_ticket;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

  const int V = kv_line<RG, 4, kDecWarps>(a, s_batch, s_scan);
  if (tid < 2 * kDecWarps) s_part[tid >> 1][tid & 1] = make_int4(-1, -1, 0, 0);
  __syncthreads();
  const int E = max(1, min((int)gridDim.x * kDecWarps, V / kDecMinTiles));  // shares
  const int k0 = blockIdx.x * kDecWarps;
  if (V == 0 || k0 >= E) return;
  auto cut = [&](int k) { return (int)((long long)k * V / E); };
  auto share_of = [&](int v) { return (int)((((long long)v + 1) * E - 1) / V); };
  const int cta0 = cut(k0), cta1 = cut(min(k0 + kDecWarps, E));

  uint8_t* ring = smem + warp * Cfg::kRing;
  const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
  float* first_part = reinterpret_cast<float*>(smem + kDecWarps * Cfg::kRing) + warp * Cfg::kSlot;
  uint32_t* meta = reinterpret_cast<uint32_t*>(smem + kDecWarps * (Cfg::kRing + Cfg::kSlot * 4)) + warp * ST;

  if (k0 + warp < E) {
    const int v0 = cut(k0 + warp), v1 = cut(k0 + warp + 1);
    // ---- producer state: runs ST tiles ahead of the arithmetic --------------
    int p_v = v0, p_r = kv_find(s_batch, a.requests, v0);
    int c_r = p_r;  // the arithmetic's place
    KvSeg ps;
    ps.tile = 0; ps.tile_end = 0; ps.pair_end = v0;
    int win = -1, win_id = 0;  // 32 block ids from `win` on, one per lane, and their exponents
    uint32_t win_meta = 0;
    const int lg = a.block_log2;
    auto issue = [&](int stage) {
      while (ps.tile >= ps.tile_end && p_v < v1) {
        kv_seg<RG, 4>(a, s_batch, p_r, p_v, v1, ps);
        p_v = min(ps.pair_end, v1);
        win = -1;
      }
      if (ps.tile < ps.tile_end) {
        const int tok = ps.tile * 16, page = tok >> lg;
        if (win < 0 || page - win >= 32) {
          win = page;
          const int p = page + lane;
          win_id = ((long long)p << lg) < ps.len ? a.table[(size_t)ps.r * a.width + p] : -1;
          if (win_id < 0 || win_id >= a.blocks) {
            win_id = -1;
            win_meta = 127u | (127u << 8);
          } else {
            const size_t cell = (size_t)win_id * a.heads + ps.h;
            win_meta = (uint32_t)a.ks[cell] | ((uint32_t)a.vs[cell] << 8);
          }
        }
        const int id = __shfl_sync(0xFFFFFFFFu, win_id, page - win);
        const uint32_t mt = __shfl_sync(0xFFFFFFFFu, win_meta, page - win);
        if (lane == 0) meta[stage] = mt;
        const size_t cell = id < 0 ? 0 : (size_t)id * a.heads + ps.h;
        const size_t off = (cell << lg) * HD + (size_t)(tok & ((1 << lg) - 1)) * HD;
        const uint8_t* k = a.k + off;
        const uint8_t* v = a.v + off;
        const uint32_t dst = ring_s + stage * Cfg::kStage;
#pragma unroll
        for (int j = 0; j < CPR / 2; ++j) {
          const int c = j * 32 + lane, row = c / CPR, ch = c % CPR;
          // tokens past the end (the rest of the last block) arrive as zeros
          const int bytes = id >= 0 && tok + row < ps.len ? 16 : 0;
          cp16(dst + tile_off<HD>(row, ch), k + c * 16, bytes);
          cp16(dst + 16 * HD + tile_off<HD>(row, ch), v + c * 16, bytes);
        }
        ++ps.tile;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < ST; ++i) issue(i);

    // ---- fixed shared-memory offsets of this lane ---------------------------
    const int tau = (g & 4) | ((g & 1) << 1) | ((g >> 1) & 1);  // token row of MMA row g (+8: tau + 8)
    uint32_t k_off[2][KJ], v_off[4];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int j = 0; j < KJ; ++j) k_off[hh][j] = tile_off<HD>(tau + 8 * hh, t + 4 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (t & 1) + 4 * (t >> 1) + (i & 1) * 2 + (i >> 1) * 8;
      v_off[i] = 16 * HD + (HD == 128 ? tile_off<HD>(row, g) : tile_off<HD>(row, g >> 1) + (g & 1) * 8);
    }

    int stage = 0;
    bool first = true;
    for (int v = v0; v < v1;) {
      KvSeg s;
      kv_seg<RG, 4>(a, s_batch, c_r, v, v1, s);
      const int seg_v0 = v;
      v = min(s.pair_end, v1);
      // ---- queries: f16 fragments and score factors --------------------------
      uint32_t qf[NT][KJ][8];
      float fac[NT][2], m[NT][2], l[NT][2];
      int lo_t[NT][2], hi_t[NT][2];
      float o[NT][MT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int row = s.row0 + nt * 8 + g;
        const bool on = row < s.rows;
        const int i = row / a.group, gh = row - i * a.group;
        const uint16_t* qp = a.q + (int64_t)(s.start + i) * a.q_stride + (int64_t)(s.h * a.group + gh) * a.q_head_stride;
        uint4 w[KJ][2];
        uint32_t mx = 0;
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            w[j][x] = on ? __ldg(reinterpret_cast<const uint4*>(qp + (t + 4 * j) * 16) + x) : make_uint4(0, 0, 0, 0);
            const uint32_t u[4] = {w[j][x].x, w[j][x].y, w[j][x].z, w[j][x].w};
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
            const uint32_t u[4] = {w[j][x].x, w[j][x].y, w[j][x].z, w[j][x].w};
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const __half2 hv = __floats2half2_rn(u2f(u[y] << 16) * down, u2f(u[y] & 0xFFFF0000u) * down);
              qf[nt][j][x * 4 + y] = *reinterpret_cast<const uint32_t*>(&hv);
            }
          }
        const float fq = a.scale_log2 * pow2f(e);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = 2 * t + c;
          fac[nt][c] = __shfl_sync(0xFFFFFFFFu, fq, col * 4);
          const int crow = s.row0 + nt * 8 + col;
          const int ci = min(crow, s.rows - 1) / a.group;
          lo_t[nt][c] = row_lo(a, s.len, s.n_all, ci);
          hi_t[nt][c] = row_hi(a, s.len, s.n_all, ci);
          m[nt][c] = -INFINITY;
          l[nt][c] = 0.0f;
        }
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) o[nt][x][y] = 0.0f;
      }
      // tiles every row of the group sees whole need no mask
      const int last_i = (min(s.row0 + RG, s.rows) - 1) / a.group;
      const int full_lo = row_lo(a, s.len, s.n_all, last_i), full_hi = row_hi(a, s.len, s.n_all, s.row0 / a.group);

      // ---- tiles ----------------------------------------------------------------
#pragma unroll 1
      for (int tile = s.tile; tile < s.tile_end; ++tile) {
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        __syncwarp();
        const uint32_t sb = ring_s + stage * Cfg::kStage;
        const uint32_t mt = meta[stage];
        float sc[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) sc[nt][x][y] = 0.0f;
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
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(sc[nt][i & 1], a0, a1, a2, a3, qf[nt][j][2 * i], qf[nt][j][2 * i + 1]);
          }
        }
        const float ksc = u2f((mt & 0xFFu) << 23);
        const int vexp = (int)((mt >> 8) & 0xFFu) - 127;
        const float ev = (float)vexp, inv = pow2f(-vexp);
        const int tok = tile * 16 + tau;
        const bool mask = tile * 16 < full_lo || tile * 16 + 16 > full_hi;
        float p[NT][4];
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int c = y & 1;
            p[nt][y] = fmaf(sc[nt][0][y] + sc[nt][1][y], fac[nt][c] * ksc, ev);
            if (mask) {
              const int at = tok + (y >> 1) * 8;
              if (at < lo_t[nt][c] || at >= hi_t[nt][c]) p[nt][y] = -INFINITY;
            }
            grow |= p[nt][y] > m[nt][c] + kKvGrow;
          }
        if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = fmaxf(p[nt][c], p[nt][2 + c]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
              const float mn = x > m[nt][c] + kKvGrow ? x - kKvTop : m[nt][c];
              const float al = m[nt][c] == -INFINITY ? 0.0f : ex2(m[nt][c] - mn);
              if (mn != m[nt][c]) {
                l[nt][c] *= al;
#pragma unroll
                for (int z = 0; z < MT; ++z) {
                  o[nt][z][c] *= al;
                  o[nt][z][2 + c] *= al;
                }
                m[nt][c] = mn;
              }
            }
        }
        uint32_t bw[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float mm = m[nt][y & 1];
            p[nt][y] = ex2(p[nt][y] - (mm == -INFINITY ? 0.0f : mm));
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) l[nt][c] = fmaf(p[nt][c] + p[nt][2 + c], inv, l[nt][c]);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const __half2 hv = __floats2half2_rn(p[nt][2 * x], p[nt][2 * x + 1]);
            bw[nt][x] = movmatrix(*reinterpret_cast<const uint32_t*>(&hv));
          }
        }
        // ---- O^T += V^T . W^T
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
        __syncwarp();
        issue(stage);  // the stage's bytes are in registers: refill it
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
        stage = stage + 1 == ST ? 0 : stage + 1;
      }

      // ---- the stretch's end -------------------------------------------------------
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nt][c] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][c], d);
          if (m[nt][c] == -INFINITY) m[nt][c] = 0.0f;  // l is 0, or NaN for a NaN score
        }
      if (seg_v0 == s.pair_v && v == s.pair_end) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int row = s.row0 + nt * 8 + 2 * t + c;
            if (row >= s.rows) continue;
            const int i = row / a.group, gh = row - i * a.group;
            const int64_t at = (int64_t)(s.start + i) * a.heads * a.group + s.h * a.group + gh;
            const float f = l[nt][c] == 0.0f ? 0.0f : 1.0f / l[nt][c];
            uint32_t w[MT];
#pragma unroll
            for (int z = 0; z < MT; ++z) w[z] = pack_bf16(o[nt][z][c] * f, o[nt][z][2 + c] * f);
            uint4* dst = reinterpret_cast<uint4*>(a.out + at * HD + g * MT * 2);
#pragma unroll
            for (int z = 0; z < MT / 4; ++z) dst[z] = make_uint4(w[4 * z], w[4 * z + 1], w[4 * z + 2], w[4 * z + 3]);
            if (a.lse && g == 0)
              a.lse[at] = kv_lse(m[nt][c], l[nt][c]);
          }
      } else {
        // a warp has at most two: its first pair's end and its last pair's beginning
        if (!first) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
        }
        float* slot = first ? first_part : reinterpret_cast<float*>(ring);
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
        if (lane == 0) s_part[warp][first ? 0 : 1] = make_int4(s.pair_v, s.pair_end, s.r, 0);
        first = false;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __syncthreads();

  // ---- join the partials -------------------------------------------------------------
  auto part_of = [&](int k) -> const float* {
    const int w = k >> 1;
    return (k & 1) ? reinterpret_cast<const float*>(smem + w * Cfg::kRing)
                   : reinterpret_cast<const float*>(smem + kDecWarps * Cfg::kRing) + w * Cfg::kSlot;
  };
#pragma unroll 1
  for (int k = 0; k < 2 * kDecWarps;) {
    const int4 pr = s_part[k >> 1][k & 1];
    if (pr.x < 0) { ++k; continue; }
    int kend = k + 1;  // partials of one pair are neighbours, with unused slots between
    for (int x = k + 1; x < 2 * kDecWarps; ++x)
      if (s_part[x >> 1][x & 1].x == pr.x) kend = x + 1;
    const bool whole = pr.x >= cta0 && pr.y <= cta1;
    const int c_first = share_of(pr.x) / kDecWarps, c_last = share_of(pr.y - 1) / kDecWarps;
    float* gp = a.partials + (size_t)(blockIdx.x * 2 + ((int)blockIdx.x == c_first ? 1 : 0)) * Cfg::kSlot;
    KvSeg s;
    int join_r = pr.z;
    kv_seg<RG, 4>(a, s_batch, join_r, pr.x, pr.y, s);
    if (tid < RG) {
      float M = -INFINITY, L = 0.0f;
      for (int x = k; x < kend; ++x) {
        const float* p = part_of(x);
        if (s_part[x >> 1][x & 1].x == pr.x && p[RG * HD + RG + tid] != 0.0f) M = fmaxf(M, p[RG * HD + tid]);
      }
      for (int x = k; x < kend; ++x) {
        const float* p = part_of(x);
        const float lx = s_part[x >> 1][x & 1].x == pr.x ? p[RG * HD + RG + tid] : 0.0f;
        const float f = lx != 0.0f ? ex2(p[RG * HD + tid] - M) : 0.0f;
        s_wt[x][tid] = f;
        L = fmaf(lx, f, L);
      }
      s_wt[2 * kDecWarps][tid] = L == 0.0f ? 0.0f : M;
      s_wt[2 * kDecWarps + 1][tid] = L;
    }
    __syncthreads();
    for (int e4 = tid; e4 < RG * HD / 4; e4 += kDecWarps * 32) {
      const int qr = e4 * 4 / HD;
      KvJoined j{make_float4(0.0f, 0.0f, 0.0f, 0.0f), s_wt[2 * kDecWarps][qr], s_wt[2 * kDecWarps + 1][qr]};
      for (int x = k; x < kend; ++x) {
        const float f = s_wt[x][qr];
        if (f == 0.0f) continue;  // unused, or a share that saw no token
        const float4 ov = *reinterpret_cast<const float4*>(part_of(x) + e4 * 4);
        j.acc.x = fmaf(ov.x, f, j.acc.x); j.acc.y = fmaf(ov.y, f, j.acc.y);
        j.acc.z = fmaf(ov.z, f, j.acc.z); j.acc.w = fmaf(ov.w, f, j.acc.w);
      }
      if (whole) {
        kv_store<HD>(a, s, e4, j);
      } else {
        __stcg(reinterpret_cast<float4*>(gp) + e4, j.acc);
        if (e4 * 4 % HD == 0) {
          __stcg(gp + RG * HD + qr, j.M);
          __stcg(gp + RG * HD + RG + qr, j.L);
        }
      }
    }
    __syncthreads();
    if (!whole) {
      // the pair crosses CTAs: the last of its CTAs to arrive joins them in order
      if (tid == 0) s_ticket = ticket_acq_rel(a.tickets + c_first);
      __syncthreads();
      if (s_ticket == (unsigned)(c_last - c_first)) {
        for (int e4 = tid; e4 < RG * HD / 4; e4 += kDecWarps * 32)
          kv_store<HD>(a, s, e4, kv_join<RG, HD, 8>(a.partials, Cfg::kSlot, c_first, c_last, e4));
        if (tid == 0) a.tickets[c_first] = 0u;
      }
      __syncthreads();
    }
    k = kend;
  }
}

template <int TYPE, int HD, int NT>
static cudaError_t launch_decode(const KvAttnArgs& a, int grid, cudaStream_t s) {
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
  k_kv_decode<TYPE, HD, NT><<<grid, kDecWarps * 32, BYTES, s>>>(a);
  return cudaGetLastError();
}

// Two row tiles of 8 when a request brings more than 8 rows per KV head.
static int dec_nt(long long rows) { return rows > 8 ? 2 : 1; }

cudaError_t kv_decode_launch(int type, int head_dim, int nt, const KvAttnArgs& a, int grid, cudaStream_t s) {
#define QG_DEC(T_, H_) nt == 1 ? launch_decode<T_, H_, 1>(a, grid, s) : launch_decode<T_, H_, 2>(a, grid, s)
  if (type == QGEMM_KV_E4M3) return head_dim == 64 ? QG_DEC(QGEMM_KV_E4M3, 64) : QG_DEC(QGEMM_KV_E4M3, 128);
  return head_dim == 64 ? QG_DEC(QGEMM_KV_INT8, 64) : QG_DEC(QGEMM_KV_INT8, 128);
#undef QG_DEC
}

size_t kv_prefill_workspace(int head_dim, int sm_count);
cudaError_t kv_prefill_launch(int type, int head_dim, const KvAttnArgs& a, int grid, cudaStream_t s);

// Requests with more rows per KV head than this run on the tcgen05 kernel.
constexpr int kKvPrefillRows = 32;

// Workspace: 4 KiB of tickets for each kernel, then their partials.
struct KvWorkspace {
  size_t decode, prefill, total;  // byte offsets of the partials
  KvWorkspace(int head_dim, long long rows, int sm_count) {
    const size_t slot = (size_t)8 * dec_nt(rows) * (head_dim + 2) * sizeof(float);
    decode = 8192;
    prefill = decode + (size_t)sm_count * 2 * slot;
    total = prefill + (rows > kKvPrefillRows ? kv_prefill_workspace(head_dim, sm_count) : 0);
  }
};

static qgemm_status_t kv_attention_run(const qgemm_kv_cache_t* c, KvAttnArgs a, void* ws, int sm_count, cudaStream_t s) {
  const long long rows = (long long)a.max_new * a.group;
  const KvWorkspace w(c->head_dim, rows, sm_count);
  const int all = a.requests;
  const int32_t *starts = a.starts, *lens = a.lens, *table = a.table;
  for (int kernel = rows > kKvPrefillRows ? 1 : 0; kernel >= 0; --kernel) {
    a.rows_min = kernel ? kKvPrefillRows : 0;
    a.rows_max = kernel ? INT32_MAX : kKvPrefillRows;
    a.tickets = reinterpret_cast<unsigned*>(static_cast<char*>(ws) + 4096 * kernel);
    a.partials = reinterpret_cast<float*>(static_cast<char*>(ws) + (kernel ? w.prefill : w.decode));
    const int nt = dec_nt(rows);
    // requests per launch: the prefix sums fit shared memory and the line 31 bits
    const long long per = kernel ? kv_line_most(a, 256, 7) : kv_line_most(a, 8 * nt, 4);
    if (per > INT32_MAX)
      return fail(QGEMM_ERR_UNSUPPORTED_SHAPE, "kv_attention: a request's rows x heads x tokens exceed 2^31 tiles");
    long long most = INT32_MAX / per;
    if (most > kKvMaxRequests) most = kKvMaxRequests;
    for (int r0 = 0; r0 < all; r0 += (int)most) {
      a.requests = all - r0 < most ? all - r0 : (int)most;
      a.starts = starts + r0;
      a.lens = lens + r0;
      a.table = table + (size_t)r0 * a.width;
      const cudaError_t e = kernel ? kv_prefill_launch(c->type, c->head_dim, a, sm_count, s)
                                   : kv_decode_launch(c->type, c->head_dim, nt, a, sm_count, s);
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
