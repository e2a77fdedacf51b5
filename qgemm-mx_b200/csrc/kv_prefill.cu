// kv_prefill.cu -- attention over the paged 8-bit cache for many query rows per
// KV head (prompt chunks), on tcgen05; no counterpart in titoatwork/qgemm-mx.
// Arithmetic: kv_attention.cuh.
//
// A pair is (request, KV head, 256 rows), the rows being the request's new
// tokens times the query heads that share the KV head, so grouped heads fill
// the tile.  The rows are two TMEM tiles A and B of 128; per tile of 128
// tokens
//   S = q . K^T    kind::f16, q and K (codes widened to f16) in shared memory
//   O += W . V     W from TMEM (over S's columns), V in shared memory as its
//                  token rows lie (N-major operand)
// and A's softmax runs while the tensor core works for B, and the reverse.
//
// Warps (17): 0-3 and 4-7 the softmax of A and B, one row per thread (TMEM
// lane = row); 8 issues the MMAs; 9-16 widen q, K and V into the swizzled
// operand tiles, their global loads one tile ahead in registers.  Widening
// costs 2 conversions per 4 codes once per 256 rows.
//
// What bounds it: exponentials.  A row and token cost one ex2, 16 a clock and
// SM, as long as its 2 x 2 x 128 multiply-adds take the tensor core at 128
// dims; at 64 dims the tensor core needs half of that.
//
// The line of all pairs' tiles is cut into one equal share per CTA
// (kv_attention.cuh), so 148 CTAs finish together whatever the pair count; pairs that
// cross CTAs leave (O, m, l) partials, joined in CTA order by the last CTA to
// arrive at the pair's ticket.
//
// Every mbarrier wait is bounded; on a timeout the kernel sets g_kv_fault,
// drains, frees its TMEM and returns (qgemm_umma_status reports it).
#include <type_traits>

#include "gemv_core.cuh"
#include "kv_attention.cuh"
#include "tc.cuh"

namespace qg {

__device__ unsigned g_kv_fault = 0;

constexpr int kPreRows = 256, kPreTokLog2 = 7, kPreTok = 128;
constexpr int kPreWarps = 17, kPreMma = 8, kPreLoad = 9;  // warps; first of each role
constexpr int kPreLoaders = 256;

template <int HD>
struct PreCfg {
  static constexpr int kTile = 128 * HD * 2;           // one f16 operand tile: 128 rows
  static constexpr int kQ = 2 * kTile;
  static constexpr int kSmem = kQ + 4 * kTile + 1024;  // q, two stages of K and V, alignment
  static constexpr int kSlot = kPreRows * (HD + 2);    // floats of a partial: O, m, l
};

__device__ __forceinline__ bool pre_wait(uint32_t bar, uint32_t parity) {
  return mbar_wait_flag(bar, parity, &g_kv_fault);
}
// D(tmem) (+)= A(smem) . B(smem)
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// N-major SWIZZLE_128B operand: rows of 64 n (128 bytes), one per k; 8 k to a
// 1024-byte atom (stride offset), the next 64 n `atom` bytes on (leading offset).
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t addr, uint32_t atom) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(atom >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void sts16(uint32_t p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(p), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Byte offset of 16-byte chunk c (0..7) of row r in a swizzled 128-byte-row tile.
__device__ __forceinline__ uint32_t sw128_off(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// Per group of 16 tokens: 2^ek, ev, 2^-ev.
struct PreMeta {
  float ks, ev, inv, pad;
};

template <int TYPE, int HD>
__global__ void __launch_bounds__(kPreWarps * 32, 1) k_kv_prefill(const KvAttnArgs a) {
  using Cfg = PreCfg<HD>;
  constexpr int RG = kPreRows, TL = kPreTokLog2, TILE = Cfg::kTile;
  extern __shared__ uint8_t smem_raw[];
  __shared__ KvBatch s_batch;
  __shared__ int s_scan[32];
  __shared__ __align__(1024) uint64_t s_bars[32];
  __shared__ PreMeta s_meta[4][8];   // by tile, four deep: read after the tile's stage may be refilled
  __shared__ float s_fq[2][RG];      // by stretch: score factor of each row
  __shared__ uint32_t s_tmem;
  __shared__ unsigned s_ticket;
  const uint32_t raw = su32(smem_raw), base = (raw + 1023u) & ~1023u;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto q_addr = [&](int x) { return base + (uint32_t)(x * TILE); };
  auto k_addr = [&](int st) { return base + (uint32_t)((2 + 2 * st) * TILE); };
  auto v_addr = [&](int st) { return base + (uint32_t)((3 + 2 * st) * TILE); };
  auto bar = [&](int i) { return su32(&s_bars[i]); };
  // barriers: K and V stages full / empty, q full / empty, per row tile S full, W full, O full
  constexpr int K_FULL = 0, K_EMPTY = 2, V_FULL = 4, V_EMPTY = 6, Q_FULL = 8, Q_EMPTY = 9, S_FULL = 10, P_FULL = 12,
                O_FULL = 14;

  int longest;
  const int V = kv_line<RG, TL, 16>(a, s_batch, s_scan, longest);
  const int E = max(1, min((int)gridDim.x, V));
  const int cta = blockIdx.x;
  if (V == 0 || cta >= E) return;
  const KvCuts cuts(V, E);
  const int v0 = cuts.at(cta), v1 = cuts.at(cta + 1);

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(K_FULL + i), kPreLoaders); mbar_init(bar(V_FULL + i), kPreLoaders);
      mbar_init(bar(K_EMPTY + i), 1); mbar_init(bar(V_EMPTY + i), 1);
      mbar_init(bar(S_FULL + i), 1); mbar_init(bar(P_FULL + i), 128); mbar_init(bar(O_FULL + i), 1);
    }
    mbar_init(bar(Q_FULL), kPreLoaders);
    mbar_init(bar(Q_EMPTY), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kPreMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&s_tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  auto s_col = [&](int x) { return tmem + (uint32_t)(x * 128); };
  auto o_col = [&](int x) { return tmem + 256u + (uint32_t)(x * 128); };
  bool ok = true;

  if (warp >= kPreLoad) {
    // ---- widening: codes -> f16 operand tiles ------------------------------------
    const int lt = tid - kPreLoad * 32;  // 0 .. 255
    constexpr int CPR = HD / 16;         // 16-code pieces per token
    constexpr int PC = 128 * CPR / kPreLoaders;  // pieces per thread of K (and of V)
    constexpr int TSTEP = kPreLoaders / CPR;     // tokens between a thread's pieces
    const int ch = lt % CPR, tok0 = lt / CPR;
    const int lg = a.block_log2;
    int n_tile = 0, n_seg = 0, r = kv_find(s_batch, a.requests, v0);
    for (int v = v0; v < v1 && ok;) {
      KvSeg s;
      kv_seg<RG, TL>(a, s_batch, r, v, v1, s);
      v = min(s.pair_end, v1);
      if (s.tile >= s.tile_end) continue;
      const int32_t* row_table = a.table + (size_t)s.r * a.width;
      // block ids of this thread's tokens in tile x; -1 past the end or outside the pool
      auto load_ids = [&](int x, int (&id)[PC]) {
#pragma unroll
        for (int i = 0; i < PC; ++i) {
          const long long t = (long long)x * kPreTok + tok0 + i * TSTEP;
          id[i] = x < s.tile_end && t < s.len ? row_table[t >> lg] : -1;
        }
      };
      auto load_codes = [&](const uint8_t* src, int x, const int (&id)[PC], uint4 (&w)[PC]) {
#pragma unroll
        for (int i = 0; i < PC; ++i) {
          w[i] = make_uint4(0, 0, 0, 0);
          if (id[i] >= 0 && id[i] < a.blocks) {
            const int t = x * kPreTok + tok0 + i * TSTEP;
            const size_t at = ((((size_t)id[i] * a.heads + s.h) << lg) + (t & ((1 << lg) - 1))) * HD + ch * 16;
            w[i] = __ldg(reinterpret_cast<const uint4*>(src + at));
          }
        }
      };
      auto widen = [&](uint32_t dst, const uint4 (&w)[PC]) {
#pragma unroll
        for (int i = 0; i < PC; ++i) {
          const int row = tok0 + i * TSTEP;
          // lanes of odd atoms store their halves the other way round, so that
          // 8 lanes meet 8 bank groups
          const int sw = (ch >> 2) & 1, c = 2 * (ch & 3) + sw;
          const uint32_t u[4] = {sw ? w[i].z : w[i].x, sw ? w[i].w : w[i].y, sw ? w[i].x : w[i].z, sw ? w[i].y : w[i].w};
          uint32_t o[8];
#pragma unroll
          for (int y = 0; y < 4; ++y) codes4_to_f16<TYPE>(u[y], o[2 * y], o[2 * y + 1]);
          const uint32_t p = dst + (uint32_t)(ch >> 2) * 16384u;
          sts16(p + sw128_off(row, c), o[0], o[1], o[2], o[3]);
          sts16(p + sw128_off(row, c ^ 1), o[4], o[5], o[6], o[7]);
        }
      };
      // block exponents of group lt of tile x (threads 0..7): K's | V's << 8
      auto meta_id = [&](int x) {
        const long long t = (long long)x * kPreTok + lt * 16;
        return lt < 8 && x < s.tile_end && t < s.len ? row_table[t >> lg] : -1;
      };
      auto meta_of = [&](int id) -> uint32_t {
        if (id < 0 || id >= a.blocks) return 127u | (127u << 8);
        const size_t cell = (size_t)id * a.heads + s.h;
        return (uint32_t)a.ks[cell] | ((uint32_t)a.vs[cell] << 8);
      };
      // codes and exponents are loaded one tile ahead, block ids two
      int id[PC];
      uint4 wk[PC], wv[PC];
      load_ids(s.tile, id);
      int id_m = meta_id(s.tile);
      load_codes(a.k, s.tile, id, wk);
      load_codes(a.v, s.tile, id, wv);
      uint32_t meta = meta_of(id_m);
      load_ids(s.tile + 1, id);
      id_m = meta_id(s.tile + 1);
      // q: 16 (8 for 64 dims) lanes a row
      if (n_seg > 0) ok = pre_wait(bar(Q_EMPTY), (n_seg - 1) & 1);
      if (ok) {
        constexpr int LPR = HD / 8;  // lanes per row
        constexpr int STEP = kPreLoaders / LPR;
        const int c8 = lt % LPR;
#pragma unroll 4
        for (int rr = lt / LPR; rr < RG; rr += STEP) {
          const int row = s.row0 + rr;
          uint4 w = make_uint4(0, 0, 0, 0);
          if (row < s.rows) {
            const int i = row / a.group, gh = row - i * a.group;
            w = __ldg(reinterpret_cast<const uint4*>(a.q + (int64_t)(s.start + i) * a.q_stride +
                                                     (int64_t)(s.h * a.group + gh) * a.q_head_stride + c8 * 8));
          }
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
          uint32_t mx = 0;
#pragma unroll
          for (int y = 0; y < 4; ++y) mx = max(mx, max(u[y] & 0x7FFFu, (u[y] >> 16) & 0x7FFFu));
#pragma unroll
          for (int d = 1; d < LPR; d <<= 1) mx = max(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
          const int e = mx >= 0x7F80u || mx < 0x0080u ? 0 : min((int)(mx >> 7) - 127, 126);
          // the sign of the scale goes into q, so that factors are never negative
          const float down = a.scale_log2 < 0.0f ? -pow2f(-e) : pow2f(-e);
          uint32_t o[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) o[y] = pack_f16(u2f(u[y] << 16) * down, u2f(u[y] & 0xFFFF0000u) * down);
          sts16(q_addr(rr >> 7) + (uint32_t)(c8 >> 3) * 16384u + sw128_off(rr & 127, c8 & 7), o[0], o[1], o[2], o[3]);
          if (c8 == 0) s_fq[n_seg & 1][rr] = fabsf(a.scale_log2) * pow2f(e);
        }
        fence_proxy_async();
        mbar_arrive(bar(Q_FULL));
      }
      for (int x = s.tile; x < s.tile_end && ok; ++x, ++n_tile) {
        const int st = n_tile & 1;
        const uint32_t par = (uint32_t)(n_tile >> 1) & 1u;
        if (n_tile >= 2) ok = pre_wait(bar(K_EMPTY + st), par ^ 1u);
        if (!ok) break;
        widen(k_addr(st), wk);
        if (lt < 8) {
          const int ev = (int)(meta >> 8) - 127;
          s_meta[n_tile & 3][lt] = PreMeta{u2f((meta & 0xFFu) << 23), (float)ev, pow2f(-ev), 0.0f};
        }
        fence_proxy_async();
        mbar_arrive(bar(K_FULL + st));
        load_codes(a.k, x + 1, id, wk);
        meta = meta_of(id_m);
        if (n_tile >= 2) ok = pre_wait(bar(V_EMPTY + st), par ^ 1u);
        if (!ok) break;
        widen(v_addr(st), wv);
        fence_proxy_async();
        mbar_arrive(bar(V_FULL + st));
        load_codes(a.v, x + 1, id, wv);
        load_ids(x + 2, id);
        id_m = meta_id(x + 2);
      }
      ++n_seg;
    }
  } else if (warp == kPreMma) {
    if (lane == 0) {
      constexpr uint32_t id_qk = idesc_f16(128, kPreTok), id_pv = idesc_f16(128, HD) | (1u << 16);
      int n_tile = 0, n_seg = 0, r = kv_find(s_batch, a.requests, v0);
      uint32_t p_par[2] = {0, 0};
      for (int v = v0; v < v1 && ok;) {
        KvSeg s;
        kv_seg<RG, TL>(a, s_batch, r, v, v1, s);
        v = min(s.pair_end, v1);
        const int nt = s.tile_end - s.tile;
        if (nt <= 0) continue;
        const int nx = s.rows - s.row0 > 128 ? 2 : 1;  // row tiles in use
        auto qk = [&](int x, int st) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t o = (uint32_t)(kk >> 2) * 16384u + (uint32_t)(kk & 3) * 32u;
            umma_f16_ss(s_col(x), sw128_desc(q_addr(x) + o), sw128_desc(k_addr(st) + o), id_qk, kk != 0);
          }
          umma_commit(bar(S_FULL + x));
        };
        auto pv = [&](int x, int st, bool first) {
#pragma unroll
          for (int kk = 0; kk < kPreTok / 16; ++kk)
            umma_f16_ts(o_col(x), s_col(x) + (uint32_t)(kk * 8), sw128_desc_mn(v_addr(st) + (uint32_t)kk * 2048u, 16384u),
                        id_pv, !(first && kk == 0));
        };
        ok = pre_wait(bar(Q_FULL), n_seg & 1) && pre_wait(bar(K_FULL + (n_tile & 1)), (n_tile >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        for (int x = 0; x < nx; ++x) qk(x, n_tile & 1);
        umma_commit(bar(K_EMPTY + (n_tile & 1)));
        if (nt == 1) umma_commit(bar(Q_EMPTY));
        for (int j = 0; j < nt && ok; ++j, ++n_tile) {
          const int st = n_tile & 1, nst = (n_tile + 1) & 1;
          ok = pre_wait(bar(V_FULL + st), (n_tile >> 1) & 1);
          for (int x = 0; x < nx && ok; ++x) {
            ok = pre_wait(bar(P_FULL + x), p_par[x]);
            if (!ok) break;
            p_par[x] ^= 1u;
            tc_fence_after();
            pv(x, st, j == 0);
            if (j + 1 < nt) {
              if (x == 0) {
                ok = pre_wait(bar(K_FULL + nst), ((n_tile + 1) >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
              }
              qk(x, nst);
            } else {
              umma_commit(bar(O_FULL + x));
            }
          }
          umma_commit(bar(V_EMPTY + st));
          if (j + 1 < nt) umma_commit(bar(K_EMPTY + nst));
          if (j + 2 == nt) umma_commit(bar(Q_EMPTY));
        }
        ++n_seg;
      }
    }
  } else {
    // ---- softmax: one row per thread -----------------------------------------------
    const int x = warp >> 2;  // row tile
    const uint32_t quad = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t sc = s_col(x) + quad, oc = o_col(x) + quad;
    const int rr = x * 128 + (warp & 3) * 32 + lane;
    int n_tile = 0, n_seg = 0, r = kv_find(s_batch, a.requests, v0);
    uint32_t s_par = 0, o_par = 0;
    for (int v = v0; v < v1;) {
      KvSeg s;
      kv_seg<RG, TL>(a, s_batch, r, v, v1, s);
      const int seg_v0 = v;
      v = min(s.pair_end, v1);
      const int nt = max(s.tile_end - s.tile, 0);
      const bool used = x * 128 < s.rows - s.row0;
      const int row = s.row0 + rr;
      const bool on = row < s.rows;
      float m = -INFINITY, l = 0.0f;
      if (nt > 0 && used) {
        const int i = min(row, s.rows - 1) / a.group;
        const int lo = row_lo(a, s.len, s.n_all, i), hi = row_hi(a, s.len, s.n_all, i);
        // tiles that every row of this warp sees whole need no mask
        const int wrow = s.row0 + x * 128 + (warp & 3) * 32;
        const int full_lo = row_lo(a, s.len, s.n_all, min(wrow + 31, s.rows - 1) / a.group);
        const int full_hi = row_hi(a, s.len, s.n_all, min(wrow, s.rows - 1) / a.group);
        float fq = 0.0f;
        for (int j = 0; j < nt && ok; ++j) {
          ok = pre_wait(bar(S_FULL + x), s_par);
          if (!ok) break;
          s_par ^= 1u;
          tc_fence_after();
          if (j == 0) fq = s_fq[n_seg & 1][rr];
          const PreMeta* meta = s_meta[(n_tile + j) & 3];
          const int t0 = (s.tile + j) * kPreTok;
          auto tile = [&](auto masked) {
            constexpr bool MASK = decltype(masked)::value;
            const int from = lo - t0, to = hi - t0;
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t w[32];
              tmem_ld32(sc + 32u * c, w);
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                float gm = -INFINITY;
#pragma unroll
                for (int y = 0; y < 16; ++y) {
                  const int t = 32 * c + 16 * g + y;
                  if (!MASK || (t >= from && t < to)) gm = fmaxf(gm, u2f(w[16 * g + y]));
                }
                const PreMeta mt = meta[2 * c + g];
                if (!MASK || gm != -INFINITY) mx = fmaxf(mx, fmaf(gm, fq * mt.ks, mt.ev));
              }
            }
            if (__any_sync(0xFFFFFFFFu, mx > m + kKvGrow)) {
              const float mn = mx > m + kKvGrow ? mx - kKvTop : m;
              const float al = mn == m ? 1.0f : m == -INFINITY ? 0.0f : ex2(m - mn);
              m = mn;
              l *= al;
              if (j > 0) {
#pragma unroll 1
                for (int c = 0; c < HD / 32; ++c) {
                  uint32_t w[32];
                  tmem_ld32(oc + 32u * c, w);
#pragma unroll
                  for (int y = 0; y < 32; ++y) w[y] = f2u(u2f(w[y]) * al);
                  tmem_st32(oc + 32u * c, w);
                }
              }
            }
            const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t w[32], p[16];
              tmem_ld32(sc + 32u * c, w);
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                const PreMeta mt = meta[2 * c + g];
                const float f = fq * mt.ks, b = mt.ev - mu;
                float sum = 0.0f;
#pragma unroll
                for (int y = 0; y < 16; y += 2) {
                  float e0 = ex2(fmaf(u2f(w[16 * g + y]), f, b)), e1 = ex2(fmaf(u2f(w[16 * g + y + 1]), f, b));
                  if (MASK) {
                    const int t = 32 * c + 16 * g + y;
                    if (t < from || t >= to) e0 = 0.0f;
                    if (t + 1 < from || t + 1 >= to) e1 = 0.0f;
                  }
                  sum += e0 + e1;
                  p[8 * g + y / 2] = pack_f16(e0, e1);
                }
                l = fmaf(sum, mt.inv, l);
              }
              tmem_st16(sc + 16u * c, p);
            }
          };
          if (t0 >= full_lo && t0 + kPreTok <= full_hi) tile(std::false_type{});
          else tile(std::true_type{});
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc_fence_before();
          mbar_arrive(bar(P_FULL + x));
        }
        if (ok) ok = pre_wait(bar(O_FULL + x), o_par);
        o_par ^= 1u;
        tc_fence_after();
      }
      // after a timeout the stretches that are left still go through the join, so
      // that the barrier below is met and the tickets return to zero
      if (m == -INFINITY) m = 0.0f;  // l is 0, or NaN for a NaN score
      const bool whole = seg_v0 == s.pair_v && v == s.pair_end;
      const int c_first = cuts.share_of(s.pair_v);
      float* slot = a.partials + (size_t)(cta * 2 + (cta == c_first ? 1 : 0)) * Cfg::kSlot;
      const int i = min(row, s.rows - 1) / a.group, gh = min(row, s.rows - 1) - i * a.group;
      const int64_t at = (int64_t)(s.start + i) * a.heads * a.group + s.h * a.group + gh;
      const float f = whole ? kv_inv(l) : 1.0f;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t w[32];
        if (nt > 0 && used) {
          tmem_ld32(oc + 32u * c, w);
        } else {
#pragma unroll
          for (int y = 0; y < 32; ++y) w[y] = 0u;
        }
        if (l == 0.0f) {
#pragma unroll
          for (int y = 0; y < 32; ++y) w[y] = 0u;
        }
        if (!whole) {
#pragma unroll
          for (int y = 0; y < 8; ++y)
            __stcg(reinterpret_cast<float4*>(slot + rr * HD + 32 * c) + y,
                   make_float4(u2f(w[4 * y]), u2f(w[4 * y + 1]), u2f(w[4 * y + 2]), u2f(w[4 * y + 3])));
        } else if (on) {
          uint4* dst = reinterpret_cast<uint4*>(a.out + at * HD + 32 * c);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            uint32_t b[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) b[z] = pack_bf16(u2f(w[8 * y + 2 * z]) * f, u2f(w[8 * y + 2 * z + 1]) * f);
            dst[y] = make_uint4(b[0], b[1], b[2], b[3]);
          }
        }
      }
      if (!whole) {
        __stcg(slot + RG * HD + rr, m);
        __stcg(slot + RG * HD + RG + rr, l);
      } else if (on && a.lse) {
        a.lse[at] = kv_lse(m, l);
      }
      tc_fence_before();  // O's reads are done before the next stretch's MMAs write it (through W full)
      if (!whole) {
        // the pair crosses CTAs: its last CTA to arrive joins them in order
        const int c_last = cuts.share_of(s.pair_end - 1);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (tid == 0) s_ticket = ticket_acq_rel(a.tickets + c_first);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (s_ticket == (unsigned)(c_last - c_first)) {
#pragma unroll 1
          for (int qr = warp; qr < min(RG, s.rows - s.row0); qr += 8) {
            const int jrow = s.row0 + qr, ji = jrow / a.group;
            kv_store<RG, HD>(a, s.start + ji, s.h * a.group + jrow - ji * a.group,
                             kv_join<RG, HD>(a.partials, Cfg::kSlot, c_first, c_last, qr));
          }
          if (tid == 0) a.tickets[c_first] = 0u;
        }
      }
      if (nt > 0) { n_tile += nt; ++n_seg; }
    }
  }
  if (!ok && lane == 0) fault_drain();
  tc_fence_before();
  __syncthreads();
  if (warp == kPreMma) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int TYPE, int HD>
static cudaError_t launch_prefill(const KvAttnArgs& a, int grid, cudaStream_t s) {
  constexpr int BYTES = PreCfg<HD>::kSmem;
  static bool attr[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !attr[dev]) {
    e = cudaFuncSetAttribute(k_kv_prefill<TYPE, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr[dev] = true;
  }
  k_kv_prefill<TYPE, HD><<<grid, kPreWarps * 32, BYTES, s>>>(a);
  return cudaGetLastError();
}

size_t kv_prefill_workspace(int head_dim, int sm_count) {
  return (size_t)sm_count * 2 * kPreRows * (head_dim + 2) * sizeof(float);
}

cudaError_t kv_prefill_launch(int type, int head_dim, const KvAttnArgs& a, int grid, cudaStream_t s) {
  if (type == QGEMM_KV_E4M3)
    return head_dim == 64 ? launch_prefill<QGEMM_KV_E4M3, 64>(a, grid, s) : launch_prefill<QGEMM_KV_E4M3, 128>(a, grid, s);
  return head_dim == 64 ? launch_prefill<QGEMM_KV_INT8, 64>(a, grid, s) : launch_prefill<QGEMM_KV_INT8, 128>(a, grid, s);
}

unsigned kv_prefill_fault() {
  unsigned f = 0;
  return cudaMemcpyFromSymbol(&f, g_kv_fault, sizeof(f)) == cudaSuccess ? f : 0xFFFFFFFFu;
}
cudaError_t kv_prefill_fault_clear() {
  const unsigned z = 0;
  return cudaMemcpyToSymbol(g_kv_fault, &z, sizeof(z));
}

}  // namespace qg
