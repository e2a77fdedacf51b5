// kv_prefill.cu -- attention over the paged 8-bit cache for many query rows per
// KV head (prompt chunks), on tcgen05; no counterpart in titoatwork/qgemm-mx.
// Arithmetic: kv_attention.cuh.
//
// A pair is (request, KV head, 256 rows), the rows being the request's new
// tokens times the query heads that share the KV head, so grouped heads fill
// the tile.  The rows are two TMEM tiles A and B of 128; per 64 tokens
//   S = q . K^T    kind::f16, q and K (codes widened to f16) in shared memory
//   O += W . V     W from TMEM (over S's columns), V in shared memory as its
//                  token rows lie (N-major operand)
// Each row tile has two S buffers, so the scores of the next 64 tokens are
// there when a row's softmax gets to them: the tensor core issues, in turn for
// A and B, W.V of step i - 2 and q.K of step i.  (With one buffer of 128 tokens
// the softmax waited for its own W.V and q.K in every step: 351 us instead of
// the 2048-row chunk's time below.)
//
// Warps (20): 0-3 and 4-7 the softmax of A and B, one row per thread (TMEM
// lane = row), 64 scores in registers at a time; 8-15 widen q, K and V into the
// swizzled operand tiles, their global loads one tile ahead in registers; 16 and
// 17 issue the MMAs of A and B (a commit holds up the warp that issues it for some
// 80 cycles: two warps overlap them).  Widening costs 2 conversions per 4 codes
// once per 256 rows.  Registers go where the data waits: 128 a softmax thread, 88
// a widening one, 40 in the MMA warps' group (together no more than the launch's
// 640 x 96).  (Codes by TMA into a ring of 64-token units, the room that is left
// beside the operand tiles, 24 KB: its round trip was longer than the ring.)
//
// What bounds it: exponentials and the tensor core alike (a row and token cost one
// ex2, 16 a clock and SM, as long as its 2 x 2 x 128 multiply-adds take at 128
// dims), and above that the roles' waiting for one another.  Measured, 2048 rows of
// 32 heads over 8 KV heads of 128 dims and 8192 tokens: 296 us, 813 TFLOP/s; by clock
// stamps a tile of 128 tokens takes 4400 to 4750 cycles where its MMAs and commits alone
// take 3200, and 9500 to 16600 pass between a stretch's last scores and the next one's
// first (8900 to 11200 at 64 dims).
//
// The line of all pairs' tiles is cut into one equal share per CTA
// (kv_attention.cuh), so all CTAs finish together whatever the pair count; pairs
// that cross CTAs leave (O, m, l) partials, which a second kernel joins in CTA
// order: 32 rows a CTA.  (By the last CTA to arrive, a pair's 256 rows took that
// CTA 50 us.)
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
constexpr int kPreWarps = 20, kPreLoad = 8, kPreMma = 16;  // warps; first of each role
constexpr int kPreLoaders = 256;
extern const int kKvPrefillRequests;
const int kKvPrefillRequests = 256;  // of a launch: they are kept in shared memory

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
// An MMA warp runs its loop with all lanes and one of them issues (`one`), and
// descriptors are passed as their low words (address and leading offset; the
// high word, stride offset 1024 and the 128-byte swizzle, is the same for all):
// so they live in uniform registers.  With 64-bit descriptors in a one-lane
// branch, issuing took longer than the MMAs.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
// D(tmem) (+)= A(smem) . B(smem)
__device__ __forceinline__ void umma_ss_one(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{ .reg .pred p, q; .reg .b64 x, y; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0;\n"
      "  mov.b64 x, {%1, %6}; mov.b64 y, {%2, %6};\n"
      "  @q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p; }"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(one), "n"(kDescHigh)
      : "memory");
}
// D(tmem) (+)= A(tmem) . B(smem)
__device__ __forceinline__ void umma_ts_one(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{ .reg .pred p, q; .reg .b64 y; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0; mov.b64 y, {%2, %6};\n"
      "  @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p; }"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(one), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void commit_one(uint32_t bar, uint32_t one) {
  asm volatile(
      "{ .reg .pred q; setp.ne.b32 q, %1, 0;\n"
      "  @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar), "r"(one) : "memory");
}
// Low descriptor words.  q and K: rows of 64 k (128 bytes), 8 to an atom.  V is
// N-major: rows of 64 n, one per k, 8 k to an atom, the next 64 n 16 KiB on.
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | ((16384u >> 4) << 16); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
// Waits for the loads into v (and all before).  v is an operand so that no use of
// it can move in front of the wait.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                 "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]),
                 "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]),
                 "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
               :: "memory");
}
// (a, b) <- (a, b) f + c and (a, b) <- (a, b) + (c, d), both halves in one instruction
__device__ __forceinline__ void fma2(float& a, float& b, float f, float c) {
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%0, %1}; mov.b64 y, {%2, %2}; mov.b64 z, {%3, %3};\n"
      "  fma.rn.f32x2 x, x, y, z; mov.b64 {%0, %1}, x; }"
      : "+f"(a), "+f"(b) : "f"(f), "f"(c));
}
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {
  asm("{ .reg .b64 x, y; mov.b64 x, {%0, %1}; mov.b64 y, {%2, %3};\n"
      "  add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }"
      : "+f"(a), "+f"(b) : "f"(c), "f"(d));
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
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
__global__ void __launch_bounds__(kPreWarps * 32, 1)
k_kv_prefill(const KvAttnArgs a) {
  using Cfg = PreCfg<HD>;
  constexpr int RG = kPreRows, TL = kPreTokLog2, TILE = Cfg::kTile;
  extern __shared__ uint8_t smem_raw[];
  __shared__ KvBatch<kKvPrefillRequests> s_batch;
  __shared__ int s_scan[16];
  __shared__ __align__(1024) uint64_t s_bars[32];
  __shared__ PreMeta s_meta[4][8];   // by tile, four deep: read after the tile's stage may be refilled
  __shared__ float s_fq[2][RG];      // by stretch: score factor of each row
  __shared__ int s_seg[2];           // by stretch, for the MMA warps: tiles * 2 + B in use; 0: the end
  __shared__ uint32_t s_tmem;
  const uint32_t raw = su32(smem_raw), base = (raw + 1023u) & ~1023u;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto q_addr = [&](int x) { return base + (uint32_t)(x * TILE); };
  auto k_addr = [&](int st) { return base + (uint32_t)((2 + 2 * st) * TILE); };
  auto v_addr = [&](int st) { return base + (uint32_t)((3 + 2 * st) * TILE); };
  auto bar = [&](int i) { return su32(&s_bars[i]); };
  // barriers: K and V stages full / empty, q full / empty; per row tile x
  // and buffer h, 2 x + h: S full (and so the W.V before it done), W full, and the
  // stretch's last two W.V done
  constexpr int K_FULL = 0, K_EMPTY = 2, V_FULL = 4, V_EMPTY = 6, Q_FULL = 8, Q_EMPTY = 9, S_FULL = 10, P_FULL = 14,
                O_DONE = 18;

  if (a.beside) {  // the wait is at the end
    pdl_launch_dependents();
    kv_look(a);
  } else {
    pdl_wait();
    kv_tell(a);
    pdl_launch_dependents();
  }
  const int V = kv_line<RG, TL, 16>(a, s_batch, s_scan);
  const int E = max(1, min((int)gridDim.x, V));
  const int cta = blockIdx.x;
  if (V == 0 || cta >= E) {
    if (a.beside) pdl_wait();
    return;
  }
  const KvCuts cuts(V, E);
  const int v0 = cuts.at(cta), v1 = cuts.at(cta + 1);

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(K_FULL + i), kPreLoaders / 32); mbar_init(bar(V_FULL + i), kPreLoaders / 32);
      mbar_init(bar(K_EMPTY + i), 2); mbar_init(bar(V_EMPTY + i), 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(S_FULL + i), 1); mbar_init(bar(P_FULL + i), 4); mbar_init(bar(O_DONE + i), 1);
    }
    mbar_init(bar(Q_FULL), kPreLoaders / 32);
    mbar_init(bar(Q_EMPTY), 2);
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
  // one arrival a warp: its lanes' writes are ordered before it
  auto warp_arrive = [&](int b) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(b));
  };

  if (warp >= kPreLoad && warp < kPreMma) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ---- widening: codes -> f16 operand tiles ------------------------------------
    const int lt = tid - kPreLoad * 32;  // 0 .. 255
    constexpr int CPR = HD / 16;         // 16-code pieces per token
    constexpr int PC = 128 * CPR / kPreLoaders;  // pieces per thread of K (and of V)
    constexpr int TSTEP = kPreLoaders / CPR;     // tokens between a thread's pieces: 32, or 64
    // 8 neighbouring lanes take two tokens' 64 dims: their stores meet 8 bank groups
    const int ch = (lt & 3) | (HD == 128 ? (lt >> 1) & 4 : 0);
    const int tok0 = (HD == 128 ? (lt >> 4) << 1 : (lt >> 3) << 1) | ((lt >> 2) & 1);
    const int lg = a.block_log2;
    const uint32_t block_bytes = (uint32_t)(a.heads << lg) * HD;
    int n_tile = 0, n_seg = 0, r = kv_find(s_batch, a.requests, v0);
    for (int v = v0; v < v1 && ok;) {
      KvSeg s;
      kv_seg<RG, TL>(a, s_batch, r, v, v1, s);
      v = min(s.pair_end, v1);
      if (s.tile >= s.tile_end) continue;
      const int32_t* row_table = a.table + (size_t)s.r * a.width;
      const uint32_t head_off = (uint32_t)(s.h << lg) * HD + ch * 16;
      // What is loaded here is looked at a tile later: one look before its use, even
      // a comparison, would hold the warp up for the load's round trip.
      // lane i < 8: block of the i-th 16 tokens of tile x; -1 past the end
      auto load_id = [&](int x) {
        const long long t = (long long)x * kPreTok + lane * 16;
        int id = -1;
        if (lane < 8 && x < s.tile_end && t < s.len) id = row_table[t >> lg];
        return id;
      };
      auto in_pool = [&](int id) { return id < a.blocks ? id : -1; };
      // and its exponents
      uint32_t ek, ev;
      auto load_exp = [&](int id) {
        ek = ev = 127u;
        if (id >= 0) {
          const size_t cell = (size_t)id * a.heads + s.h;
          ek = a.ks[cell];
          ev = a.vs[cell];
        }
      };
      auto load_codes = [&](const uint8_t* src, int x, int id, uint4 (&w)[PC]) {
        const int room = s.len - x * kPreTok;  // tokens of tile x (and more)
#pragma unroll
        for (int i = 0; i < PC; ++i) {
          const int t = tok0 + i * TSTEP;
          const int b = __shfl_sync(0xFFFFFFFFu, id, t >> 4);
          w[i] = make_uint4(0, 0, 0, 0);
          if (b >= 0 && t < room)
            w[i] = ld16(reinterpret_cast<const uint4*>(src + (uint64_t)(uint32_t)b * block_bytes + head_off +
                                                        (t & ((1 << lg) - 1)) * HD));
        }
      };
      auto widen = [&](uint32_t dst, const uint4 (&w)[PC]) {
#pragma unroll
        for (int i = 0; i < PC; ++i) {
          const int row = tok0 + i * TSTEP;
          const int c = 2 * (ch & 3);
          const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          uint32_t o[8];
#pragma unroll
          for (int y = 0; y < 4; ++y) codes4_to_f16<TYPE>(u[y], o[2 * y], o[2 * y + 1]);
          const uint32_t p = dst + (uint32_t)(ch >> 2) * 16384u;
          sts16(p + sw128_off(row, c), o[0], o[1], o[2], o[3]);
          sts16(p + sw128_off(row, c + 1), o[4], o[5], o[6], o[7]);
        }
      };
      // codes and exponents are loaded one tile ahead, block ids three
      int id = load_id(s.tile), id1 = load_id(s.tile + 1), id2 = load_id(s.tile + 2);
      uint4 wk[PC], wv[PC];
      // q: 16 (8 for 64 dims) lanes a row.  All of its loads are under way while the
      // last stretch's q is still read and before that stretch's partials are
      // written, whose stores would hold them up for 3000 to 7000 cycles: a stretch's
      // start is a pause for all other warps.
      {
        constexpr int LPR = HD / 8;  // lanes per row
        constexpr int STEP = kPreLoaders / LPR, BATCHES = RG / (4 * STEP);
        const int c8 = lt % LPR, r0 = lt / LPR;
        // row0 + x over group, x < 256: exact in float
        const int i0 = s.row0 / a.group, g0 = s.row0 - i0 * a.group;
        const float inv_group = 1.0f / (float)a.group;
        const int rows = min(RG, s.rows - s.row0);
        const uint16_t* const q0 = a.q + (int64_t)(s.start + i0) * a.q_stride + (int64_t)(s.h * a.group) * a.q_head_stride + c8 * 8;
        auto load_q = [&](int batch, uint4 (&w)[4]) {
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int rr = r0 + (batch * 4 + y) * STEP;
            const int i = (int)(((float)(g0 + rr) + 0.5f) * inv_group), gh = g0 + rr - i * a.group;
            w[y] = make_uint4(0, 0, 0, 0);
            if (rr < rows) w[y] = ld16(reinterpret_cast<const uint4*>(q0 + i * a.q_stride + gh * a.q_head_stride));
          }
        };
        auto put_q = [&](int batch, const uint4 (&w)[4]) {
          uint32_t mx[4];  // the rows' maxima side by side, one chain of shuffles for all
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            mx[y] = max_u16x2(max_u16x2(w[y].x & 0x7FFF7FFFu, w[y].y & 0x7FFF7FFFu),
                              max_u16x2(w[y].z & 0x7FFF7FFFu, w[y].w & 0x7FFF7FFFu));
          }
#pragma unroll
          for (int d = 1; d < LPR; d <<= 1)
#pragma unroll
            for (int y = 0; y < 4; ++y) mx[y] = max_u16x2(mx[y], __shfl_xor_sync(0xFFFFFFFFu, mx[y], d));
          uint32_t o[4][4];
          float fq[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t u[4] = {w[y].x, w[y].y, w[y].z, w[y].w};
            const uint32_t top = max(mx[y] & 0xFFFFu, mx[y] >> 16);
            const int e = top >= 0x7F80u || top < 0x0080u ? 0 : min((int)(top >> 7) - 127, 126);
            // the sign of the scale goes into q, so that factors are never negative
            const float down = a.scale_log2 < 0.0f ? -pow2f(-e) : pow2f(-e);
#pragma unroll
            for (int z = 0; z < 4; ++z) o[y][z] = pack_f16(u2f(u[z] << 16) * down, u2f(u[z] & 0xFFFF0000u) * down);
            fq[y] = fabsf(a.scale_log2) * pow2f(e);
          }
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int rr = r0 + (batch * 4 + y) * STEP;
            sts16(q_addr(rr >> 7) + (uint32_t)(c8 >> 3) * 16384u + sw128_off(rr & 127, c8 & 7), o[y][0], o[y][1], o[y][2],
                  o[y][3]);
            if (c8 == 0) s_fq[n_seg & 1][rr] = fq[y];
          }
        };
        uint4 wq[BATCHES][4];
#pragma unroll
        for (int k = 0; k < BATCHES; ++k) load_q(k, wq[k]);
        id = in_pool(id);
        load_exp(id);
        if (n_seg > 0) ok = pre_wait(bar(Q_EMPTY), (n_seg - 1) & 1);
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < BATCHES; ++k) {
          put_q(k, wq[k]);
          if (k == BATCHES / 2 - 1) {  // into the registers of the queries that are done
            load_codes(a.k, s.tile, id, wk);
            load_codes(a.v, s.tile, id, wv);
          }
        }
        // the MMA warps' view of the stretch: tiles, and whether B has rows
        if (lt == 0) s_seg[n_seg & 1] = (s.tile_end - s.tile) * 2 + (rows > 128 ? 1 : 0);
        fence_proxy_async();
        warp_arrive(Q_FULL);
      }
#pragma unroll 1
      for (int x = s.tile; x < s.tile_end && ok; ++x, ++n_tile) {
        const int st = n_tile & 1;
        const uint32_t par = (uint32_t)(n_tile >> 1) & 1u;
        if (n_tile >= 2) ok = pre_wait(bar(K_EMPTY + st), par ^ 1u);
        if (!ok) break;
        widen(k_addr(st), wk);
        if (lt < 8) {
          const int e = (int)ev - 127;
          s_meta[n_tile & 3][lt] = PreMeta{u2f(ek << 23), (float)e, pow2f(-e), 0.0f};
        }
        fence_proxy_async();
        warp_arrive(K_FULL + st);
        id = in_pool(id1);
        id1 = id2;
        id2 = load_id(x + 3);
        load_codes(a.k, x + 1, id, wk);
        load_exp(id);
        if (n_tile >= 2) ok = pre_wait(bar(V_EMPTY + st), par ^ 1u);
        if (!ok) break;
        widen(v_addr(st), wv);
        fence_proxy_async();
        warp_arrive(V_FULL + st);
        load_codes(a.v, x + 1, id, wv);
      }
      ++n_seg;
    }
    // no stretch is left
    if (n_seg > 0 && ok) ok = pre_wait(bar(Q_EMPTY), (n_seg - 1) & 1);
    if (ok) {
      if (lt == 0) s_seg[n_seg & 1] = 0;
      warp_arrive(Q_FULL);
    }
  } else if (warp >= kPreMma) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp < kPreMma + 2) {
      constexpr uint32_t id_qk = idesc_f16(128, 64), id_pv = idesc_f16(128, HD) | (1u << 16);
      const uint32_t one = lane == 0, tm = __reduce_or_sync(0xFFFFFFFFu, tmem);  // uniform
      const uint32_t x = __reduce_or_sync(0xFFFFFFFFu, (unsigned)(warp - kPreMma));  // row tile
      auto wait = [&](uint32_t b, uint32_t parity) { return __all_sync(0xFFFFFFFFu, pre_wait(bar(b), parity)) != 0; };
      uint32_t st = 0, par = 0;   // stage and phase of the next tile's K
      uint32_t sv = 0, parv = 0;  // and of the next tile's V
      uint32_t pp = 0;            // phases of W full, one bit a buffer
#pragma unroll 1
      for (int n_seg = 0; ok; ++n_seg) {
        ok = wait(Q_FULL, n_seg & 1);
        if (!ok) break;
        const int seg = (int)__reduce_or_sync(0xFFFFFFFFu, (unsigned)*const_cast<volatile int*>(&s_seg[n_seg & 1]));
        const int steps = seg & ~1;  // two to a tile
        if (steps == 0) break;
        const bool used = x == 0 || (seg & 1);
        // step i: W.V of step i - 2, then q.K of step i into the buffer it frees
#pragma unroll 1
        for (int i = 0; i < steps + 2 && ok; ++i) {
          const uint32_t h = (uint32_t)i & 1u, b = 2 * x + h;
          if (i >= 2) {
            if (h == 0) ok = wait(V_FULL + sv, parv);
            if (used) {
              ok = ok && wait(P_FULL + b, (pp >> h) & 1u);
              pp ^= 1u << h;
              tc_fence_after();
              const uint32_t vd = desc_mn(v_addr(sv) + h * 8192u), acc = i > 2;
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_ts_one(tm + 256u + x * 128u, tm + x * 128u + h * 64u + (uint32_t)(kk * 8), vd + (uint32_t)(kk * 128),
                            id_pv, kk > 0 ? 1u : acc, one);
            }
            if (h == 1) {
              commit_one(bar(V_EMPTY + sv), one);
              sv ^= 1u;
              parv ^= sv ^ 1u;
            }
          }
          if (i < steps) {
            if (h == 0) ok = ok && wait(K_FULL + st, par);
            if (used) {
              tc_fence_after();
              const uint32_t q = desc_k(q_addr(x)), k = desc_k(k_addr(st) + h * 8192u);
#pragma unroll
              for (int kk = 0; kk < HD / 16; ++kk) {
                const uint32_t o = ((uint32_t)(kk >> 2) * 16384u + (uint32_t)(kk & 3) * 32u) >> 4;
                umma_ss_one(tm + x * 128u + h * 64u, q + o, k + o, id_qk, kk != 0, one);
              }
              commit_one(bar(S_FULL + b), one);
            }
            if (h == 1) {
              commit_one(bar(K_EMPTY + st), one);
              if (i + 1 == steps) commit_one(bar(Q_EMPTY), one);
              st ^= 1u;
              par ^= st ^ 1u;
            }
          } else if (used) {
            commit_one(bar(O_DONE + b), one);
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    // ---- softmax: one row per thread -----------------------------------------------
    const int x = warp >> 2;  // row tile
    const uint32_t quad = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t sc = s_col(x) + quad, oc = o_col(x) + quad;
    const int rr = x * 128 + (warp & 3) * 32 + lane;
    int n_tile = 0, n_seg = 0, r = kv_find(s_batch, a.requests, v0);
    uint32_t s_par = 0;  // phases of S full, one bit per buffer
    uint32_t o_par = 0;  // phase of W.V done, one a stretch
    for (int v = v0; v < v1;) {
      KvSeg s;
      kv_seg<RG, TL>(a, s_batch, r, v, v1, s);
      const int seg_v0 = v;
      v = min(s.pair_end, v1);
      const int nt = max(s.tile_end - s.tile, 0);
      const bool used = x * 128 < s.rows - s.row0;
      const int row = s.row0 + rr;
      const bool on = row < s.rows;
      float m = 0.0f, l = 0.0f;
      bool fresh = true;  // no visible token yet
      if (nt > 0 && used) {
        const int i = min(row, s.rows - 1) / a.group;
        const int lo = row_lo(a, s.len, s.n_all, i), hi = row_hi(a, s.len, s.n_all, i);
        // steps that every row of this warp sees whole need no mask
        const int wrow = s.row0 + x * 128 + (warp & 3) * 32;
        const int full_lo = row_lo(a, s.len, s.n_all, min(wrow + 31, s.rows - 1) / a.group);
        const int full_hi = row_hi(a, s.len, s.n_all, min(wrow, s.rows - 1) / a.group);
        float fq = 0.0f;
#pragma unroll 1
        for (int j = 0; j < 2 * nt && ok; ++j) {
          const int h = j & 1;
          ok = pre_wait(bar(S_FULL + 2 * x + h), (s_par >> h) & 1u);
          if (!ok) break;
          s_par ^= 1u << h;
          tc_fence_after();
          if (j == 0) fq = s_fq[n_seg & 1][rr];
          const PreMeta* meta = s_meta[(n_tile + (j >> 1)) & 3] + 4 * h;
          const int t0 = s.tile * kPreTok + j * 64;
          const uint32_t scol = sc + 64u * h;
          auto step = [&](auto masked) {
            constexpr bool MASK = decltype(masked)::value;
            float p[64];
            {
              uint32_t (&w)[2][32] = reinterpret_cast<uint32_t (&)[2][32]>(p);
              tmem_ld32(scol, w[0]);
              tmem_ld32(scol + 32u, w[1]);
              tmem_ld_wait(w[0]);
              tmem_ld_wait(w[1]);
            }
            // exponents relative to m, and their maximum
            float mxa[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float f = fq * meta[g].ks, b = meta[g].ev - m;
#pragma unroll
              for (int y = 0; y < 16; y += 2) {
                const int t = 16 * g + y;
                fma2(p[t], p[t + 1], f, b);
                if (MASK) {
                  if (t0 + t < lo || t0 + t >= hi) p[t] = -INFINITY;
                  if (t0 + t + 1 < lo || t0 + t + 1 >= hi) p[t + 1] = -INFINITY;
                }
                mxa[g] = fmaxf(mxa[g], fmaxf(p[t], p[t + 1]));
              }
            }
            const float mx = fmaxf(fmaxf(mxa[0], mxa[1]), fmaxf(mxa[2], mxa[3]));
            // m moves, by a whole number, when a weight would pass 2^15, and at a
            // row's first visible token (fresh: nothing is summed yet).  Rounded down,
            // so that the largest weight is 2^10 at least, as kv_attention.cuh says.
            const bool move = mx > kKvGrow || (fresh && mx > -INFINITY);
            if (__any_sync(0xFFFFFFFFu, move)) {
              const float by = move ? fminf(floorf(mx) - kKvTop, 1e30f) : 0.0f;
              const bool scale = move && !fresh;  // by > 0
              const float al = pow2f(scale ? -(int)fminf(by, 126.0f) : 0);
              if (move) fresh = false;
              m += by;
              l *= al;
#pragma unroll
              for (int t = 0; t < 64; t += 2) add2(p[t], p[t + 1], -by, -by);
              if (j > 0 && __any_sync(0xFFFFFFFFu, scale)) {
                // O holds the steps up to the last once its W.V is done: before the
                // next step's q.K is, or for the last step, before the end is marked
                const uint32_t b = 2 * x + (h ^ 1);
                ok = __all_sync(0xFFFFFFFFu, j + 1 < 2 * nt ? pre_wait(bar(S_FULL + b), (s_par >> (h ^ 1)) & 1u)
                                                            : pre_wait(bar(O_DONE + b), o_par));
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD / 32; ++c) {
                  uint32_t w[32];
                  tmem_ld32(oc + 32u * c, w);
                  tmem_ld_wait(w);
#pragma unroll
                  for (int y = 0; y < 32; ++y) w[y] = f2u(u2f(w[y]) * al);
                  tmem_st32(oc + 32u * c, w);
                }
              }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t w[16];
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                for (int y = 0; y < 16; y += 2) {
                  const int t = 32 * c + 16 * g + y;
                  const float e0 = ex2(p[t]), e1 = ex2(p[t + 1]);
                  add2(s0, s1, e0, e1);
                  w[8 * g + y / 2] = pack_f16(e0, e1);
                }
                l = fmaf(s0 + s1, meta[2 * c + g].inv, l);
              }
              tmem_st16(scol + 16u * c, w);
            }
          };
          if (t0 >= full_lo && t0 + 64 <= full_hi) step(std::false_type{});
          else step(std::true_type{});
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc_fence_before();
          warp_arrive(P_FULL + 2 * x + h);
        }
        if (ok) ok = pre_wait(bar(O_DONE + 2 * x + 1), o_par);
        o_par ^= 1u;
        tc_fence_after();
      }
      // after a timeout the stretches that are left still write their partials, which the
      // join kernel reads, and the barrier below is met
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
          tmem_ld_wait(w);
        } else {
#pragma unroll
          for (int y = 0; y < 32; ++y) w[y] = 0u;
        }
        if (l == 0.0f) {
#pragma unroll
          for (int y = 0; y < 32; ++y) w[y] = 0u;
        }
        if (!whole) {  // four dims of all rows after one another: a warp writes 512 bytes together
#pragma unroll
          for (int y = 0; y < 8; ++y)
            __stcg(reinterpret_cast<float4*>(slot) + (8 * c + y) * RG + rr,
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
      if (nt > 0) { n_tile += nt; ++n_seg; }
    }
  }
  if (!ok && lane == 0) fault_drain();
  if (a.beside) pdl_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == kPreMma) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Joins the pairs that cross CTAs of k_kv_prefill (E of them, cut the same way):
// CTA (c, y) takes rows 32 y .. of the pair that begins in CTA c and goes on.
template <int HD>
__global__ void __launch_bounds__(256) k_kv_prefill_join(const KvAttnArgs a, int grid) {
  constexpr int RG = kPreRows, TL = kPreTokLog2, N4 = 32 * HD / 4 / 256;  // float4 per thread
  __shared__ KvBatch<kKvPrefillRequests> s_batch;
  __shared__ int s_scan[8];
  const int tid = threadIdx.x;
  // the requests are known; only the partials come from the kernel before
  pdl_launch_dependents();
  kv_look(a);
  const int V = kv_line<RG, TL, 8>(a, s_batch, s_scan);
  const int E = max(1, min(grid, V)), c_first = blockIdx.x;
  auto clear = [&] {  // after the wait; a block of this kernel that looks later waits instead
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0)
      asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(a.ready), "r"(0u) : "memory");
  };
  if (c_first + 1 >= E) {
    pdl_wait();
    clear();
    return;
  }
  const KvCuts cuts(V, E);
  const int v = cuts.at(c_first + 1);
  KvSeg s;
  int r = kv_find(s_batch, a.requests, v);
  kv_seg<RG, TL>(a, s_batch, r, v, INT32_MAX, s);
  const int rows = s.rows - s.row0 - (int)blockIdx.y * 32;  // of this CTA's 32
  pdl_wait();
  clear();
  if (s.pair_v == v || s.pair_v < cuts.at(c_first) || rows <= 0) return;
  const int c_last = cuts.share_of(s.pair_end - 1);
  KvJoined<RG, 128> j[N4];  // 4 values each
#pragma unroll
  for (int i = 0; i < N4; ++i) {
    j[i].M = -INFINITY;
    j[i].L = 0.0f;
#pragma unroll
    for (int y = 0; y < 4; ++y) j[i].acc[y] = 0.0f;
  }
#pragma unroll 1
  for (int c = c_first; c <= c_last; ++c) {
    const float* p = a.partials + (size_t)(c == c_first ? 2 * c + 1 : 2 * c) * PreCfg<HD>::kSlot;
    float m[N4], l[N4];
    float4 o[N4];
#pragma unroll
    for (int i = 0; i < N4; ++i) {
      const int qr = blockIdx.y * 32 + (tid & 31), d4 = i * 8 + (tid >> 5);
      m[i] = __ldcg(p + RG * HD + qr);
      l[i] = __ldcg(p + RG * HD + RG + qr);
      o[i] = __ldcg(reinterpret_cast<const float4*>(p) + d4 * RG + qr);
    }
#pragma unroll
    for (int i = 0; i < N4; ++i) {
      if (l[i] == 0.0f) continue;
      const float top = fmaxf(j[i].M, m[i]), f0 = ex2(j[i].M - top), f1 = ex2(m[i] - top);
      j[i].M = top;
      j[i].L = fmaf(l[i], f1, j[i].L * f0);
      j[i].acc[0] = fmaf(o[i].x, f1, j[i].acc[0] * f0); j[i].acc[1] = fmaf(o[i].y, f1, j[i].acc[1] * f0);
      j[i].acc[2] = fmaf(o[i].z, f1, j[i].acc[2] * f0); j[i].acc[3] = fmaf(o[i].w, f1, j[i].acc[3] * f0);
    }
  }
#pragma unroll
  for (int i = 0; i < N4; ++i) {
    const int qr = tid & 31, d = 4 * (i * 8 + (tid >> 5));
    if (qr >= rows) continue;
    const int row = s.row0 + blockIdx.y * 32 + qr, tk = row / a.group;
    const int64_t at = (int64_t)(s.start + tk) * (a.heads * a.group) + s.h * a.group + row - tk * a.group;
    const float f = kv_inv(j[i].L);
    *reinterpret_cast<uint2*>(a.out + at * HD + d) =
        make_uint2(pack_bf16(j[i].acc[0] * f, j[i].acc[1] * f), pack_bf16(j[i].acc[2] * f, j[i].acc[3] * f));
    if (a.lse && d == 0) a.lse[at] = kv_lse(j[i].M, j[i].L);
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
  e = pdl_launch(k_kv_prefill<TYPE, HD>, dim3((unsigned)grid), dim3(kPreWarps * 32), BYTES, s, a);
  if (e != cudaSuccess) return e;
  return pdl_launch(k_kv_prefill_join<HD>, dim3((unsigned)grid, kPreRows / 32), dim3(256), 0, s, a, grid);
}

size_t kv_prefill_workspace(int head_dim, int sm_count) {
  return (size_t)sm_count * 2 * kPreRows * (head_dim + 2) * sizeof(float);
}

cudaError_t kv_prefill_launch(int type, int head_dim, const KvAttnArgs& a, int grid, cudaStream_t s) {
  if (type == QGEMM_KV_E4M3)
    return head_dim == 64 ? launch_prefill<QGEMM_KV_E4M3, 64>(a, grid, s)
                          : launch_prefill<QGEMM_KV_E4M3, 128>(a, grid, s);
  return head_dim == 64 ? launch_prefill<QGEMM_KV_INT8, 64>(a, grid, s)
                        : launch_prefill<QGEMM_KV_INT8, 128>(a, grid, s);
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
