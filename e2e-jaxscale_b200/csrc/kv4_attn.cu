// Attention over the 4-bit key/value pages (kv4.cuh), causal, with an optional
// sliding window and first tokens that stay visible.
//
// Row (b, i) of T tokens per sequence is at position p = positions[b] + i and sees
// cache row j when j <= p, (no window or j > p - window or j < sinks) and j's page is
// present; o = sum_j softmax_j(scale q . k_j) v_j, and 0 when it sees nothing.
//
// Split.  The G = nq / nkv query heads of a kv head times the T tokens are its rows;
// an item is one (sequence, kv head, tile of 16 rows), a chunk 128 cache rows.  The
// chunks of all items form one list, cut into equal ranges, one per CTA, so a long
// sequence among short ones loads every SM alike; lengths are read on the device.  A
// CTA that holds only part of an item writes (max, sum, unnormalised output) to the
// workspace, and the last CTA of each group of 16 to arrive joins the group, in part
// order: the result does not depend on who is last.
//
// Inside a CTA a chunk's codes and scales are copied into a ring of shared-memory
// stages (cp.async.bulk, 18 KB per stage at head_dim 128) and four warps take 32 of its
// 128 cache rows each, with their own running maximum and sum.  S = Q K^T and O += P V run on
// mma.sync m16n8k16 f16: a stored value (at most 6 significant bits) is exact in f16,
// q is scaled per row by a power of two into f16's range (also exact, short of values
// 2^-23 below the row's largest), P is rounded to f16, everything else is fp32.
// The MMA's k index is only a summation index, so the dimensions (for S) and the
// columns of O are dealt to lanes such that a lane reads whole 16-byte (K) and 8-byte
// (V) pieces of a row: lane t of a quad holds dimensions t D/4 .. of a K row, column c of O
// stands for dimensions c D/8 .. .  For P V, whose operand pairs two rows, the nibbles
// of two rows are interleaved before they are converted.
//
// Bound: not the bytes but the mix of conversions, multiplications and MMAs of 16 cache rows x
// 16 query rows, which share the schedulers: two mma.sync (18.8 cycles of a scheduler alone),
// four conversions (12.8) and four hmul2 (8.3) take 27 together, the loop runs at 88% of that.
// 32 sequences of up to 32768 rows, 32 heads on 2: 69 us = 2.8 TB/s of the pages, 0.43 of the
// copy rate; 64 sequences with a window of 4096: 27.5 us; one sequence of 1025 rows: 10.9 us,
// latency of a chain of place, pages, product and join.  Measured and not taken: three CTAs
// per SM of 128 registers (73 us), one of twelve warps with 16-row pieces (75), copies issued
// by a computing warp (106).
#include <math.h>

#include "kv4_attn.cuh"
#include "launch.cuh"

namespace jsx {

constexpr int kKaRows = 16;     // query rows per item
constexpr int kKaWarps = 4;     // computing warps, 32 cache rows of a chunk each
constexpr int kKaKeys = kKaChunk / kKaWarps;
constexpr int kKaPieces = kKaKeys / 16;
constexpr int kKaThreads = (kKaWarps + 1) * 32;  // and one that copies
constexpr int kKaPerSm = 2;     // CTAs per SM (three of 128 registers a thread measured slower: 73 against 70 us)
constexpr int kKaStages = 3;
constexpr int kKaFan = 16;      // parts joined at once
constexpr int kKaLevels = 3;    // 16^3 parts of an item at most

int read_clear_kv4_error(uint32_t* out) {
  const uint32_t zero = 0;
  JSX_CUDA(cudaMemcpyFromSymbol(out, g_kv4_error, sizeof(*out)));
  if (*out) JSX_CUDA(cudaMemcpyToSymbol(g_kv4_error, &zero, sizeof(zero)));
  return JSX_OK;
}

template <int D>
struct KaShape {
  static constexpr int kStage = kv4_block_bytes(kKaChunk, D);
  static constexpr int kRecord = kKaRows * D + 2 * kKaRows;  // floats: output, maxima, sums
  static constexpr int kQRow = D * 2 + 16;                   // bytes: rows' pieces in different banks
};

__device__ __forceinline__ void ka_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // the computing warps
// Four values of a row's result; `l` is the weights' sum.
__device__ __forceinline__ void ka_store(bf16* out, float4 o, float l) {
  const float f = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2(o.x * f, o.y * f), pack2(o.z * f, o.w * f));
}

template <int D>
__global__ void __launch_bounds__(kKaThreads, kKaPerSm) k_kv4_attn(const __grid_constant__ KaArgs a) {
  using S = KaShape<D>;
  constexpr int KW = D / 32;      // words of codes per lane and K row
  constexpr int NV = D / 8;       // n tiles of O = dimensions per column
  constexpr int VW = D / 64;      // words of codes per lane and V row
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ __align__(16) float join[kKaWarps * kKaRows * D];  // the warps' outputs
  __shared__ __align__(16) float join_m[kKaRows * kKaWarps], join_l[kKaRows * kKaWarps];
  __shared__ __align__(16) unsigned char qrow[2][kKaRows * S::kQRow];  // q's rows of this item and the next
  __shared__ uint4 qfrag[D / 16 * 32];                                 // q as MMA operands
  __shared__ __align__(16) uint32_t q_top[kKaRows * kKaWarps];         // rows' largest magnitudes, per quarter
  __shared__ int cum[kKaListMax + 1];
  __shared__ KaPos place[2];  // this item and the next, as the copying warp finds them
  __shared__ uint64_t full[kKaStages], empty[kKaStages], begun[2], ended[2];
  __shared__ uint32_t present[kKaStages];  // pages of the stage that were copied
  __shared__ uint32_t flags[2];            // [0] a wait gave up, [1] last to arrive
  __shared__ float* recs[kKaFan];
  volatile uint32_t* abort = flags;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int s = 0; s < kKaStages; ++s) {
      tc_mbar_init(&full[s], 1);
      tc_mbar_init(&empty[s], kKaWarps);
    }
    for (int s = 0; s < 2; ++s) {
      tc_mbar_init(&begun[s], 1);
      tc_mbar_init(&ended[s], kKaWarps);
    }
    flags[0] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  const uint32_t block = kv4_block_bytes(a.pt, D);

  if (warp == kKaWarps) {
    // ---- places, q's rows and pages: the copying warp runs ahead of the others ----
    const int pages = kKaChunk >> a.pt_log;
    uint32_t f = 0, k = 0;
    KaPos first = ka_first(a, cum, lane);
    if (lane == 0) place[0] = first;
    __syncwarp();
    for (;; ++k) {
      KaPos& p = place[k & 1];
      // q's rows: a lane each
      const int row = p.tile * kKaRows + lane, i = ka_div_g(a, row);
      const bool q_on = p.live && lane < kKaRows && row < a.G * a.T;
      const uint32_t q_rows = __popc(__ballot_sync(0xffffffffu, q_on));
      if (lane == 0) tc_expect_tx(&begun[k & 1], q_rows * D * 2);
      __syncwarp();
      if (q_on)
        ka_copy(&qrow[k & 1][lane * S::kQRow],
                a.q + ((int64_t)p.b * a.T + i) * a.q_stride + (int64_t)(p.h * a.G + row - i * a.G) * D, D * 2, &begun[k & 1]);
      if (!p.live) break;
      const int c0 = p.c0, c1 = p.c1, lo_chunk = p.x.lo_chunk, sink_chunks = p.x.sink_chunks, hi = p.x.hi;
      const int sinks = min(a.sinks, hi);
      const int32_t* table = a.table + (int64_t)p.b * a.slots;
      const int64_t head = p.h;
      auto look_up = [&](int c) {
        const int chunk = c < sink_chunks ? c : lo_chunk + c - sink_chunks;
        const int slot = chunk * pages + lane;
        return lane < pages && (slot << a.pt_log) < (c < sink_chunks ? sinks : hi) && slot < a.slots ? table[slot] : -1;
      };
      int soon = c0 < c1 ? look_up(c0) : -1;  // pages are looked up a chunk ahead
      for (int c = c0; c < c1; ++c, ++f) {
        const uint32_t s = f % kKaStages;
        const int page = soon;
        if (c + 1 < c1) soon = look_up(c + 1);
        if (f >= kKaStages && !ka_wait(&empty[s], (f / kKaStages - 1) & 1, abort))
          goto landed;
        const uint32_t have = __ballot_sync(0xffffffffu, page >= 0 && page < a.num_pages);
        if (lane == 0) {
          present[s] = have;
          tc_expect_tx(&full[s], __popc(have) * block);
        }
        __syncwarp();
        if (have >> lane & 1u)
          ka_copy(ring + s * S::kStage + lane * block, a.pool + ((int64_t)page * a.nkv + head) * block, block, &full[s]);
      }
      if (k >= 1 && !ka_wait(&ended[(k + 1) & 1], ((k + 1) / 2 - 1) & 1, abort)) goto landed;
      if (lane == 0) {
        place[(k + 1) & 1] = p;
        ka_next(a, cum, &place[(k + 1) & 1]);
      }
      __syncwarp();
    }
  landed:
    // the copies in flight land before this CTA's shared memory is given away, also when a wait gave up
    for (uint32_t x = f > kKaStages ? f - kKaStages : 0; x < f; ++x)
      tc_wait_err(&full[x % kKaStages], (x / kKaStages) & 1, nullptr, &g_kv4_error);
    for (uint32_t x = k > 0 ? k - 1 : 0; x <= k; ++x) tc_wait_err(&begun[x & 1], (x / 2) & 1, nullptr, &g_kv4_error);
    return;
  }

  // ---- the computing warps ----
  const int g = lane >> 2, t = lane & 3;
  // K's rows are dealt to a tile's columns (column 2i: row i, column 2i + 1: row 4 + (i ^ 1) of
  // eight) such that neither K's 16-byte nor V's 8-byte loads of a lane group share banks more than twice
  const int v_row1 = 4 + (t ^ 1), k_row = g & 1 ? 4 + ((g >> 1) ^ 1) : g >> 1;
  const uint32_t ring_at = s_u32(ring), q_at = s_u32(qfrag) + lane * 16;
  const uint32_t v_codes = kv4_off_v(a.pt, D), v_scales = a.pt * (D / 16);
  int piece_page[kKaPieces], piece_code[kKaPieces], piece_scale[kKaPieces];
#pragma unroll
  for (int u = 0; u < kKaPieces; ++u) {
    const int r = warp * kKaKeys + u * 16;
    piece_page[u] = r >> a.pt_log;
    piece_code[u] = piece_page[u] * block + (r & (a.pt - 1)) * (D / 2);
    piece_scale[u] = piece_page[u] * block + kv4_off_ks(a.pt, D) + (r & (a.pt - 1)) * (D / 16);
  }
  bool bad = false;
  uint32_t stage = 0, phase = 0;
  for (uint32_t item = 0;; ++item) {
      // (a wait that gave up in one warp ends the loop in all)
      if (!epi_all(ka_wait(&begun[item & 1], (item / 2) & 1, abort))) break;
      const KaPos& it = place[item & 1];
      if (!it.live) break;
      // q as MMA operands: each warp converts its quarter of the dimensions, after the rows'
      // largest magnitudes have met in shared memory
      constexpr int QW = D / 32;  // words of two values per lane and row
      float sc[2];
      int rowpos[2];
      uint32_t qv[2][QW];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = g + 8 * k, row = it.tile * kKaRows + r;
        const bool live = row < a.G * a.T;
        const uint32_t at = s_u32(&qrow[item & 1][r * S::kQRow]) + t * (D / 2) + warp * (D / 8);
        if constexpr (D == 128) {
          const uint4 v = ka_lds128(at);
          qv[k][0] = v.x, qv[k][1] = v.y, qv[k][2] = v.z, qv[k][3] = v.w;
        } else {
          const uint2 v = ka_lds64(at);
          qv[k][0] = v.x, qv[k][1] = v.y;
        }
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < QW; ++i) {
          qv[k][i] = live ? qv[k][i] : 0u;
          mx = __vmaxu2(mx, qv[k][i] & 0x7fff7fffu);
        }
        mx = max(mx & 0xffffu, mx >> 16);
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (t == 0) q_top[r * kKaWarps + warp] = mx;
        rowpos[k] = it.x.pos + (live ? ka_div_g(a, row) : 0);
      }
      ka_sync();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint4 tops = *reinterpret_cast<const uint4*>(q_top + (g + 8 * k) * kKaWarps);
        float undo;
        const float mul = ka_q_scale(max(max(tops.x, tops.y), max(tops.z, tops.w)), &undo);
        sc[k] = fmaxf(a.scale_log2 * undo, 1e-37f);  // never 0: 0 x -inf
        const float f = a.negate ? -mul : mul;
        uint32_t* q32 = reinterpret_cast<uint32_t*>(qfrag);
#pragma unroll
        for (int i = 0; i < QW; ++i)  // steps QW / 2 x warp + i / 2
          q32[((warp * (QW / 2) + i / 2) * 32 + lane) * 4 + (i & 1) * 2 + k] = ka_h2(bf_lo(qv[k][i]) * f, bf_hi(qv[k][i]) * f);
      }
      ka_sync();
      float o[NV][4];
#pragma unroll
      for (int i = 0; i < NV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[4] = {0.f, 0.f, 0.f, 0.f};  // l: sums of rows g and g + 8 in [0] and [2]
      // cache rows that every row of the tile sees
      const int all_hi = it.x.pos + it.x.t0;
      const int all_lo = a.window > 0 ? it.x.pos + it.x.t1 - a.window + 1 : 0;

      const int sink_chunks = it.x.sink_chunks, lo_chunk = it.x.lo_chunk, c_end = it.c1, window = a.window, sinks = a.sinks;
      for (int c = it.c0; c < c_end; ++c) {
        if (!bad) bad = !ka_wait(&full[stage], phase, abort);
        const int key0 = (c < sink_chunks ? c : lo_chunk + c - sink_chunks) * kKaChunk + warp * kKaKeys;
        // this warp's 16-row pieces: whether their pages are there, and where
        const uint32_t st = ring_at + stage * S::kStage;
        const uint32_t have = bad ? 0u : present[stage];
        uint32_t here = 0, piece[kKaPieces], piece_ks[kKaPieces];
#pragma unroll
        for (int u = 0; u < kKaPieces; ++u) {
          here |= (have >> piece_page[u] & 1u) << u;
          piece[u] = st + piece_code[u];
          piece_ks[u] = st + piece_scale[u];
        }
        if (here) {
          const bool masked = here != (1u << kKaPieces) - 1u || key0 + kKaKeys - 1 > all_hi ||
                              (key0 < all_lo && key0 + kKaKeys > sinks);
          auto see = [&](int e, int p) {  // cache row key0 + e from position p
            const int key = key0 + e;
            return key <= p && (window == 0 || key > p - window || key < sinks) && (here >> (e / 16) & 1u);
          };
          // ---- S = Q K^T ----
          float sa[kKaKeys / 8][4];
          uint32_t kw[kKaKeys / 8][KW], kf[kKaKeys / 8];
#pragma unroll
          for (int j = 0; j < kKaKeys / 8; ++j) {
            const uint32_t kc = piece[j / 2] + (j % 2 * 8) * (D / 2) + k_row * (D / 2) + t * (D / 8);
            const uint32_t ks = piece_ks[j / 2] + (j % 2 * 8) * (D / 16) + k_row * (D / 16) + t * (D / 64);
            if constexpr (D == 128) {
              const uint4 v = ka_lds128(kc);
              kw[j][0] = v.x;
              kw[j][1] = v.y;
              kw[j][2] = v.z;
              kw[j][3] = v.w;
              kf[j] = e4m3x2_to_h2(ka_lds16(ks));
            } else {
              const uint2 v = ka_lds64(kc);
              kw[j][0] = v.x;
              kw[j][1] = v.y;
              const uint32_t x = ka_lds8(ks);
              kf[j] = e4m3x2_to_h2(x | (x << 8));
            }
            sa[j][0] = sa[j][1] = sa[j][2] = sa[j][3] = 0.f;
          }
#pragma unroll
          for (int k = 0; k < KW; ++k) {
            const uint4 q0 = ka_lds128(q_at + 2 * k * 512), q1 = ka_lds128(q_at + (2 * k + 1) * 512);
            const uint32_t qa0[4] = {q0.x, q0.y, q0.z, q0.w}, qa1[4] = {q1.x, q1.y, q1.z, q1.w};
#pragma unroll
            for (int j = 0; j < kKaKeys / 8; ++j) {
              uint32_t h[4];
              e2m1x8_to_h2(kw[j][k], h);
              const uint32_t f = D == 128 ? __byte_perm(kf[j], 0, k < KW / 2 ? 0x1010 : 0x3232) : kf[j];
              ka_mma(sa[j], qa0, hmul2_u(h[0], f), hmul2_u(h[1], f));
              ka_mma(sa[j], qa1, hmul2_u(h[2], f), hmul2_u(h[3], f));
            }
          }
          if (masked) {
#pragma unroll
            for (int j = 0; j < kKaKeys / 8; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!see(j * 8 + (e & 1 ? v_row1 : t), rowpos[e >> 1])) sa[j][e] = -INFINITY;
          }
          // ---- running reference, weights ----
          bool move = false;
          float top[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            top[k] = fmaxf(sa[0][2 * k], sa[0][2 * k + 1]);
#pragma unroll
            for (int j = 1; j < kKaKeys / 8; ++j) top[k] = fmaxf(top[k], fmaxf(sa[j][2 * k], sa[j][2 * k + 1]));
            top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
            top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 2)) * sc[k];
            move |= top[k] > m[k] + kKaLazy;
          }
          if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float to = top[k] > m[k] + kKaLazy ? top[k] : m[k];
              const float f = m[k] == -INFINITY ? 0.f : ka_exp2(m[k] - to);
              m[k] = to;
              l[2 * k] *= f;
#pragma unroll
              for (int i = 0; i < NV; ++i) {
                o[i][2 * k] *= f;
                o[i][2 * k + 1] *= f;
              }
            }
          }
          const float ref[2] = {m[0] == -INFINITY ? 0.f : kKaOff - m[0], m[1] == -INFINITY ? 0.f : kKaOff - m[1]};
          uint32_t pa[kKaPieces][4];
#pragma unroll
          for (int j = 0; j < kKaKeys / 8; ++j) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] = ka_exp2(__fmaf_rn(sa[j][e], sc[e >> 1], ref[e >> 1]));
            pa[j / 2][j % 2 * 2] = ka_h2(p[0], p[1]);
            pa[j / 2][j % 2 * 2 + 1] = ka_h2(p[2], p[3]);
          }
          // ---- O += P V, and the weights' sum as one more column of ones ----
#pragma unroll
          for (int u = 0; u < kKaPieces; ++u) {
            // this lane's rows 2t, 2t + 1 of both 8-row halves, column g
            const uint32_t vc = piece[u] + v_codes, vs = piece_ks[u] + v_scales;
            // this lane's two rows of both 8-row halves, column g
            uint32_t sv[4], w[4][VW];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = (k >> 1) * 8 + (k & 1 ? v_row1 : t);
              sv[k] = ka_lds8(vs + r * (D / 16) + g * NV / 16);
              if constexpr (D == 128) {
                const uint2 v = ka_lds64(vc + r * (D / 2) + g * (NV / 2));
                w[k][0] = v.x;
                w[k][1] = v.y;
              } else {
                w[k][0] = ka_lds32(vc + r * (D / 2) + g * (NV / 2));
              }
            }
            if (masked) {
              // a weight of 0 does not silence a NaN: rows that some of the tile must not see
              // enter without their NaN scales, which are put into the rows that do see them
              bool odd = false;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                odd |= ka_nan_scale(sv[k]);
                if (ka_nan_scale(sv[k])) sv[k] = 0;
              }
              if (__any_sync(0xffffffffu, odd)) {
                for (int e = 0; e < 16; ++e)
#pragma unroll
                  for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int col = 0; col < 2; ++col)
                      if (see(u * 16 + e, rowpos[k]) && ka_nan_scale(ka_lds8(vs + e * (D / 16) + (2 * t + col) * NV / 16)))
#pragma unroll
                        for (int i = 0; i < NV; ++i) o[i][2 * k + col] = NAN;
              }
            }
            const uint32_t f0 = e4m3x2_to_h2(sv[0] | (sv[1] << 8)), f1 = e4m3x2_to_h2(sv[2] | (sv[3] << 8));
            ka_mma(l, pa[u], 0x3c003c00u, 0x3c003c00u);
#pragma unroll
            for (int x = 0; x < VW; ++x) {
              uint32_t h0[4], h1[4];  // even dimensions of the word, then odd ones
              e2m1x8_to_h2((w[0][x] & 0x0f0f0f0fu) | ((w[1][x] << 4) & 0xf0f0f0f0u), h0);
              e2m1x8_to_h2((w[2][x] & 0x0f0f0f0fu) | ((w[3][x] << 4) & 0xf0f0f0f0u), h1);
#pragma unroll
              for (int k = 0; k < 4; ++k) ka_mma(o[8 * x + 2 * k], pa[u], hmul2_u(h0[k], f0), hmul2_u(h1[k], f1));
              e2m1x8_to_h2(((w[0][x] >> 4) & 0x0f0f0f0fu) | (w[1][x] & 0xf0f0f0f0u), h0);
              e2m1x8_to_h2(((w[2][x] >> 4) & 0x0f0f0f0fu) | (w[3][x] & 0xf0f0f0f0u), h1);
#pragma unroll
              for (int k = 0; k < 4; ++k) ka_mma(o[8 * x + 2 * k + 1], pa[u], hmul2_u(h0[k], f0), hmul2_u(h1[k], f1));
            }
          }
        }
        __syncwarp();
        if (lane == 0) tc_arrive(&empty[stage]);
        if (++stage == kKaStages) {
          stage = 0;
          phase ^= 1u;
        }
      }

      // ---- join the four warps ----
      // a column's 16-byte pieces are dealt such that a quarter-warp's accesses meet all banks
      auto at = [&](int w, int r, int column, int piece) {
        return reinterpret_cast<float4*>(join + (w * kKaRows + r) * D + (column ^ (r & 1)) * NV +
                                         4 * (piece ^ (D == 128 ? column >> 1 : column >> 2)));
      };
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = g + 8 * k;
        if (t == 0) {
          join_m[r * kKaWarps + warp] = m[k];
          join_l[r * kKaWarps + warp] = l[2 * k];
        }
#pragma unroll
        for (int col = 0; col < 2; ++col)
#pragma unroll
          for (int q0 = 0; q0 < NV / 4; ++q0)
            *at(warp, r, 2 * t + col, q0) = make_float4(o[4 * q0][2 * k + col], o[4 * q0 + 1][2 * k + col],
                                                        o[4 * q0 + 2][2 * k + col], o[4 * q0 + 3][2 * k + col]);
      }
      ka_sync();
      // parts of this item: CTAs first .. first + parts - 1
      const bool whole = it.c1 - it.c0 == it.x.n;
      const int u0 = it.w - it.c0, used = it.x.used;
      int first = 0, parts = 1;
      if (!whole) {
        first = ka_owner(it, u0);
        parts = ka_owner(it, u0 + it.x.n - 1) - first + 1;
      }
      // a CTA's range holds one item's end and another's beginning at most: two records per CTA
      auto slot_of = [&](int p) { return 2 * (first + p) + (ka_range(it, first + p) < u0 ? 1 : 0); };
      auto finish = [&](int r, int d, float4 v, float sum) {
        const int row = it.tile * kKaRows + r, i = ka_div_g(a, row);
        if (row >= a.G * a.T) return;
        const bool on = i < used;
        ka_store(a.out + ((int64_t)it.b * a.T + i) * a.out_stride + (int64_t)(it.h * a.G + row - i * a.G) * D + d,
                 on ? v : make_float4(0.f, 0.f, 0.f, 0.f), on ? sum : 0.f);
      };
      const int my_part = blockIdx.x - first;
      float* rec = whole ? nullptr : a.parts + (size_t)slot_of(my_part) * S::kRecord;
#pragma unroll
      for (int k = 0; k < kKaRows * D / 4 / (kKaWarps * 32); ++k) {
        const int e = tid + k * kKaWarps * 32, r = e / (D / 4), d = e % (D / 4) * 4;
        const float4 mw = *reinterpret_cast<const float4*>(join_m + r * kKaWarps);
        const float4 lw = *reinterpret_cast<const float4*>(join_l + r * kKaWarps);
        const float top = fmaxf(fmaxf(mw.x, mw.y), fmaxf(mw.z, mw.w));
        const float ms[4] = {mw.x, mw.y, mw.z, mw.w}, ls[4] = {lw.x, lw.y, lw.z, lw.w};
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kKaWarps; ++w) {
          const float f = ms[w] == -INFINITY ? 0.f : ka_exp2(ms[w] - top);
          const float4 x = *at(w, r, d / NV, d % NV / 4);
          sum += ls[w] * f;
          v = make_float4(v.x + x.x * f, v.y + x.y * f, v.z + x.z * f, v.w + x.w * f);
        }
        if (whole) {
          finish(r, d, v, sum);
        } else {
          *reinterpret_cast<float4*>(rec + r * D + d) = v;
          if (d == 0) {
            rec[kKaRows * D + r] = top;
            rec[kKaRows * D + kKaRows + r] = sum;
          }
        }
      }
      // ---- join the CTAs ----
      int idx = my_part, count = parts, span = 1;
#pragma unroll 1
      for (int level = 0; count > 1; ++level) {
        const int lead = idx / kKaFan * kKaFan;
        const int members = min(kKaFan, count - lead);
        const bool final = count <= kKaFan;
        if (members > 1) {
          ka_sync();
          if (tid == 0) {
            // the barrier orders every thread's stores before this release, and the others' loads after
            // this acquire by the next one
            uint32_t* ctr = a.arrived + level * 2 * gridDim.x + slot_of(lead * span);
            uint32_t before;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(ctr) : "memory");
            const bool last = before == (uint32_t)members - 1;
            if (last) *ctr = 0;
            flags[1] = last;
          }
          if (tid >= 32 && tid < 32 + kKaFan)  // (the last record again where there are fewer)
            recs[tid - 32] = a.parts + (size_t)slot_of((lead + min(tid - 32, members - 1)) * span) * S::kRecord;
          ka_sync();
          if (!flags[1]) break;
          // this thread's 16-byte pieces, four parts of each at a time: 16 loads in flight
          constexpr int kMine = kKaRows * D / 4 / (kKaWarps * 32);
          float4 v[kMine][4];
          auto load = [&](int q0) {
#pragma unroll
            for (int k = 0; k < kMine; ++k)
#pragma unroll
              for (int p = 0; p < 4; ++p)
                v[k][p] = __ldcg(reinterpret_cast<const float4*>(recs[q0 + p]) + tid + k * kKaWarps * 32);
          };
          load(0);
          // thread (part group, row): maxima and sums of two parts
          float* wgt = join;                    // [16 parts][16 rows]
          float* sums = join + kKaFan * kKaRows;
          const int r0 = tid % kKaRows, p0 = tid / kKaRows;  // parts p0 and p0 + 8
          float mp[2], lp[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            mp[k] = __ldcg(recs[p0 + 8 * k] + kKaRows * D + r0);
            lp[k] = __ldcg(recs[p0 + 8 * k] + kKaRows * D + kKaRows + r0);
            if (p0 + 8 * k >= members) mp[k] = -INFINITY;
            wgt[(p0 + 8 * k) * kKaRows + r0] = mp[k];
          }
          ka_sync();
          float top = -INFINITY;
#pragma unroll
          for (int p = 0; p < kKaFan; ++p) top = fmaxf(top, wgt[p * kKaRows + r0]);
          ka_sync();
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float f = mp[k] == -INFINITY ? 0.f : ka_exp2(mp[k] - top);
            wgt[(p0 + 8 * k) * kKaRows + r0] = f;
            sums[(p0 + 8 * k) * kKaRows + r0] = p0 + 8 * k < members ? lp[k] * f : 0.f;
          }
          ka_sync();
          if (tid < kKaRows) {
            float sum = 0.f;
#pragma unroll
            for (int p = 0; p < kKaFan; ++p) sum += sums[p * kKaRows + tid];
            join_m[tid] = top;
            join_l[tid] = sum;
          }
          ka_sync();
          float* dst = recs[0];
          float4 acc[kMine];
#pragma unroll
          for (int k = 0; k < kMine; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
          for (int q0 = 0; q0 < members; q0 += 4) {
            if (q0) load(q0);
#pragma unroll
            for (int p = 0; p < 4; ++p)
              if (q0 + p < members)
#pragma unroll
                for (int k = 0; k < kMine; ++k) {
                  const float f = wgt[(q0 + p) * kKaRows + (tid + k * kKaWarps * 32) / (D / 4)];
                  acc[k] = make_float4(acc[k].x + v[k][p].x * f, acc[k].y + v[k][p].y * f, acc[k].z + v[k][p].z * f,
                                       acc[k].w + v[k][p].w * f);
                }
          }
#pragma unroll
          for (int k = 0; k < kMine; ++k) {
            const int e = tid + k * kKaWarps * 32, r = e / (D / 4), d = e % (D / 4) * 4;
            if (final) {
              finish(r, d, acc[k], join_l[r]);
            } else {
              *reinterpret_cast<float4*>(dst + r * D + d) = acc[k];
              if (d == 0) {
                dst[kKaRows * D + r] = join_m[r];
                dst[kKaRows * D + kKaRows + r] = join_l[r];
              }
            }
          }
          ka_sync();
        }
        idx /= kKaFan;
        count = (count + kKaFan - 1) / kKaFan;
        span *= kKaFan;
      }
      ka_sync();  // (the joining buffers are free, the place is read)
      if (lane == 0) tc_arrive(&ended[item & 1]);
  }

  // rows of items without a chunk
  if (a.listed) {
    const int items = a.B * a.nkv * a.tiles;
    for (int k = blockIdx.x; k < items; k += gridDim.x) {
      const int tile = k % a.tiles, h = k / a.tiles % a.nkv, b = k / a.tiles / a.nkv;
      if (ka_tile(a, b, tile).n) continue;
      for (int e = tid; e < kKaRows * D / 4; e += kKaWarps * 32) {
        const int row = tile * kKaRows + e / (D / 4), i = row / a.G;
        if (row < a.G * a.T)
          *reinterpret_cast<uint2*>(a.out + ((int64_t)b * a.T + i) * a.out_stride + (h * a.G + row - i * a.G) * D +
                                    e % (D / 4) * 4) = make_uint2(0u, 0u);
      }
    }
  }
}

// kv4_attn_wide.cu: items of 128 query rows
size_t kv4_wide_workspace(int B, int T, int nq, int nkv);
int kv4_wide_launch(KaArgs a, void* workspace, cudaStream_t s);

// Chunks per item of the rows that a call can see, by the table and the window (the lengths
// are on the device).
static int64_t ka_chunks(int64_t table_rows, int T, int window, int sinks) {
  const int64_t seen = window > 0 ? (int64_t)window + T + sinks + 2 * kKaChunk : table_rows;
  return ((seen < table_rows ? seen : table_rows) + kKaChunk - 1) / kKaChunk;
}
// Which kernel: fitted to both, the 16-row one takes 10 us + 3.5 ns and the 128-row one
// 20 us + 10.7 ns per chunk of an item, so the latter begins to pay where it saves the 16-row
// kernel 2048 chunks beyond three times its own.  Where each sequence has a count of tokens
// of its own, half of T are taken to be used.  head_dim 128, 16-row / 128-row kernel, us:
//   32 heads on 2, 16 sequences of up to 8192 rows: T 2: 27 / 40, 4: 40 / 41, 5: 48 / 41,
//     8: 70 / 45, 16: 130 / 64, 64: 490 / 198;  5 with counts of 0 to 5: 36 / 42
//   8 heads on 1, 64 sequences of up to 4000 rows: T 5: 36 / 39, 9: 51 / 42, 16: 76 / 47
//   32 heads on 2, one sequence of 4000 rows: T 8: 17 / 23, 33: 29 / 34, 64: 44 / 34
// Up to 48 query rows per kv head it never does.  The lengths are on the device, so the chunks are
// those of the table's capacity (or the window): short sequences in a long table may get the
// 128-row kernel and its 20 us.  head_dim 64 has the 16-row kernel alone (64 tokens of 16 sequences
// of up to 8191 rows: 328 us; a prompt of 8192 tokens with a window of 4096: 1576 us).
static bool ka_wide_ever(int T, int nq, int nkv, int head_dim) { return head_dim == 128 && (int64_t)(nq / nkv) * T > 3 * kKaRows; }
static bool ka_wide(int B, int T, int nq, int nkv, int head_dim, bool counts, int64_t chunks) {
  if (!ka_wide_ever(T, nq, nkv, head_dim)) return false;
  const int64_t rows = (int64_t)(nq / nkv) * (counts ? (T + 1) / 2 : T), lists = (int64_t)B * nkv * chunks;
  return lists * ((rows + kKaRows - 1) / kKaRows) - 3 * lists * ((rows + 127) / 128) >= 2048;
}

// CTAs of a launch: kKaPerSm per SM, or as many as there are chunks (items) at most.
static int ka_grid_max() { return kKaPerSm * sm_count(); }
static size_t ka_arrived_bytes() { return ((size_t)kKaLevels * 2 * ka_grid_max() * 4 + 255) / 256 * 256; }
static size_t ka_record_bytes(int D) { return (size_t)(kKaRows * D + 2 * kKaRows) * 4; }

template <int D>
static int ka_launch(const KaArgs& a, int grid, cudaStream_t s) {
  static bool done[128] = {};
  int dev = 0;
  JSX_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 128 || !done[dev]) {
    JSX_CUDA(cudaFuncSetAttribute(k_kv4_attn<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)KaShape<D>::kStage * kKaStages));
    if (dev >= 0 && dev < 128) done[dev] = true;
  }
  JSX_CUDA(launch_kernel(k_kv4_attn<D>, dim3(grid), dim3(kKaThreads), KaShape<D>::kStage * kKaStages, s, a));
  return JSX_OK;
}

}  // namespace jsx

using namespace jsx;

extern "C" int jsx_kv4_attn_workspace_size(int B, int T, int nq, int nkv, int head_dim, size_t* bytes) {
  JSX_REQUIRE(bytes && B >= 1 && T >= 1 && nq >= 1 && nkv >= 1 && nq % nkv == 0 && (head_dim == 64 || head_dim == 128),
              "bad arguments");
  const size_t records = 2 * (size_t)ka_grid_max() * ka_record_bytes(head_dim);
  const size_t wide = ka_wide_ever(T, nq, nkv, head_dim) ? kv4_wide_workspace(B, T, nq, nkv) : 0;
  *bytes = ka_arrived_bytes() + (wide > records ? wide : records);
  return JSX_OK;
}

extern "C" int jsx_kv4_attn(const void* q, int64_t q_stride, const void* pool, int num_pages, const int32_t* table,
                            int table_slots, const int32_t* positions, const int32_t* n_tokens, void* out,
                            int64_t out_stride, int B, int T, int nq, int nkv, int head_dim, int page_tokens,
                            int window, int sinks, float scale, void* workspace, size_t workspace_bytes,
                            void* stream) {
  JSX_REQUIRE(q && out && positions, "null pointer argument");
  JSX_KV4_REQUIRE(pool, num_pages, table, table_slots, nkv, head_dim, page_tokens);
  JSX_REQUIRE(nq >= 1 && nq % nkv == 0, "nq=%d is not a multiple of nkv=%d", nq, nkv);
  JSX_REQUIRE(B >= 1 && T >= 1 && (int64_t)B * T * nq <= (1 << 30), "B=%d T=%d", B, T);
  JSX_REQUIRE((int64_t)table_slots * page_tokens <= (1 << 30), "a table of %d pages of %d tokens", table_slots, page_tokens);
  JSX_REQUIRE(aligned16(q) && aligned16(out) && q_stride % 8 == 0 && out_stride % 8 == 0 &&
                  q_stride >= (int64_t)nq * head_dim && out_stride >= (int64_t)nq * head_dim,
              "q and out must be 16-byte aligned, with token strides of at least nq * head_dim in multiples of 8");
  JSX_REQUIRE(window >= 0 && sinks >= 0, "window=%d sinks=%d", window, sinks);
  JSX_REQUIRE(fabsf(scale) <= 1e30f, "scale %g", (double)scale);
  size_t need = 0;
  const int st = jsx_kv4_attn_workspace_size(B, T, nq, nkv, head_dim, &need);
  if (st) return st;
  JSX_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, "workspace of %zu bytes, %zu needed",
              workspace_bytes, need);
  KaArgs a;
  a.q = (const bf16*)q;
  a.out = (bf16*)out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.pool = (const uint8_t*)pool;
  a.table = table;
  a.positions = positions;
  a.n_tokens = n_tokens;
  a.arrived = (uint32_t*)workspace;
  a.parts = (float*)((char*)workspace + ka_arrived_bytes());
  a.num_pages = num_pages;
  a.slots = table_slots;
  a.B = B;
  a.T = T;
  a.nkv = nkv;
  a.G = nq / nkv;
  JSX_REQUIRE((int64_t)a.G * (a.G * T + 128) < (1ll << 32), "%d tokens of %d heads per kv head", T, a.G);
  a.per_g = (uint32_t)(((1ull << 32) + a.G - 1) / a.G);
  a.rows = kKaRows;
  a.tiles = (a.G * T + kKaRows - 1) / kKaRows;
  a.pt = page_tokens;
  a.pt_log = page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7;
  a.window = window < (1 << 30) ? window : 1 << 30;  // (positions are below 2^30)
  a.sinks = sinks;
  a.negate = scale < 0.f;
  a.scale_log2 = fabsf(scale) * 1.4426950408889634f;
  if (ka_wide(B, T, nq, nkv, head_dim, n_tokens != nullptr, ka_chunks((int64_t)table_slots * page_tokens, T, a.window, sinks)))
    return kv4_wide_launch(a, a.parts, (cudaStream_t)stream);
  const int64_t items = (int64_t)B * nkv * a.tiles;
  const int64_t chunks = items * (((int64_t)table_slots * page_tokens + kKaChunk - 1) / kKaChunk);
  a.listed = (int64_t)B * a.tiles <= kKaListMax && chunks < (1 << 30);
  const int64_t units = a.listed ? chunks : items;
  const int grid = (int)(units < ka_grid_max() ? units : ka_grid_max());
  return head_dim == 128 ? ka_launch<128>(a, grid, (cudaStream_t)stream) : ka_launch<64>(a, grid, (cudaStream_t)stream);
}
