// Attention over the 4-bit key/value pages for many query rows per kv head (several tokens
// per sequence): items of 128 rows on the tcgen05 tensor cores, head_dim 128.
//
// The kernel of 16-row items (kv4_attn.cu) converts every cache row again for each 16 query
// rows, and its MMA, conversions and multiplications share the issue slots; here a cache row is converted
// once for 128 query rows and both products are issued by one thread.  Per 64 cache rows:
//   warps 6..13  codes -> f16 operands in shared memory, 128-byte swizzled: K [64][128] as it is,
//                V transposed to [128][64] (the nibbles of two rows interleaved before the
//                conversion give a pair along the summed axis);
//   warp 5       S = Q K^T (M 128, N 64, K 128) into one of two TMEM accumulators, then
//                O += P V (M 128, N 128, K 64) once P is there;
//   warps 0..3   a thread per query row: tcgen05.ld of its 64 scores, mask, running reference,
//                weights as f16 into P; O stays in TMEM and is rescaled there on the rare
//                occasions that a row's reference moves;
//   warp 4       places and pages (cp.async.bulk), running ahead.
// S of step n + 1 is issued before P of step n is waited for, so conversions, products and
// weights of neighbouring steps overlap.  A stored value is exact in f16, q is scaled by a
// power of two per row, P has 11 bits: the same roundings as the 16-row kernel's.
//
// NaN: a row's NaN scale enters V as 0 (it would reach every query row through weights of
// 0) and is noted; the query rows that see it get their NaN when they are written.
//
// Items that several CTAs share leave (output, maximum, sum) records, which a second launch
// joins, 16 rows per CTA, in part order.
#include "kv4_attn.cuh"
#include "launch.cuh"

namespace jsx {

constexpr int kKwRows = 128;
constexpr int kKwStep = 64;  // cache rows per product
constexpr int kKwD = 128;
constexpr int kKwStages = 3;
constexpr int kKwThreads = 14 * 32;
constexpr int kKwCopyWarp = 4, kKwMmaWarp = 5, kKwKWarp = 6, kKwVWarp = 10;
constexpr int kKwStage = kv4_block_bytes(kKaChunk, kKwD);
constexpr int kKwQBytes = kKwRows * kKwD * 2;       // two blocks of [128 rows][64]
constexpr int kKwKBytes = kKwStep * kKwD * 2;       // two blocks of [64 rows][64]
constexpr int kKwVBytes = kKwD * kKwStep * 2;       // [128 dimensions][64 rows]
constexpr int kKwPBytes = kKwRows * kKwStep * 2;    // [128 query rows][64 rows]
constexpr int kKwOffK = kKwQBytes, kKwOffV = kKwOffK + 2 * kKwKBytes, kKwOffP = kKwOffV + 2 * kKwVBytes;
constexpr int kKwOffRing = kKwOffP + 2 * kKwPBytes;
constexpr int kKwSmem = kKwOffRing + kKwStages * kKwStage + 1024 /* align */;
constexpr uint32_t kKwTmemCols = 256, kKwTmemO = 128;  // S 0..63, 64..127, O 128..255
constexpr int kKwRecord = kKwRows * kKwD + 2 * kKwRows;  // floats: output, maxima, sums
// f16 x f16 -> f32, both operands K-major
constexpr uint32_t kw_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

int read_clear_kv4_wide_error(uint32_t* out) {
  const uint32_t zero = 0;
  JSX_CUDA(cudaMemcpyFromSymbol(out, g_kv4_error, sizeof(*out)));
  if (*out) JSX_CUDA(cudaMemcpyToSymbol(g_kv4_error, &zero, sizeof(zero)));
  return JSX_OK;
}

__device__ __forceinline__ void kw_sts128(uint32_t p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void kw_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void kw_st32(uint32_t taddr, const float (&v)[32]) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// 16-byte piece c of row r of a 128-byte-swizzled operand block
__device__ __forceinline__ uint32_t kw_at(uint32_t base, int r, int c) { return base + r * 128 + ((c ^ (r & 7)) << 4); }

struct KwInfo {
  int first, parts, odd, pad;  // CTAs of an item: first .. first + parts - 1; odd: the first one's second record
};

__global__ void __launch_bounds__(kKwThreads, 1) k_kv4_attn_wide(const __grid_constant__ KaArgs a, KwInfo* info) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ int cum[kKaListMax + 1];
  __shared__ KaPos place[2];
  __shared__ uint64_t full[kKwStages], empty[kKwStages], kv_full[2], s_full[2], p_full[2], pv_done[2], begun[2], ended[2], q_ready, drained;
  __shared__ uint32_t present[kKwStages];  // pages of the stage that were copied
  __shared__ uint32_t step_rows[2];        // 16-row pieces of the step that are there
  __shared__ uint32_t nan_any[2];          // a byte per V warp
  __shared__ __align__(16) uint8_t nan_row[2][4][kKwStep];  // per V warp (two groups of 16 dimensions) and cache row
  __shared__ uint32_t flags[2], tmem_at;
  volatile uint32_t* abort = flags;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = s_u32(smem);

  if (tid == 0) {
    for (int s = 0; s < kKwStages; ++s) {
      tc_mbar_init(&full[s], 1);
      tc_mbar_init(&empty[s], 8);
    }
    for (int s = 0; s < 2; ++s) {
      tc_mbar_init(&kv_full[s], 8);
      tc_mbar_init(&s_full[s], 1);
      tc_mbar_init(&p_full[s], 4);
      tc_mbar_init(&pv_done[s], 1);
      tc_mbar_init(&begun[s], 1);
      tc_mbar_init(&ended[s], 13);
      nan_any[s] = 0;
    }
    tc_mbar_init(&q_ready, 4);
    tc_mbar_init(&drained, 1);
    flags[0] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < 2 * 4 * kKwStep / 4) reinterpret_cast<uint32_t*>(nan_row)[tid] = 0;
  // rows of P that no thread writes are zero for good
  for (int e = tid; e < 2 * kKwPBytes / 16; e += kKwThreads) kw_sts128(base + kKwOffP + e * 16, 0, 0, 0, 0);
  kw_proxy_fence();
  if (warp == kKwMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(&tmem_at)), "r"(kKwTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  pdl_wait();
  const uint32_t block = kv4_block_bytes(a.pt, kKwD);

  if (warp == kKwCopyWarp) {
    // ---- places and pages ----
    const int pages = kKaChunk >> a.pt_log;
    uint32_t f = 0, k = 0;
    const KaPos first = ka_first(a, cum, lane);
    if (lane == 0) place[0] = first;
    __syncwarp();
    bool ok = true;
    for (;; ++k) {
      KaPos& p = place[k & 1];
      if (lane == 0) tc_arrive(&begun[k & 1]);
      __syncwarp();
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
      int soon = c0 < c1 ? look_up(c0) : -1;
      for (int c = c0; c < c1 && ok; ++c) {
        const uint32_t s = f % kKwStages;
        const int page = soon;
        if (c + 1 < c1) soon = look_up(c + 1);
        if (f >= kKwStages && !ka_wait(&empty[s], (f / kKwStages - 1) & 1, abort)) {
          ok = false;
          break;
        }
        const uint32_t have = __ballot_sync(0xffffffffu, page >= 0 && page < a.num_pages);
        if (lane == 0) {
          present[s] = have;
          tc_expect_tx(&full[s], __popc(have) * block);
        }
        __syncwarp();
        if (have >> lane & 1u)
          ka_copy(smem + kKwOffRing + s * kKwStage + lane * block, a.pool + ((int64_t)page * a.nkv + head) * block, block,
                  &full[s]);
        ++f;
      }
      if (ok && k >= 1) ok = ka_wait(&ended[(k + 1) & 1], ((k + 1) / 2 - 1) & 1, abort);
      if (!ok) break;
      if (lane == 0) {
        place[(k + 1) & 1] = p;
        ka_next(a, cum, &place[(k + 1) & 1]);
      }
      __syncwarp();
    }
    // the copies in flight land before this CTA's shared memory is given away, also when a wait gave up
    for (uint32_t x = f > kKwStages ? f - kKwStages : 0; x < f; ++x)
      tc_wait_err(&full[x % kKwStages], (x / kKwStages) & 1, nullptr, &g_kv4_error);

  } else if (warp == kKwMmaWarp) {
    // ---- products ----
    uint32_t st = 0, asked = 0;  // steps and items with steps so far
    bool ok = true;
    for (uint32_t item = 0; ok; ++item) {
      ok = ka_wait(&begun[item & 1], (item / 2) & 1, abort);
      if (!ok || !place[item & 1].live) break;
      const int steps = (place[item & 1].c1 - place[item & 1].c0) * (kKaChunk / kKwStep);
      if (steps) {
        ok = ka_wait(&q_ready, asked & 1, abort);
        ++asked;
      }
      auto scores = [&](uint32_t x) {  // S of step x
        const uint32_t buf = x & 1;
        if (!ka_wait(&kv_full[buf], (x >> 1) & 1, abort)) return false;
        tc_fence_after();
        if (lane == 0) {
#pragma unroll
          for (int kk = 0; kk < kKwD / 16; ++kk)
            tc_mma(tmem + buf * kKwStep,
                   umma_desc_sw128(base + (kk / 4) * (kKwQBytes / 2) + (kk % 4) * 32),
                   umma_desc_sw128(base + kKwOffK + buf * kKwKBytes + (kk / 4) * (kKwKBytes / 2) + (kk % 4) * 32),
                   kw_idesc(kKwRows, kKwStep), kk > 0);
          tc_commit(&s_full[buf]);
        }
        __syncwarp();
        return true;
      };
      if (ok && steps) ok = scores(st);
      for (int n = 0; n < steps && ok; ++n) {
        const uint32_t x = st + n, buf = x & 1;
        if (n + 1 < steps) ok = scores(x + 1);
        if (ok) ok = ka_wait(&p_full[buf], (x >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
#pragma unroll
          for (int kk = 0; kk < kKwStep / 16; ++kk)
            tc_mma(tmem + kKwTmemO, umma_desc_sw128(base + kKwOffP + buf * kKwPBytes + kk * 32),
                   umma_desc_sw128(base + kKwOffV + buf * kKwVBytes + kk * 32), kw_idesc(kKwRows, kKwD), n > 0 || kk > 0);
          tc_commit(&pv_done[buf]);
        }
        __syncwarp();
      }
      st += steps;
      __syncwarp();
      if (lane == 0) tc_arrive(&ended[item & 1]);
    }
    // products in flight end before TMEM is given back (only after a wait gave up are there any)
    if (lane == 0) tc_commit(&drained);
    __syncwarp();
    tc_wait_err(&drained, 0, nullptr, &g_kv4_error);

  } else if (warp >= kKwKWarp) {
    // ---- codes to operands ----
    const bool is_v = warp >= kKwVWarp;
    const int w = warp - (is_v ? kKwVWarp : kKwKWarp);
    uint32_t st = 0, f = 0;
    bool ok = true;
    for (uint32_t item = 0; ok; ++item) {
      ok = ka_wait(&begun[item & 1], (item / 2) & 1, abort);
      if (!ok || !place[item & 1].live) break;
      const int chunks = place[item & 1].c1 - place[item & 1].c0;
      for (int c = 0; c < chunks && ok; ++c, ++f) {
        const uint32_t s = f % kKwStages;
        ok = ka_wait(&full[s], (f / kKwStages) & 1, abort);
        if (!ok) break;
        const uint32_t ring = base + kKwOffRing + s * kKwStage, have = present[s];
        for (int half = 0; half < kKaChunk / kKwStep && ok; ++half, ++st) {
          const uint32_t buf = st & 1;
          if (st >= 2) ok = ka_wait(&pv_done[buf], ((st >> 1) - 1) & 1, abort);
          if (!ok) break;
          if (!is_v) {
            // four (row, group) units per thread; eight lanes of a phase have eight rows and one group
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int combo = w * 4 + j, key = (combo & 7) * 8 + (lane & 7), g = (combo >> 3) * 4 + (lane >> 3);
              const int r = half * kKwStep + key, page = r >> a.pt_log, in = r & (a.pt - 1);
              const uint32_t at = ring + page * block;
              const uint2 code = ka_lds64(at + in * (kKwD / 2) + g * 8);
              const uint32_t sc = ka_lds8(at + kv4_off_ks(a.pt, kKwD) + in * (kKwD / 16) + g);
              const uint32_t f2 = e4m3x2_to_h2(sc | (sc << 8));
              uint32_t h[8];
              e2m1x8_to_h2(code.x, reinterpret_cast<uint32_t(&)[4]>(h[0]));
              e2m1x8_to_h2(code.y, reinterpret_cast<uint32_t(&)[4]>(h[4]));
#pragma unroll
              for (int i = 0; i < 8; ++i) h[i] = hmul2_u(h[i], f2);
              const uint32_t dst = base + kKwOffK + buf * kKwKBytes + (g >> 2) * (kKwKBytes / 2);
              kw_sts128(kw_at(dst, key, (g & 3) * 2), h[0], h[1], h[2], h[3]);
              kw_sts128(kw_at(dst, key, (g & 3) * 2 + 1), h[4], h[5], h[6], h[7]);
            }
            if (w == 0 && lane == 0) {
              uint32_t rows = 0;
              for (int u = 0; u < kKwStep / 16; ++u) rows |= (have >> ((half * kKwStep + u * 16) >> a.pt_log) & 1u) << u;
              step_rows[buf] = rows;
            }
          } else {
            // eight rows x eight dimensions per thread; eight lanes of a phase have eight row octets
            const int t = w * 32 + lane, ko = t & 7, dimo = t >> 3;
            uint32_t c8[8], s8[8];
            bool odd = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int r = half * kKwStep + ko * 8 + j, page = r >> a.pt_log, in = r & (a.pt - 1);
              const uint32_t at = ring + page * block;
              c8[j] = ka_lds32(at + kv4_off_v(a.pt, kKwD) + in * (kKwD / 2) + dimo * 4);
              s8[j] = ka_lds8(at + kv4_off_vs(a.pt, kKwD) + in * (kKwD / 16) + dimo / 2);
              if (!(have >> page & 1u)) s8[j] = 0;
              odd |= ka_nan_scale(s8[j]);
            }
            uint8_t* any = reinterpret_cast<uint8_t*>(&nan_any[buf]) + w;
            const bool before = *any != 0;
            __syncwarp();
            if (before || __any_sync(0xffffffffu, odd)) {  // this warp's two groups: note the rows
              nan_row[buf][w][lane] = nan_row[buf][w][lane + 32] = 0;
              if (lane == 0) *any = 0;
              __syncwarp();
              for (int half_group = 0; half_group < 2; ++half_group) {  // (bytes of a row are written by one group at a time)
                if ((dimo >> 1 & 1) == half_group && !(dimo & 1)) {
                  for (int j = 0; j < 8; ++j)
                    if (ka_nan_scale(s8[j])) {
                      nan_row[buf][w][ko * 8 + j] |= (uint8_t)(1u << half_group);
                      *any = 1;
                    }
                }
                __syncwarp();
              }
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (ka_nan_scale(s8[j])) s8[j] = 0;
            }
            uint32_t f2[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) f2[p] = e4m3x2_to_h2(s8[2 * p] | (s8[2 * p + 1] << 8));
            const uint32_t dst = base + kKwOffV + buf * kKwVBytes;
#pragma unroll
            for (int par = 0; par < 2; ++par) {  // even and odd dimensions
              uint32_t h[4][4];
#pragma unroll
              for (int p = 0; p < 4; ++p) {
                const uint32_t x = c8[2 * p], y = c8[2 * p + 1];
                e2m1x8_to_h2(par == 0 ? (x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u) : ((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u),
                             h[p]);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                kw_sts128(kw_at(dst, dimo * 8 + 2 * i + par, ko), hmul2_u(h[0][i], f2[0]), hmul2_u(h[1][i], f2[1]),
                          hmul2_u(h[2][i], f2[2]), hmul2_u(h[3][i], f2[3]));
            }
          }
          kw_proxy_fence();
          __syncwarp();
          if (lane == 0) tc_arrive(&kv_full[buf]);
        }
        __syncwarp();
        if (ok && lane == 0) tc_arrive(&empty[s]);
      }
      __syncwarp();
      if (ok && lane == 0) tc_arrive(&ended[item & 1]);
    }

  } else {
    // ---- a query row per thread ----
    const int r = tid;
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    uint32_t st = 0;
    bool ok = true;
    for (uint32_t item = 0; ok; ++item) {
      ok = ka_wait(&begun[item & 1], (item / 2) & 1, abort);
      if (!ok || !place[item & 1].live) break;
      const KaPos& it = place[item & 1];
      const int c0 = it.c0, c1 = it.c1, row = it.tile * kKwRows + r;
      const bool live = row < a.G * a.T;
      const bool busy = __any_sync(0xffffffffu, live);  // rows of this warp are someone's
      const int i = live ? ka_div_g(a, row) : 0, rowpos = it.x.pos + i;
      bf16* out = a.out + ((int64_t)it.b * a.T + i) * a.out_stride + (int64_t)(it.h * a.G + row - i * a.G) * kKwD;
      const bool on = live && i < it.x.used;
      float sc = 1e-37f;
      if (c0 < c1) {
        // q as f16, scaled per row by a power of two
        const uint4* q = reinterpret_cast<const uint4*>(a.q + ((int64_t)it.b * a.T + i) * a.q_stride +
                                                        (int64_t)(it.h * a.G + row - i * a.G) * kKwD);
        uint32_t mx = 0;
#pragma unroll 4
        for (int c = 0; c < kKwD / 8; ++c) {
          const uint4 v = live ? q[c] : make_uint4(0, 0, 0, 0);
          mx = __vmaxu2(__vmaxu2(mx, v.x & 0x7fff7fffu), __vmaxu2(v.y & 0x7fff7fffu, __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
        }
        float undo;
        float mul = ka_q_scale(max(mx & 0xffffu, mx >> 16), &undo);
        sc = fmaxf(a.scale_log2 * undo, 1e-37f);  // never 0: 0 x -inf
        if (a.negate) mul = -mul;
#pragma unroll 4
        for (int c = 0; c < kKwD / 8; ++c) {
          const uint4 v = live ? q[c] : make_uint4(0, 0, 0, 0);
          kw_sts128(kw_at(base + (c / 8) * (kKwQBytes / 2), r, c % 8), ka_h2(bf_lo(v.x) * mul, bf_hi(v.x) * mul),
                    ka_h2(bf_lo(v.y) * mul, bf_hi(v.y) * mul), ka_h2(bf_lo(v.z) * mul, bf_hi(v.z) * mul),
                    ka_h2(bf_lo(v.w) * mul, bf_hi(v.w) * mul));
        }
        kw_proxy_fence();
        __syncwarp();
        if (lane == 0) tc_arrive(&q_ready);
      }
      float m = -INFINITY, l = 0.f;
      uint32_t nan_groups = 0;
      const int all_hi = it.x.pos + it.x.t0, all_lo = a.window > 0 ? it.x.pos + it.x.t1 - a.window + 1 : 0;
      const int sink_chunks = it.x.sink_chunks, lo_chunk = it.x.lo_chunk;
      const int steps = (c1 - c0) * (kKaChunk / kKwStep);
      for (int n = 0; n < steps && ok; ++n, ++st) {
        const uint32_t buf = st & 1, phase = (st >> 1) & 1;
        ok = ka_wait(&kv_full[buf], phase, abort) && ka_wait(&s_full[buf], phase, abort);
        if (!ok) break;
        tc_fence_after();
        if (busy) {
          const int c = c0 + n / 2;
          const int key0 = (c < sink_chunks ? c : lo_chunk + c - sink_chunks) * kKaChunk + (n & 1) * kKwStep;
          const uint32_t rows = step_rows[buf];
          float s[kKwStep];
          tc_ld32(lanes + buf * kKwStep, reinterpret_cast<float(&)[32]>(s[0]));
          tc_ld32(lanes + buf * kKwStep + 32, reinterpret_cast<float(&)[32]>(s[32]));
          auto see = [&](int e) {
            const int key = key0 + e;
            return key <= rowpos && (a.window == 0 || key > rowpos - a.window || key < a.sinks) && (rows >> (e / 16) & 1u);
          };
          if (rows != 0xfu || key0 + kKwStep - 1 > all_hi || (key0 < all_lo && key0 + kKwStep > a.sinks)) {
#pragma unroll
            for (int e = 0; e < kKwStep; ++e)
              if (!see(e)) s[e] = -INFINITY;
          }
          if (nan_any[buf] != 0) {
            for (int e = 0; e < kKwStep; ++e)
              if (see(e))
                for (int x = 0; x < 4; ++x) nan_groups |= (uint32_t)nan_row[buf][x][e] << (2 * x);
          }
          float top = s[0];
#pragma unroll
          for (int e = 1; e < kKwStep; ++e) top = fmaxf(top, s[e]);
          top *= sc;
          const bool move = top > m + kKaLazy;
          if (__any_sync(0xffffffffu, move)) {
            const float f = !move ? 1.f : m == -INFINITY ? 0.f : ka_exp2(m - top);
            if (move) m = top;
            l *= f;
            if (n > 0) {  // O of the steps before is complete, and nothing adds to it until P is handed over
              ok = ka_wait(&pv_done[(st - 1) & 1], ((st - 1) >> 1) & 1, abort);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int x = 0; x < kKwD / 32; ++x) {
                float v[32];
                tc_ld32(lanes + kKwTmemO + x * 32, v);
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] *= f;
                kw_st32(lanes + kKwTmemO + x * 32, v);
              }
            }
          }
          const float ref = m == -INFINITY ? 0.f : kKaOff - m;
          float sum[2] = {0.f, 0.f};
          uint32_t p2[kKwStep / 2];
#pragma unroll
          for (int e = 0; e < kKwStep; e += 2) {
            const float x = ka_exp2(__fmaf_rn(s[e], sc, ref)), y = ka_exp2(__fmaf_rn(s[e + 1], sc, ref));
            sum[0] += x;
            sum[1] += y;
            p2[e / 2] = ka_h2(x, y);
          }
          l += sum[0] + sum[1];
          if (st >= 2) ok = ka_wait(&pv_done[buf], ((st >> 1) - 1) & 1, abort);
          if (!ok) break;
#pragma unroll
          for (int x = 0; x < kKwStep / 8; ++x)
            kw_sts128(kw_at(base + kKwOffP + buf * kKwPBytes, r, x), p2[4 * x], p2[4 * x + 1], p2[4 * x + 2], p2[4 * x + 3]);
          kw_proxy_fence();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) tc_arrive(&p_full[buf]);
      }
      if (!ok) break;
      // ---- the item's end: O out of TMEM ----
      const bool whole = c1 - c0 == it.x.n;
      const int u0 = it.w - c0;
      int first = blockIdx.x, parts = 1;
      if (!whole) {
        first = ka_owner(it, u0);
        parts = ka_owner(it, u0 + it.x.n - 1) - first + 1;
      }
      const int odd = !whole && ka_range(it, first) < u0;
      if (tid == 0 && c0 == 0) info[((int64_t)it.b * a.nkv + it.h) * a.tiles + it.tile] = {first, parts, odd, 0};
      if (steps) {
        ok = ka_wait(&pv_done[(st - 1) & 1], ((st - 1) >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
      }
      float* rec = a.parts + (size_t)(2 * blockIdx.x + (blockIdx.x == (unsigned)first ? odd : 0)) * kKwRecord;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (busy) {
#pragma unroll 1
        for (int x = 0; x < kKwD / 32; ++x) {
          float v[32];
          if (steps) {
            tc_ld32(lanes + kKwTmemO + x * 32, v);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0.f;
          }
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (nan_groups >> (2 * x + e / 16) & 1u) v[e] = NAN;
          if (!live) continue;
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = on ? v[e] * inv : 0.f;
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(out + x * 32 + e) =
                  make_uint4(pack2(v[e], v[e + 1]), pack2(v[e + 2], v[e + 3]), pack2(v[e + 4], v[e + 5]), pack2(v[e + 6], v[e + 7]));
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(rec + r * kKwD + x * 32 + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        }
        if (!whole && live) {
          rec[kKwRows * kKwD + r] = m;
          rec[kKwRows * kKwD + kKwRows + r] = l;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) tc_arrive(&ended[item & 1]);
    }
    // rows of items without a chunk
    if (a.listed) {
      const int items = a.B * a.nkv * a.tiles;
      for (int k = blockIdx.x; k < items; k += gridDim.x) {
        const int tile = k % a.tiles, h = k / a.tiles % a.nkv, b = k / a.tiles / a.nkv;
        if (ka_tile(a, b, tile).n) continue;
        if (tid == 0) info[k] = {0, 1, 0, 0};
        const int row = tile * kKwRows + r, i = ka_div_g(a, row);
        if (row < a.G * a.T)
          for (int d = 0; d < kKwD; d += 8)
            *reinterpret_cast<uint4*>(a.out + ((int64_t)b * a.T + i) * a.out_stride + (int64_t)(h * a.G + row - i * a.G) * kKwD + d) =
                make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kKwMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kKwTmemCols));
  }
}

constexpr int kKjRows = 16, kKjThreads = 128, kKjMost = 160;  // (parts of an item: at most the SMs)

// grid (items, row groups of 16): joins the records of items that several CTAs shared.
__global__ void __launch_bounds__(kKjThreads) k_kv4_join(const __grid_constant__ KaArgs a, const KwInfo* info, int ctas) {
  __shared__ float wgt[kKjMost * kKjRows], part_sum[kKjThreads];
  pdl_wait();
  const int item = blockIdx.x, r0 = blockIdx.y * kKjRows, tid = threadIdx.x;
  const KwInfo x = info[item];
  const int tile = item % a.tiles, h = item / a.tiles % a.nkv, b = item / a.tiles / a.nkv;
  // (the bounds hold unless the first launch gave up before it wrote this)
  if (x.parts <= 1 || x.first < 0 || x.parts > ctas || x.first > ctas - x.parts || tile * kKwRows + r0 >= a.G * a.T) return;
  auto record = [&](int p) { return a.parts + (size_t)(2 * (x.first + p) + (p == 0 && x.odd ? 1 : 0)) * kKwRecord; };
  const int row = tid % kKjRows, p0 = tid / kKjRows, step = kKjThreads / kKjRows;
  float top = -INFINITY;
  for (int p = p0; p < x.parts; p += step) {
    const float m = record(p)[kKwRows * kKwD + r0 + row];
    wgt[p * kKjRows + row] = m;
    top = fmaxf(top, m);
  }
  part_sum[tid] = top;
  __syncthreads();
#pragma unroll
  for (int y = 0; y < kKjThreads / kKjRows; ++y) top = fmaxf(top, part_sum[y * kKjRows + row]);
  __syncthreads();
  float sum = 0.f;
  for (int p = p0; p < x.parts; p += step) {
    const float m = wgt[p * kKjRows + row], f = m == -INFINITY ? 0.f : ka_exp2(m - top);
    wgt[p * kKjRows + row] = f;
    sum += record(p)[kKwRows * kKwD + kKwRows + r0 + row] * f;
  }
  part_sum[tid] = sum;
  __syncthreads();
  constexpr int kMine = kKjRows * kKwD / 4 / kKjThreads;
  float4 acc[kMine];
#pragma unroll
  for (int k = 0; k < kMine; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int q = 0; q < x.parts; q += 4) {
    float4 v[kMine][4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float4* rec = reinterpret_cast<const float4*>(record(min(q + p, x.parts - 1)) + r0 * kKwD);
#pragma unroll
      for (int k = 0; k < kMine; ++k) v[k][p] = rec[tid + k * kKjThreads];
    }
#pragma unroll
    for (int p = 0; p < 4; ++p)
      if (q + p < x.parts)
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
          const float f = wgt[(q + p) * kKjRows + (tid + k * kKjThreads) / (kKwD / 4)];
          acc[k] = make_float4(acc[k].x + v[k][p].x * f, acc[k].y + v[k][p].y * f, acc[k].z + v[k][p].z * f, acc[k].w + v[k][p].w * f);
        }
  }
  const int used = a.n_tokens ? min(max(a.n_tokens[b], 0), a.T) : a.T;
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int e = tid + k * kKjThreads, r = e / (kKwD / 4), d = e % (kKwD / 4) * 4;
    const int query = tile * kKwRows + r0 + r, i = ka_div_g(a, query);
    if (query >= a.G * a.T) continue;
    float l = 0.f;
#pragma unroll
    for (int y = 0; y < kKjThreads / kKjRows; ++y) l += part_sum[y * kKjRows + r];
    const float f = l == 0.f || i >= used ? 0.f : 1.f / l;
    uint2 o = make_uint2(pack2(acc[k].x * f, acc[k].y * f), pack2(acc[k].z * f, acc[k].w * f));
    if (i >= used) o = make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>(a.out + ((int64_t)b * a.T + i) * a.out_stride + (int64_t)(h * a.G + query - i * a.G) * kKwD + d) = o;
  }
}

static size_t kw_info_bytes(int64_t items) { return ((size_t)items * sizeof(KwInfo) + 255) / 256 * 256; }
size_t kv4_wide_workspace(int B, int T, int nq, int nkv) {
  const int64_t items = (int64_t)B * nkv * ((nq / nkv * (int64_t)T + kKwRows - 1) / kKwRows);
  return kw_info_bytes(items) + 2 * (size_t)sm_count() * kKwRecord * 4;
}

// a: all but rows, tiles, listed and the workspace
int kv4_wide_launch(KaArgs a, void* workspace, cudaStream_t s) {
  static bool done[128] = {};
  int dev = 0;
  JSX_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 128 || !done[dev]) {
    JSX_CUDA(cudaFuncSetAttribute(k_kv4_attn_wide, cudaFuncAttributeMaxDynamicSharedMemorySize, kKwSmem));
    if (dev >= 0 && dev < 128) done[dev] = true;
  }
  a.rows = kKwRows;
  a.tiles = (a.G * a.T + kKwRows - 1) / kKwRows;
  const int64_t items = (int64_t)a.B * a.nkv * a.tiles;
  const int64_t chunks = items * (((int64_t)a.slots * a.pt + kKaChunk - 1) / kKaChunk);
  a.listed = (int64_t)a.B * a.tiles <= kKaListMax && chunks < (1 << 30);
  const int64_t units = a.listed ? chunks : items;
  const int most = sm_count() < kKjMost ? sm_count() : kKjMost;
  KwInfo* info = (KwInfo*)workspace;
  a.parts = (float*)((char*)workspace + kw_info_bytes(items));
  a.arrived = nullptr;
  const int ctas = (int)(units < most ? units : most);
  JSX_CUDA(launch_kernel(k_kv4_attn_wide, dim3(ctas), dim3(kKwThreads), kKwSmem, s, a, info));
  if (a.listed) {
    const int rows = a.G * a.T < kKwRows ? a.G * a.T : kKwRows;
    JSX_CUDA(launch_kernel(k_kv4_join, dim3((unsigned)items, (rows + kKjRows - 1) / kKjRows), dim3(kKjThreads), 0, s, a,
                           (const KwInfo*)info, ctas));
  }
  return JSX_OK;
}

}  // namespace jsx
