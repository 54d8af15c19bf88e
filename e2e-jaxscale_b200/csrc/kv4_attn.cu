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
// Inside a CTA one warp copies a chunk's codes and scales into a ring of shared-memory
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
#include <math.h>

#include "common.cuh"
#include "kv4.cuh"
#include "launch.cuh"
#include "tc_core.cuh"

namespace jsx {

constexpr int kKaRows = 16;     // query rows per item
constexpr int kKaChunk = 128;   // cache rows per stage
constexpr int kKaWarps = 4;     // computing warps, 32 cache rows of a chunk each
constexpr int kKaKeys = kKaChunk / kKaWarps;
constexpr int kKaPieces = kKaKeys / 16;
constexpr int kKaThreads = (kKaWarps + 1) * 32;
constexpr int kKaStages = 3;
constexpr int kKaFan = 16;      // parts joined at once
constexpr int kKaLevels = 3;    // 16^3 parts of an item at most
constexpr int kKaListMax = 1024;  // (sequence, row tile) pairs up to which the chunk list is cut into ranges
constexpr float kKaOff = 10.f;  // weights are 2^(s - m + 10): f16 holds them down to 2^-34 of the largest
constexpr float kKaLazy = 4.f;  // the reference m moves when the maximum exceeds it by this much

static __device__ uint32_t g_kv4_error;

int read_clear_kv4_error(uint32_t* out) {
  const uint32_t zero = 0;
  JSX_CUDA(cudaMemcpyFromSymbol(out, g_kv4_error, sizeof(*out)));
  if (*out) JSX_CUDA(cudaMemcpyToSymbol(g_kv4_error, &zero, sizeof(zero)));
  return JSX_OK;
}

struct KaArgs {
  const bf16* q;
  bf16* out;
  int64_t q_stride, out_stride;  // per token, elements
  const uint8_t* pool;
  const int32_t* table;
  const int32_t* positions;
  const int32_t* n_tokens;
  float* parts;       // [2 x CTAs] records
  uint32_t* arrived;  // [kKaLevels][2 x CTAs], zero between calls
  int num_pages, slots, B, T, nkv, G, tiles, pt, window, sinks;
  int listed;  // chunk list cut into ranges; else whole items per CTA
  uint32_t negate;   // 0x80000000 when the scale is negative
  float scale_log2;  // its magnitude x log2(e)
};

template <int D>
struct KaShape {
  static constexpr int kStage = kv4_block_bytes(kKaChunk, D);
  static constexpr int kRecord = kKaRows * D + 2 * kKaRows;  // floats
  static constexpr int kPad = D + 16;                        // row stride of the joining buffer, floats
  static constexpr int kJoin = kKaWarps * kKaRows * (kPad + 2) * 4;
  static constexpr size_t kSmem = (size_t)kKaStages * kStage + kJoin + (kKaListMax + 1) * 8 + 256;
};

// Rows of one (sequence, row tile): tokens t0..t1, cache rows below `hi`, chunks.
struct KaTile {
  int pos, t0, t1, used, hi, lo_chunk, sink_chunks, n;
};

__device__ __forceinline__ KaTile ka_tile(const KaArgs& a, int b, int tile) {
  KaTile x;
  x.pos = min(a.positions[b], 1 << 30);
  x.used = a.n_tokens ? min(max(a.n_tokens[b], 0), a.T) : a.T;
  x.t0 = tile * kKaRows / a.G;
  x.t1 = min(min(tile * kKaRows + kKaRows - 1, a.G * a.T - 1) / a.G, x.used - 1);
  x.hi = min(max(x.pos + x.t1 + 1, 0), a.slots * a.pt);
  x.n = x.lo_chunk = x.sink_chunks = 0;
  if (x.t0 > x.t1 || x.hi == 0) return x;
  const int lo = a.window > 0 ? max(x.pos + x.t0 - a.window + 1, 0) : 0;
  x.lo_chunk = lo / kKaChunk;
  const int end = (x.hi + kKaChunk - 1) / kKaChunk;
  x.sink_chunks = min((min(a.sinks, x.hi) + kKaChunk - 1) / kKaChunk, x.lo_chunk);
  x.n = x.sink_chunks + max(end - x.lo_chunk, 0);
  return x;
}

// The items of one CTA, in order, with the chunks [c0, c1) of each that are its own.
struct KaWalk {
  const KaArgs& a;
  const long long* cum;  // [B + 1] chunks before each sequence
  long long w, w1, total, ctas;  // ctas: CTAs with a range (at least one chunk each)
  int b, h, tile, c0, c1;
  long long item;
  KaTile x;
  __device__ KaWalk(const KaArgs& args, const long long* sums) : a(args), cum(sums) {}
  __device__ void locate() {
    h = (int)(item / a.tiles % a.nkv);
    b = (int)(item / a.tiles / a.nkv);
    tile = (int)(item % a.tiles);
    x = ka_tile(a, b, tile);
    c0 = 0;
    c1 = x.n;
  }
  __device__ bool begin() {
    if (!a.listed) {
      item = blockIdx.x;
      if (item >= (long long)a.B * a.nkv * a.tiles) return false;
      locate();
      return true;
    }
    total = cum[a.B];
    ctas = min((long long)gridDim.x, total);
    if (blockIdx.x >= ctas) return false;
    w = total * blockIdx.x / ctas;
    w1 = total * (blockIdx.x + 1) / ctas;
    int lo = 0, hi = a.B;  // the last sequence whose chunks begin at or before w
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid] <= w) lo = mid;
      else hi = mid;
    }
    b = lo;
    long long off = w - cum[b];
    const long long per = (cum[b + 1] - cum[b]) / a.nkv;
    h = (int)(off / per);
    off -= h * per;
    for (tile = 0;; ++tile) {
      x = ka_tile(a, b, tile);
      if (off < x.n) break;
      off -= x.n;
    }
    c0 = (int)off;
    c1 = (int)min((long long)x.n, off + (w1 - w));
    return true;
  }
  __device__ bool next() {
    if (!a.listed) {
      item += gridDim.x;
      if (item >= (long long)a.B * a.nkv * a.tiles) return false;
      locate();
      return true;
    }
    w += c1 - c0;
    if (w >= w1) return false;
    do {
      if (++tile == a.tiles) {
        tile = 0;
        if (++h == a.nkv) {
          h = 0;
          do ++b;
          while (cum[b + 1] == cum[b]);
        }
      }
      x = ka_tile(a, b, tile);
    } while (x.n == 0);
    c0 = 0;
    c1 = (int)min((long long)x.n, w1 - w);
    return true;
  }
  __device__ int first_key(int c) const {
    return (c < x.sink_chunks ? c : x.lo_chunk + c - x.sink_chunks) * kKaChunk;
  }
};

__device__ __forceinline__ void ka_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(s_u32(dst)),
               "l"(src), "r"(bytes), "r"(s_u32(bar))
               : "memory");
}
__device__ __forceinline__ void ka_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ka_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t ka_h2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ void ka_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool ka_nan_scale(uint32_t s) { return (s & 0x7fu) == 0x7fu; }

// One row's D / 4 values of q at `p` as f16 pairs, scaled by the power of two that brings
// the row's largest magnitude to 2^8 .. 2^9; returns what undoes it.
template <int N>
__device__ __forceinline__ float ka_load_q(const bf16* p, bool live, uint32_t (&h)[N / 2], uint32_t negate) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    const uint4 v = live ? *reinterpret_cast<const uint4*>(p + 8 * i) : make_uint4(0, 0, 0, 0);
    w[4 * i] = v.x;
    w[4 * i + 1] = v.y;
    w[4 * i + 2] = v.z;
    w[4 * i + 3] = v.w;
  }
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) mx = __vmaxu2(mx, w[i] & 0x7fff7fffu);
  uint32_t top = max(mx & 0xffffu, mx >> 16);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int e = (int)(top >> 7);  // exponent field of the largest
  const int f = e == 255 ? 127 : min(262 - e, 254);
  const float mul = __uint_as_float((uint32_t)f << 23 | negate);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) h[i] = ka_h2(bf_lo(w[i]) * mul, bf_hi(w[i]) * mul);
  return f == 254 ? 0x1p-127f : __uint_as_float((uint32_t)(254 - f) << 23);
}

// This thread's part of a row tile's result: 4 values of row r from dimension d on.
__device__ __forceinline__ void ka_store(const KaArgs& a, const KaWalk& it, int D, int r, int d, float4 o, float l) {
  const int row = it.tile * kKaRows + r;
  if (row >= a.G * a.T) return;
  const int i = row / a.G, g = row % a.G;
  const float f = l == 0.f || i >= it.x.used ? 0.f : 1.f / l;
  uint2 v = make_uint2(pack2(o.x * f, o.y * f), pack2(o.z * f, o.w * f));
  if (i >= it.x.used) v = make_uint2(0, 0);
  *reinterpret_cast<uint2*>(a.out + ((int64_t)it.b * a.T + i) * a.out_stride + (it.h * a.G + g) * D + d) = v;
}

template <int D>
__global__ void __launch_bounds__(kKaThreads, 2) k_kv4_attn(KaArgs a) {
  using S = KaShape<D>;
  constexpr int KW = D / 32;      // words of codes per lane and K row
  constexpr int NV = D / 8;       // n tiles of O = dimensions per column
  constexpr int VW = D / 64;      // words of codes per lane and V row
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* ring = smem;
  float* join = reinterpret_cast<float*>(smem + kKaStages * S::kStage);  // [warps][16][kPad], then m and l
  float* join_m = join + kKaWarps * kKaRows * S::kPad;                   // [warps][16]
  float* join_l = join_m + kKaWarps * kKaRows;
  long long* cum = reinterpret_cast<long long*>(smem + kKaStages * S::kStage + S::kJoin);
  uint64_t* full = reinterpret_cast<uint64_t*>(cum + kKaListMax + 1);
  uint64_t* empty = full + kKaStages;
  uint32_t* present = reinterpret_cast<uint32_t*>(empty + kKaStages);  // per stage: 16-row pieces that were copied
  uint32_t* flags = present + kKaStages;                               // [0] a wait gave up, [1] last to arrive
  volatile uint32_t* abort = flags;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int s = 0; s < kKaStages; ++s) {
      tc_mbar_init(&full[s], 1);
      tc_mbar_init(&empty[s], kKaWarps);
    }
    flags[0] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  if (a.listed && warp == 0) {
    // chunks before each sequence
    long long run = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int b = b0 + lane;
      long long n = 0;
      if (b < a.B)
        for (int t = 0; t < a.tiles; ++t) n += ka_tile(a, b, t).n;
      n *= a.nkv;
      long long v = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
      }
      if (b < a.B) cum[b + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) cum[0] = 0;
  }
  __syncthreads();

  if (warp == kKaWarps) {
    // ---- copies: lane = (page of the chunk, array) ----
    KaWalk it(a, cum);
    const int run = min(a.pt, kKaChunk), pages = kKaChunk / run;
    const int j = lane >> 2, arr = lane & 3;
    uint32_t n = 0;
    if (it.begin()) do {
        for (int c = it.c0; c < it.c1; ++c, ++n) {
          const uint32_t s = n % kKaStages;
          const int key = it.first_key(c) + j * run, slot = key / a.pt;
          const int lim = c < it.x.sink_chunks ? min(a.sinks, it.x.hi) : it.x.hi;
          int rows = j < pages ? min(max((lim - key + 15) & ~15, 0), run) : 0;
          int page = -1;
          if (rows > 0 && slot < a.slots) page = a.table[(int64_t)it.b * a.slots + slot];
          if (page < 0 || page >= a.num_pages) rows = 0;
          const uint32_t bytes = rows * (arr < 2 ? D / 2 : D / 16);
          const uint32_t sum = __reduce_add_sync(0xffffffffu, bytes);
          const uint32_t bits = __reduce_or_sync(0xffffffffu, arr == 0 ? ((1u << (rows / 16)) - 1u) << (j * run / 16) : 0u);
          if (n >= kKaStages &&
              !__all_sync(0xffffffffu, tc_wait_err(&empty[s], (n / kKaStages - 1) & 1, abort, &g_kv4_error)))
            goto drained;
          if (lane == 0) {
            present[s] = bits;
            tc_expect_tx(&full[s], sum);
          }
          __syncwarp();
          if (bytes) {
            const uint8_t* src = a.pool + ((int64_t)page * a.nkv + it.h) * kv4_block_bytes(a.pt, D);
            const int row = key - slot * a.pt;
            unsigned char* dst = ring + s * S::kStage;
            if (arr < 2)
              ka_copy(dst + arr * kv4_off_v(kKaChunk, D) + j * run * (D / 2),
                      src + arr * kv4_off_v(a.pt, D) + row * (D / 2), bytes, &full[s]);
            else
              ka_copy(dst + (arr == 2 ? kv4_off_ks(kKaChunk, D) : kv4_off_vs(kKaChunk, D)) + j * run * (D / 16),
                      src + (arr == 2 ? kv4_off_ks(a.pt, D) : kv4_off_vs(a.pt, D)) + row * (D / 16), bytes, &full[s]);
          }
        }
      } while (it.next());
  drained:
    // the copies in flight land before this CTA's shared memory is given away, also when a wait gave up
    for (uint32_t k = n >= kKaStages ? n - kKaStages : 0; k < n; ++k)
      tc_wait_err(&full[k % kKaStages], (k / kKaStages) & 1, nullptr, &g_kv4_error);
    return;
  }

  // ---- the computing warps ----
  const int g = lane >> 2, t = lane & 3;
  bool bad = false;
  uint32_t n = 0;
  KaWalk it(a, cum);
  if (it.begin()) do {
      uint32_t qa[2 * KW][4];
      float sc[2];
      int rowpos[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = it.tile * kKaRows + g + 8 * k, i = row / a.G;
        const bool live = row < a.G * a.T;
        const bf16* p = a.q + ((int64_t)it.b * a.T + (live ? i : 0)) * a.q_stride +
                        (it.h * a.G + (live ? row % a.G : 0)) * D + t * (D / 4);
        uint32_t h[D / 8];
        sc[k] = fmaxf(a.scale_log2 * ka_load_q<D / 4>(p, live, h, a.negate), 1e-37f);  // never 0: 0 x -inf
#pragma unroll
        for (int s = 0; s < 2 * KW; ++s) {
          qa[s][k] = h[2 * s];
          qa[s][2 + k] = h[2 * s + 1];
        }
        rowpos[k] = it.x.pos + min(i, a.T - 1);
      }
      float o[NV][4];
#pragma unroll
      for (int i = 0; i < NV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[4] = {0.f, 0.f, 0.f, 0.f};  // l: sums of rows g and g + 8 in [0] and [2]
      // cache rows that every row of the tile sees
      const int all_hi = it.x.pos + it.x.t0;
      const int all_lo = a.window > 0 ? it.x.pos + it.x.t1 - a.window + 1 : 0;

      for (int c = it.c0; c < it.c1; ++c, ++n) {
        const uint32_t s = n % kKaStages;
        if (!bad) bad = !__all_sync(0xffffffffu, tc_wait_err(&full[s], (n / kKaStages) & 1, abort, &g_kv4_error));
        const int key0 = it.first_key(c) + warp * kKaKeys;
        // 16-row pieces of this warp's rows that were copied
        const uint32_t here = bad ? 0u : (present[s] >> (warp * kKaPieces)) & ((1u << kKaPieces) - 1u);
        if (here) {
          const unsigned char* st = ring + s * S::kStage;
          const bool masked = here != (1u << kKaPieces) - 1u || key0 + kKaKeys - 1 > all_hi ||
                              (key0 < all_lo && key0 + kKaKeys > a.sinks);
          auto see = [&](int e, int p) {  // cache row key0 + e from position p
            const int key = key0 + e;
            return key <= p && (a.window == 0 || key > p - a.window || key < a.sinks) && (here >> (e / 16) & 1u);
          };
          // ---- S = Q K^T ----
          float sa[kKaKeys / 8][4];
          uint32_t kw[kKaKeys / 8][KW], kf[kKaKeys / 8][2];
#pragma unroll
          for (int j = 0; j < kKaKeys / 8; ++j) {
            const int r = warp * kKaKeys + j * 8 + g;
            if constexpr (D == 128) {
              const uint4 v = *reinterpret_cast<const uint4*>(st + r * (D / 2) + t * 16);
              kw[j][0] = v.x;
              kw[j][1] = v.y;
              kw[j][2] = v.z;
              kw[j][3] = v.w;
              const uint32_t x = e4m3x2_to_h2(*reinterpret_cast<const uint16_t*>(st + kv4_off_ks(kKaChunk, D) + r * 8 + t * 2));
              kf[j][0] = __byte_perm(x, 0, 0x1010);
              kf[j][1] = __byte_perm(x, 0, 0x3232);
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(st + r * (D / 2) + t * 8);
              kw[j][0] = v.x;
              kw[j][1] = v.y;
              const uint32_t x = st[kv4_off_ks(kKaChunk, D) + r * 4 + t];
              kf[j][0] = kf[j][1] = e4m3x2_to_h2(x | (x << 8));
            }
            sa[j][0] = sa[j][1] = sa[j][2] = sa[j][3] = 0.f;
          }
#pragma unroll
          for (int k = 0; k < KW; ++k)
#pragma unroll
            for (int j = 0; j < kKaKeys / 8; ++j) {
              uint32_t h[4];
              e2m1x8_to_h2(kw[j][k], h);
              const uint32_t f = kf[j][k * 2 / KW];
              ka_mma(sa[j], qa[2 * k], hmul2_u(h[0], f), hmul2_u(h[1], f));
              ka_mma(sa[j], qa[2 * k + 1], hmul2_u(h[2], f), hmul2_u(h[3], f));
            }
          if (masked) {
#pragma unroll
            for (int j = 0; j < kKaKeys / 8; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!see(j * 8 + 2 * t + (e & 1), rowpos[e >> 1])) sa[j][e] = -INFINITY;
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
          const unsigned char* vs = st + kv4_off_vs(kKaChunk, D) + warp * kKaKeys * (D / 16);
          const unsigned char* vc = st + kv4_off_v(kKaChunk, D) + warp * kKaKeys * (D / 2);
#pragma unroll
          for (int u = 0; u < kKaPieces; ++u) {
            // this lane's rows 2t, 2t + 1 of both 8-row halves, column g
            uint32_t sv[4], w[4][VW];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = u * 16 + (k >> 1) * 8 + 2 * t + (k & 1);
              sv[k] = vs[r * (D / 16) + g * NV / 16];
              if constexpr (D == 128) {
                const uint2 v = *reinterpret_cast<const uint2*>(vc + r * (D / 2) + g * (NV / 2));
                w[k][0] = v.x;
                w[k][1] = v.y;
              } else {
                w[k][0] = *reinterpret_cast<const uint32_t*>(vc + r * (D / 2) + g * (NV / 2));
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
                for (int e = u * 16; e < u * 16 + 16; ++e)
#pragma unroll
                  for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int col = 0; col < 2; ++col)
                      if (see(e, rowpos[k]) && ka_nan_scale(vs[e * (D / 16) + (2 * t + col) * NV / 16]))
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
        if (lane == 0) tc_arrive(&empty[s]);
      }

      // ---- join the four warps ----
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = g + 8 * k;
        if (t == 0) {
          join_m[warp * kKaRows + r] = m[k];
          join_l[warp * kKaRows + r] = l[2 * k];
        }
        float* row = join + (warp * kKaRows + r) * S::kPad;
#pragma unroll
        for (int col = 0; col < 2; ++col)
#pragma unroll
          for (int q0 = 0; q0 < NV / 4; ++q0) {
            const int d = (2 * t + col) * NV + 4 * q0;
            *reinterpret_cast<float4*>(row + d) =
                make_float4(o[4 * q0][2 * k + col], o[4 * q0 + 1][2 * k + col], o[4 * q0 + 2][2 * k + col], o[4 * q0 + 3][2 * k + col]);
          }
      }
      ka_sync();
      // parts of this item: CTAs first .. last of the grid
      const bool whole = it.c1 - it.c0 == it.x.n;
      long long u0 = 0, first = 0, parts = 1;
      if (!whole) {
        u0 = it.w - it.c0;
        first = ((u0 + 1) * it.ctas - 1) / it.total;
        parts = ((u0 + it.x.n) * it.ctas - 1) / it.total - first + 1;
      }
      auto slot_of = [&](long long p) {
        const long long cta = first + p;
        return 2 * cta + (it.total * cta / it.ctas < u0 ? 1 : 0);
      };
      const long long my_part = blockIdx.x - first;
      float* rec = whole ? nullptr : a.parts + slot_of(my_part) * S::kRecord;
      for (int e = tid; e < kKaRows * D / 4; e += kKaWarps * 32) {
        const int r = e / (D / 4), d = e % (D / 4) * 4;
        float top = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kKaWarps; ++w) top = fmaxf(top, join_m[w * kKaRows + r]);
#pragma unroll
        for (int w = 0; w < kKaWarps; ++w) {
          const float mw = join_m[w * kKaRows + r];
          const float f = mw == -INFINITY ? 0.f : ka_exp2(mw - top);
          const float4 v = *reinterpret_cast<const float4*>(join + (w * kKaRows + r) * S::kPad + d);
          sum += join_l[w * kKaRows + r] * f;
          acc.x += v.x * f;
          acc.y += v.y * f;
          acc.z += v.z * f;
          acc.w += v.w * f;
        }
        if (whole) {
          ka_store(a, it, D, r, d, acc, sum);
        } else {
          *reinterpret_cast<float4*>(rec + r * D + d) = acc;
          if (d == 0) {
            rec[kKaRows * D + r] = top;
            rec[kKaRows * D + kKaRows + r] = sum;
          }
        }
      }
      ka_sync();
      // ---- join the CTAs ----
      long long idx = my_part, count = parts, span = 1;
      for (int level = 0; count > 1; ++level) {
        const long long lead = idx / kKaFan * kKaFan;
        const int members = (int)min((long long)kKaFan, count - lead);
        const bool final = count <= kKaFan;
        if (members > 1) {
          __threadfence();
          ka_sync();
          if (tid == 0) {
            uint32_t* ctr = a.arrived + (long long)level * 2 * gridDim.x + slot_of(lead * span);
            const bool last = atomicAdd(ctr, 1u) == (uint32_t)members - 1;
            if (last) *ctr = 0;
            flags[1] = last;
          }
          ka_sync();
          if (!flags[1]) break;
          __threadfence();
          float* wgt = join;                                              // [members][16]
          float** recs = reinterpret_cast<float**>(join + kKaFan * kKaRows);  // [members]
          if (tid < members) recs[tid] = a.parts + slot_of((lead + tid) * span) * S::kRecord;
          ka_sync();
          for (int e = tid; e < members * kKaRows; e += kKaWarps * 32)
            wgt[e] = __ldcg(recs[e / kKaRows] + kKaRows * D + e % kKaRows);
          float lp[kKaFan * kKaRows / (kKaWarps * 32)];
#pragma unroll
          for (int k = 0; k < kKaFan * kKaRows / (kKaWarps * 32); ++k) {
            const int e = tid + k * kKaWarps * 32;
            lp[k] = e < members * kKaRows ? __ldcg(recs[e / kKaRows] + kKaRows * D + kKaRows + e % kKaRows) : 0.f;
          }
          ka_sync();
          float top = -INFINITY;  // of row tid % 16
          for (int p = 0; p < members; ++p) top = fmaxf(top, wgt[p * kKaRows + tid % kKaRows]);
          ka_sync();
          float* sums = join + kKaFan * kKaRows * 2;  // [members][16]
#pragma unroll
          for (int k = 0; k < kKaFan * kKaRows / (kKaWarps * 32); ++k) {
            const int e = tid + k * kKaWarps * 32;
            if (e < members * kKaRows) {
              const float f = wgt[e] == -INFINITY ? 0.f : ka_exp2(wgt[e] - top);
              wgt[e] = f;
              sums[e] = lp[k] * f;
            }
          }
          ka_sync();
          if (tid < kKaRows) {
            float sum = 0.f;
            for (int p = 0; p < members; ++p) sum += sums[p * kKaRows + tid];
            join_m[tid] = top;
            join_l[tid] = sum;
          }
          ka_sync();
          float* dst = recs[0];
          for (int e = tid; e < kKaRows * D / 4; e += kKaWarps * 32) {
            const int r = e / (D / 4), d = e % (D / 4) * 4;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int p = 0; p < kKaFan; ++p) {
              if (p >= members) break;
              const float4 v = __ldcg(reinterpret_cast<const float4*>(recs[p] + r * D + d));
              const float f = wgt[p * kKaRows + r];
              acc.x += v.x * f;
              acc.y += v.y * f;
              acc.z += v.z * f;
              acc.w += v.w * f;
            }
            if (final) {
              ka_store(a, it, D, r, d, acc, join_l[r]);
            } else {
              *reinterpret_cast<float4*>(dst + r * D + d) = acc;
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
    } while (it.next());

  // rows of items without a chunk
  if (a.listed) {
    const long long items = (long long)a.B * a.nkv * a.tiles;
    for (long long k = blockIdx.x; k < items; k += gridDim.x) {
      it.item = k;
      it.locate();
      if (it.x.n) continue;
      for (int e = tid; e < kKaRows * D / 4; e += kKaWarps * 32)
        ka_store(a, it, D, e / (D / 4), e % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
    }
  }
}

// CTAs of a launch: two per SM, or as many as there are chunks (items) at most.
static int ka_grid_max() { return 2 * sm_count(); }
static size_t ka_arrived_bytes() { return ((size_t)kKaLevels * 2 * ka_grid_max() * 4 + 255) / 256 * 256; }
static size_t ka_record_bytes(int D) { return (size_t)(kKaRows * D + 2 * kKaRows) * 4; }

template <int D>
static int ka_launch(const KaArgs& a, int grid, cudaStream_t s) {
  static bool done[128] = {};
  int dev = 0;
  JSX_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 128 || !done[dev]) {
    JSX_CUDA(cudaFuncSetAttribute(k_kv4_attn<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)KaShape<D>::kSmem));
    if (dev >= 0 && dev < 128) done[dev] = true;
  }
  JSX_CUDA(launch_kernel(k_kv4_attn<D>, dim3(grid), dim3(kKaThreads), KaShape<D>::kSmem, s, a));
  return JSX_OK;
}

}  // namespace jsx

using namespace jsx;

extern "C" int jsx_kv4_attn_workspace_size(int B, int T, int nq, int nkv, int head_dim, size_t* bytes) {
  JSX_REQUIRE(bytes && B >= 1 && T >= 1 && nq >= 1 && nkv >= 1 && nq % nkv == 0 && (head_dim == 64 || head_dim == 128),
              "bad arguments");
  *bytes = ka_arrived_bytes() + 2 * (size_t)ka_grid_max() * ka_record_bytes(head_dim);
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
  JSX_REQUIRE(B >= 1 && T >= 1 && (int64_t)B * T * nq <= INT32_MAX, "B=%d T=%d", B, T);
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
  a.tiles = (a.G * T + kKaRows - 1) / kKaRows;
  a.pt = page_tokens;
  a.window = window < (1 << 30) ? window : 1 << 30;  // (positions are below 2^30)
  a.sinks = sinks;
  a.negate = scale < 0.f ? 0x80000000u : 0u;
  a.scale_log2 = fabsf(scale) * 1.4426950408889634f;
  a.listed = (int64_t)B * a.tiles <= kKaListMax;
  const int64_t items = (int64_t)B * nkv * a.tiles;
  const int64_t units = a.listed ? items * (((int64_t)table_slots * page_tokens + kKaChunk - 1) / kKaChunk) : items;
  const int grid = (int)(units < ka_grid_max() ? units : ka_grid_max());
  return head_dim == 128 ? ka_launch<128>(a, grid, (cudaStream_t)stream) : ka_launch<64>(a, grid, (cudaStream_t)stream);
}
