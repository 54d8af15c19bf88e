// Verification of drafted tokens (speculative sampling) from given uniforms.
//
// The target's distribution of row (b, i), i = 0..T, is p = softmax(logits / temperature);
// drafts x_0..x_{n-1} of sequence b come from q (or are certain when no draft
// distribution is given: q(x_i) = 1).  Draft i is accepted while
//     u_i q_i(x_i) < p_i(x_i);
// the first refused one is replaced by a draw from max(p_i - q_i, 0), and when
// none is refused one more token is drawn from p_n, so the output is distributed
// like the target's own samples.
//
// Order-free arithmetic.  Sums over a vocabulary in floating point depend on
// their order, and an inverse-CDF draw turns the last bit into another token.
// So a row's weights are integers, w_v = floor(exp(x_v - max) 2^40): their sum
// Z <= 2^60 is exact in any order, p_v = float(w_v) / float(Z), a residual's
// weight is floor(max(p_v - q_v, 0) 2^40), and the draw is the first v whose
// running sum exceeds floor(u total), u taken to 24 bits.  The floor costs a row
// at most V 2^-41 of its mass (7e-8 at 151552 tokens).
//
// Launches over slices of rows.  With draft distributions three: the rows' maxima, their sums,
// and the weights of the one row per sequence that a token is drawn from, summed per step of 32
// vectors.  Without, the second launch keeps the sums of its steps, which are those weights'.  At
// temperature 0 (greedy: p is 1 at the lowest index of the maximum) one launch finds the maxima
// with their indexes.  The last CTA of a sequence to arrive decides, finds the step with the
// crossing and weighs it again.  Slices meet in integer atomics (maximum, sum), so they need no
// order and no wait; the second pass over the logits comes from L2 (at most 126 MB of it).
// Bound: from some 20 rows on the exponentials' instructions (18 per logit with the exact
// sum, 75% of the issue slots) rather than the bytes; launches below.  32 sequences of up
// to 5 rows of 151552 (129 with their counts) with draft distributions: 44 us, 12 of them the
// maxima (39.1 MB, 3.2 TB/s) and 21 the sums (19.6 million exponentials); 1 x 5
// without: 13.0 us; 16 x up to 8 rows (81) of 32003, greedy: 5.8 us (7.9 in three launches, which also
// cost the host 5 us more).  One cluster per row with distributed shared memory instead of
// atomics: 79 us; one cooperative launch in which the slices wait for one another: 17.7 against
// 13.5 us at 1 x 5.
// NaN logits and a row's -inf entries have no mass; a row with no mass at all, or
// with +inf, accepts nothing and draws token -1 (greedy takes +inf as the maximum).
// A finite maximum whose quotient by the temperature overflows (a row whose mask left only the
// type's lowest value, say) leaves the mass to the entries equal to it: see vf_inv.
#include <math.h>

#include "common.cuh"
#include "launch.cuh"

namespace jsx {

constexpr int kVfThreads = 256;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfMaxDraft = 31;
constexpr int kVfMaxVocab = 1 << 20;
constexpr int kVfMaxPer = 8;  // vectors a thread weighs before its warp adds them up (32 bits hold 15 x 8 x 32 x 2^20)

// Per (sequence, position).  Zero between calls: the slices add and take maxima.
struct __align__(16) VfRow {
  unsigned long long sum;  // Z; at temperature 0 the maximum's key and, below it, ~its index; 0: no distribution
  uint32_t top;            // order key of the largest logit, 0: none
  uint32_t arrived;        // (a sequence's first row) slices done
  float logit, q;          // of the drafted token
  int drafted, pad;        // there is one, inside the vocabulary
};
// (past L1: other CTAs' atomics, and neighbours in a line)
__device__ __forceinline__ VfRow vf_row(const VfRow* r) {
  VfRow x;
  reinterpret_cast<uint4*>(&x)[0] = __ldcg(reinterpret_cast<const uint4*>(r));
  reinterpret_cast<uint4*>(&x)[1] = __ldcg(reinterpret_cast<const uint4*>(r) + 1);
  return x;
}

struct VfArgs {
  const void* logits;
  const int32_t* ids;
  const float* probs;  // [B][T][V] or null
  const int32_t* n_draft;
  const float* u;  // [B][T + 1]
  VfRow* rows;     // [B][T + 1]
  unsigned long long* steps;  // [B][T + 1][step_stride] sums of 32 vectors each (with q: a sequence's first row only)
  int32_t* accepted;
  int32_t* tokens;
  float* accept_prob;
  int64_t row_stride;  // of logits, elements
  int T, V, per, step_stride;
  float inv_temp;  // 0: greedy
};

// A row as 16-byte vectors: vector j holds elements j N - skew .. + N - 1, where
// skew is the row's distance from the 16-byte boundary below it.
template <typename E>
struct VfVec {
  static constexpr int N = 16 / sizeof(E);
  const E* base;
  int skew, V, count;
  __device__ VfVec(const E* row, int v) : base(row), V(v) {
    skew = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(E));
    count = (skew + V + N - 1) / N;
  }
  __device__ int first(int j) const { return j * N - skew; }
  // elements outside the row read as -inf
  __device__ uint4 load(int j) const {
    const int e = first(j);
    if (e >= 0 && e + N <= V) return *reinterpret_cast<const uint4*>(base + e);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(E) == 2) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base);
        const uint32_t lo = e + 2 * i >= 0 && e + 2 * i < V ? p[e + 2 * i] : 0xff80u;
        const uint32_t hi = e + 2 * i + 1 >= 0 && e + 2 * i + 1 < V ? p[e + 2 * i + 1] : 0xff80u;
        w[i] = lo | hi << 16;
      } else {
        w[i] = e + i >= 0 && e + i < V ? __float_as_uint(base[e + i]) : 0xff800000u;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static void unpack(const uint4& w, float (&x)[N]) {
    if constexpr (sizeof(E) == 2) {
      unpack8(w, x);
    } else {
      x[0] = __uint_as_float(w.x);
      x[1] = __uint_as_float(w.y);
      x[2] = __uint_as_float(w.z);
      x[3] = __uint_as_float(w.w);
    }
  }
  // the larger of top and a vector's elements, NaN ignored
  __device__ static float max(const uint4& w, float top) {
    if constexpr (sizeof(E) == 2) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
      const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(top, fmaxf(__low2float(m), __high2float(m)));
    } else {
      return fmaxf(fmaxf(fmaxf(top, __uint_as_float(w.x)), fmaxf(__uint_as_float(w.y), __uint_as_float(w.z))),
                   __uint_as_float(w.w));
    }
  }
};

// floor(e 2^40) for e in [0, 1], NaN as 0, without conversions: adding 8 (2^-17) with
// rounding towards zero leaves the multiples of 2^-20 (2^-40) in the low mantissa bits.
// hi and lo collect the raw bits of n numbers; the constants' share is taken off at the end.
constexpr float kVfHi = 8.f, kVfLo = 0x1p-17f;
struct VfFix {
  uint32_t hi = 0, lo = 0, n = 0;
  // adds one, and returns it truncated to a multiple of 2^-40
  __device__ __forceinline__ float add(float e) {
    e = fmaxf(e, 0.f);
    const float f = __fadd_rz(e, kVfHi), t = f - kVfHi;
    const float g = __fadd_rz(e - t, kVfLo);
    hi += __float_as_uint(f);
    lo += __float_as_uint(g);
    ++n;
    return t + (g - kVfLo);
  }
  __device__ __forceinline__ unsigned long long sum() const {
    return ((unsigned long long)(hi - n * __float_as_uint(kVfHi)) << 20) + (lo - n * __float_as_uint(kVfLo));
  }
  // over the warp: 32 x 8 x 8 numbers of at most 2^20 in each part
  __device__ __forceinline__ unsigned long long warp_sum() const {
    const uint32_t h = __reduce_add_sync(0xffffffffu, hi - n * __float_as_uint(kVfHi));
    const uint32_t l = __reduce_add_sync(0xffffffffu, lo - n * __float_as_uint(kVfLo));
    return ((unsigned long long)h << 20) + l;
  }
};
// The product is rounded before the subtraction (no fused multiply-add): the row's
// maximum is the maximum of rounded products, and its own weight is exactly 2^40.
__device__ __forceinline__ float vf_exp(float logit, float inv_temp, float mx) {
  return expf(__fsub_rn(__fmul_rn(logit, inv_temp), mx));
}

// larger floats have larger keys; -inf has 0x007fffff, NaN is not asked
__device__ __forceinline__ uint32_t vf_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float vf_unkey(uint32_t k) {
  return k == 0 ? -INFINITY : __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// The factor of a row's logits before the exponential: 1 / temperature, or, where the row's largest
// logit is finite and that product is not, a power of two that brings the largest to 2^100.  Two
// logits of such a row differ by at least 2^-24 of the largest's magnitude, far more than a
// weight can span under either factor: equal ones weigh 1, the others 0.  (1 / temperature is
// below 2^128, so the largest's magnitude is at least 1/2 there and the exponent in range.)
__device__ __forceinline__ float vf_inv(float top, float inv_temp) {
  if (fabsf(__fmul_rn(top, inv_temp)) < INFINITY || !(fabsf(top) < INFINITY)) return inv_temp;
  const uint32_t e = (__float_as_uint(top) >> 23) & 0xffu;
  return __uint_as_float((354u - e) << 23);
}
__device__ __forceinline__ int vf_drafts(const VfArgs& a, int b) {
  return a.n_draft ? min(max(a.n_draft[b], 0), a.T) : a.T;
}

// grid (slices, rows): a CTA has kVfThreads x per vectors of a row.  Rows after a
// sequence's last draft but one are not looked at.
template <typename E>
__global__ void __launch_bounds__(kVfThreads) k_verify_max(VfArgs a) {
  pdl_wait();
  const int b = blockIdx.y / (a.T + 1), i = blockIdx.y % (a.T + 1), nd = vf_drafts(a, b);
  if (i > nd) return;
  const E* lg = (const E*)a.logits + (int64_t)blockIdx.y * a.row_stride;
  VfRow* row = a.rows + blockIdx.y;
  const VfVec<E> vec(lg, a.V);
  float top = -INFINITY;
  const int j0 = blockIdx.x * kVfThreads * a.per + threadIdx.x;
  const uint32_t low = sizeof(E) == 2 ? 0xff80ff80u : 0xff800000u;
  for (int k = 0; k < a.per; k += 4) {  // four loads in flight
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + (k + u) * kVfThreads;
      v[u] = k + u < a.per && j < vec.count ? vec.load(j) : make_uint4(low, low, low, low);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) top = vec.max(v[u], top);
  }
  const uint32_t key = __reduce_max_sync(0xffffffffu, vf_key(fmaxf(top, -INFINITY)));
  if ((threadIdx.x & 31) == 0 && key > vf_key(-INFINITY)) atomicMax(&row->top, key);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    int drafted = 0;
    if (i < nd) {
      const int id = a.ids[(int64_t)b * a.T + i];
      drafted = id >= 0 && id < a.V;
      if (drafted) {
        row->logit = (float)lg[id];
        row->q = a.probs ? a.probs[((int64_t)b * a.T + i) * a.V + id] : 1.f;
      }
    }
    row->drafted = drafted;
  }
}

// What a sequence's rows say: drafts accepted, and the row the next token is drawn from.
struct VfSeq {
  VfRow row;
  int accepted;
  bool refused;
};
// By a whole warp, lane i for draft i; prob: lane i's min(1, p / q).
__device__ __forceinline__ VfSeq vf_decide(const VfArgs& a, int b, float* prob) {
  const int lane = threadIdx.x & 31, nd = vf_drafts(a, b);
  const VfRow* rows = a.rows + (int64_t)b * (a.T + 1);
  bool ok = false;
  *prob = 0.f;
  if (lane < nd) {
    const VfRow r = vf_row(rows + lane);
    if (a.inv_temp == 0.f) {
      ok = r.sum != 0 && (int)~(uint32_t)r.sum == a.ids[(int64_t)b * a.T + lane];
      *prob = ok ? 1.f : 0.f;
    } else if (r.drafted) {
      {
        VfFix f;
        const float top = vf_unkey(r.top), inv = vf_inv(top, a.inv_temp);
        const float w = f.add(vf_exp(r.logit, inv, __fmul_rn(top, inv)));
        const float p = r.sum ? __fdiv_rn(w, (float)r.sum * 0x1p-40f) : 0.f;
        ok = __fmul_rn(a.u[(int64_t)b * (a.T + 1) + lane], r.q) < p;
        *prob = r.q > 0.f ? fminf(__fdiv_rn(p, r.q), 1.f) : p > 0.f ? 1.f : 0.f;
      }
    }
  }
  VfSeq s;
  s.accepted = __ffs((int)__ballot_sync(0xffffffffu, !ok)) - 1;  // nd <= 31: lane nd has none
  s.refused = s.accepted < nd;
  s.row = vf_row(rows + s.accepted);
  return s;
}

// The weights of the row that a token is drawn from.
template <typename E>
struct VfDraw {
  static constexpr int N = VfVec<E>::N;
  VfVec<E> vec;
  const float* q;
  bool q_vec, residual;
  int id;
  float z, mx, inv_temp;
  __device__ VfDraw(const VfArgs& a, int b, const VfSeq& s)
      : vec((const E*)a.logits + ((int64_t)b * (a.T + 1) + s.accepted) * a.row_stride, a.V) {
    residual = s.refused;
    id = s.refused ? a.ids[(int64_t)b * a.T + s.accepted] : -1;
    q = s.refused && a.probs ? a.probs + ((int64_t)b * a.T + s.accepted) * a.V : nullptr;
    q_vec = ((reinterpret_cast<uintptr_t>(q) - vec.skew * 4) & 15u) == 0;
    z = (float)s.row.sum * 0x1p-40f;
    const float top = vf_unkey(s.row.top);
    inv_temp = vf_inv(top, a.inv_temp);
    mx = __fmul_rn(top, inv_temp);
  }
  // adds the weights of vector j to f; `each`: the running sums after every element
  __device__ __forceinline__ void weigh(int j, VfFix& f, unsigned long long* each) const {
    float x[N], d[N];
    vec.unpack(vec.load(j), x);
    const int v0 = vec.first(j);
    if (residual && q) {
      if (q_vec && v0 >= 0 && v0 + N <= vec.V) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          const float4 y = *reinterpret_cast<const float4*>(q + v0 + e);
          d[e] = y.x;
          d[e + 1] = y.y;
          d[e + 2] = y.z;
          d[e + 3] = y.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) d[e] = v0 + e >= 0 && v0 + e < vec.V ? q[v0 + e] : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float y = vf_exp(x[e], inv_temp, mx);
      if (residual) {
        if (!q) {
          if (v0 + e == id) y = 0.f;
        } else {
          VfFix one;
          const float p = __fdiv_rn(one.add(y), z);
          y = p > d[e] ? p - d[e] : 0.f;
        }
      }
      f.add(y);
      if (each) each[e] = f.sum();
    }
  }
};

// floor(total u) with u taken to 24 bits; total < 2^63
__device__ __forceinline__ unsigned long long vf_threshold(unsigned long long total, float u) {
  float t = u * 16777216.f;
  t = t > 0.f ? fminf(t, 16777215.f) : 0.f;
  const unsigned long long f = (unsigned long long)t;
  return (total >> 32) * f * 256ull + (((total & 0xffffffffull) * f) >> 24);
}
__device__ __forceinline__ unsigned long long vf_scan(unsigned long long x) {  // inclusive, over a warp
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// By one CTA per sequence: the draw, the outputs, and the workspace zero again.
// steps: of the row that is drawn from; without q they are the row's own weights.
template <typename E>
__device__ __forceinline__ void vf_pick(const VfArgs& a, int b, const VfSeq& s, float prob, float u, unsigned long long* steps) {
  __shared__ unsigned long long warps[kVfWarps], reached;
  __shared__ int token;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, T = a.T;
  if (tid < T) a.accept_prob[(int64_t)b * T + tid] = prob;
  if (tid == 0) {
    a.accepted[b] = s.accepted;
    token = a.inv_temp == 0.f && s.row.sum != 0 ? (int)~(uint32_t)s.row.sum : -1;
  }
  if (a.inv_temp != 0.f && s.row.sum != 0) {
    VfDraw<E> draw(a, b, s);
    constexpr int N = VfDraw<E>::N;
    const int n = (draw.vec.count + 31) / 32, per = (n + kVfThreads - 1) / kVfThreads;
    unsigned long long mine, before, total;
    if (!a.probs && s.refused && s.row.drafted) {  // without the refused token
      if (tid == 0) {
        VfFix f;
        f.add(vf_exp(s.row.logit, draw.inv_temp, draw.mx));
        steps[(draw.id + draw.vec.skew) / N / 32] -= f.sum();
      }
      __syncthreads();
    }
    for (;;) {
      // thread t has steps [t per, (t + 1) per)
      mine = 0;
#pragma unroll 4
      for (int k = tid * per; k < min(n, (tid + 1) * per); ++k) mine += __ldcg(steps + k);
      const unsigned long long x = vf_scan(mine);
      if (lane == 31) warps[warp] = x;
      __syncthreads();
      before = x - mine;
      total = 0;
#pragma unroll
      for (int w = 0; w < kVfWarps; ++w) {
        if (w < warp) before += warps[w];
        total += warps[w];
      }
      if (total != 0 || !draw.residual) break;
      // p nowhere above q (rounding): the target's own distribution, weighed here
      draw.residual = false;
      __syncthreads();
      for (int k = warp; k < n; k += kVfWarps) {
        VfFix f;
        if (k * 32 + lane < draw.vec.count) draw.weigh(k * 32 + lane, f, nullptr);
        const unsigned long long y = f.warp_sum();
        if (lane == 0) steps[k] = y;
      }
      __syncthreads();
    }
    const unsigned long long at = vf_threshold(total, u);
    if (before <= at && at < before + mine) {  // one thread: its step with the crossing
      int k = tid * per;
      for (unsigned long long x; before + (x = __ldcg(steps + k)) <= at; ++k) before += x;
      reached = before;
      token = k;
    }
    __syncthreads();
    const int j = token * 32 + lane;
    before = reached;
    __syncthreads();
    if (warp == 0) {
      unsigned long long each[N], sum = 0;
      VfFix f;
      if (j < draw.vec.count) {
        draw.weigh(j, f, each);
        sum = f.sum();
      }
      const unsigned long long upto = before + vf_scan(sum);
      if (upto - sum <= at && at < upto) {
        int e = 0;
        while (upto - sum + each[e] <= at) ++e;
        token = draw.vec.first(j) + e;
      }
    }
  }
  __syncthreads();
  if (tid <= T) {
    int t = -1;
    if (tid < s.accepted) t = a.ids[(int64_t)b * T + tid];
    if (tid == s.accepted) t = token;
    a.tokens[(int64_t)b * (T + 1) + tid] = t;
    a.rows[(int64_t)b * (T + 1) + tid] = VfRow{};
  }
  if (a.inv_temp != 0.f) {  // (the next call's records may lie here)
    const int64_t n = (int64_t)a.step_stride * (a.probs ? 1 : T + 1);
    for (int64_t k = tid; k < n; k += kVfThreads) a.steps[(int64_t)b * (T + 1) * a.step_stride + k] = 0;
  }
}

// grid as above: the rows' sums.  Without draft distributions (kDraw) also the sums of every
// step (32 vectors, a warp), which are all that a draw needs: the last CTA of a sequence to
// arrive draws its token.
template <typename E, bool kDraw>
__global__ void __launch_bounds__(kVfThreads) k_verify_sum(VfArgs a) {
  pdl_wait();
  const int b = blockIdx.y / (a.T + 1), i = blockIdx.y % (a.T + 1), nd = vf_drafts(a, b);
  if (i > nd) return;
  constexpr int N = VfVec<E>::N;
  VfRow* row = a.rows + blockIdx.y;
  const VfVec<E> vec((const E*)a.logits + (int64_t)blockIdx.y * a.row_stride, a.V);
  // rounding is monotonic: the largest product is the largest logit's
  const float top = vf_unkey(row->top), inv_temp = vf_inv(top, a.inv_temp), mx = __fmul_rn(top, inv_temp);
  const int lane = threadIdx.x & 31, first = blockIdx.x * kVfThreads * a.per;
  if (fabsf(mx) < INFINITY) {
    VfFix f;
    unsigned long long sum = 0;
    for (int k = 0; k < a.per; ++k) {
      const int j = first + k * kVfThreads + (int)threadIdx.x;
      if (j - lane >= vec.count) break;
      if (j < vec.count) {
        float x[N];
        vec.unpack(vec.load(j), x);
#pragma unroll
        for (int e = 0; e < N; ++e) f.add(vf_exp(x[e], inv_temp, mx));
      }
      if (kDraw) {
        const unsigned long long y = f.warp_sum();
        if (lane == 0) a.steps[(int64_t)blockIdx.y * a.step_stride + j / 32] = y;
        sum += y;
        f = VfFix();
      }
    }
    if (!kDraw) sum = f.warp_sum();
    if (lane == 0 && sum) atomicAdd(&row->sum, sum);
  }
  if (!kDraw) return;
  __shared__ bool last;
  if (lane == 0) __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&a.rows[(int64_t)b * (a.T + 1)].arrived, 1u) == gridDim.x * (nd + 1) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  float prob;
  const VfSeq s = vf_decide(a, b, &prob);
  vf_pick<E>(a, b, s, prob, a.u[(int64_t)b * (a.T + 1) + a.T],
             a.steps + ((int64_t)b * (a.T + 1) + s.accepted) * a.step_stride);
}

// grid (slices, sequences), with draft distributions: the weights' sums of every step of the
// row that a token is drawn from; the last CTA of a sequence to arrive draws it
template <typename E>
__global__ void __launch_bounds__(kVfThreads) k_verify_weigh(VfArgs a) {
  __shared__ bool last;
  pdl_wait();
  const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float u = a.u[(int64_t)b * (a.T + 1) + a.T];
  float prob;
  const VfSeq s = vf_decide(a, b, &prob);
  unsigned long long* steps = a.steps + (int64_t)b * (a.T + 1) * a.step_stride;
  if (s.row.sum != 0) {
    const VfDraw<E> draw(a, b, s);
    for (int k = 0; k < a.per; ++k) {
      const int step = (blockIdx.x * a.per + k) * kVfWarps + warp, j = step * 32 + lane;
      if (step * 32 >= draw.vec.count) break;
      VfFix f;
      if (j < draw.vec.count) draw.weigh(j, f, nullptr);
      const unsigned long long x = f.warp_sum();
      if (lane == 0) steps[step] = x;
    }
  }
  if (lane == 0) __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&a.rows[(int64_t)b * (a.T + 1)].arrived, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  vf_pick<E>(a, b, s, prob, u, steps);
}

// Temperature 0, one launch: grid (slices, rows); slices meet in the maximum of (key, ~index),
// and the last CTA of a sequence to arrive decides.
template <typename E>
__global__ void __launch_bounds__(kVfThreads) k_verify_greedy(VfArgs a) {
  __shared__ bool last;
  pdl_wait();
  const int b = blockIdx.y / (a.T + 1), i = blockIdx.y % (a.T + 1), nd = vf_drafts(a, b);
  if (i > nd) return;
  constexpr int N = VfVec<E>::N;
  const VfVec<E> vec((const E*)a.logits + (int64_t)blockIdx.y * a.row_stride, a.V);
  float best = -INFINITY;
  int at = 0;
  const int j0 = blockIdx.x * kVfThreads * a.per + threadIdx.x;
  const uint32_t low = sizeof(E) == 2 ? 0xff80ff80u : 0xff800000u;
  for (int k = 0; k < a.per; k += 4) {  // four loads in flight
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + (k + u) * kVfThreads;
      v[u] = k + u < a.per && j < vec.count ? vec.load(j) : make_uint4(low, low, low, low);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float was = best;
      best = vec.max(v[u], best);
      if (best > was) {  // a new maximum: its first index in this vector
        float x[N];
        vec.unpack(v[u], x);
        at = vec.first(j0 + (k + u) * kVfThreads);
        int e = 0;
#pragma unroll
        for (int y = N - 1; y >= 0; --y)
          if (x[y] == best) e = y;
        at += e;
      }
    }
  }
  // (-0 as +0: they are equal, the first of them counts)
  unsigned long long key = best > -INFINITY ? (unsigned long long)vf_key(best + 0.f) << 32 | (uint32_t)~at : 0ull;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long y = __shfl_xor_sync(0xffffffffu, key, o);
    key = y > key ? y : key;
  }
  if ((threadIdx.x & 31) == 0) {
    if (key) atomicMax(&a.rows[blockIdx.y].sum, key);
    __threadfence();
  }
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&a.rows[(int64_t)b * (a.T + 1)].arrived, 1u) == gridDim.x * (nd + 1) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  float prob;
  const VfSeq s = vf_decide(a, b, &prob);
  vf_pick<E>(a, b, s, prob, 0.f, nullptr);
}

template <typename E>
static int verify_launch(VfArgs& a, int B, cudaStream_t s) {
  // eight CTAs per SM (a full one) where the rows suffice: more, shorter ones cost more to
  // launch than they even out (32 x 5 rows of 151552: 12.7 us for the maxima, 20.9 us at one vector a thread)
  const int most = (a.V + 2 * VfVec<E>::N - 2) / VfVec<E>::N;  // vectors of a row, wherever it begins
  auto cut = [&](int rows) {
    const int64_t units = (int64_t)rows * ((most + kVfThreads - 1) / kVfThreads);
    const int64_t per = (units + 8ll * sm_count() - 1) / (8ll * sm_count());
    a.per = (int)(per < 1 ? 1 : per > kVfMaxPer ? kVfMaxPer : per);
    return (unsigned)((most + kVfThreads * a.per - 1) / (kVfThreads * a.per));
  };
  const unsigned slices = cut(B * (a.T + 1));
  const dim3 grid(slices, B * (a.T + 1));
  if (a.inv_temp == 0.f) {
    JSX_CUDA(launch_kernel(k_verify_greedy<E>, grid, dim3(kVfThreads), 0, s, a));
    return JSX_OK;
  }
  JSX_CUDA(launch_kernel(k_verify_max<E>, grid, dim3(kVfThreads), 0, s, a));
  if (!a.probs) {
    JSX_CUDA(launch_kernel(k_verify_sum<E, true>, grid, dim3(kVfThreads), 0, s, a));
    return JSX_OK;
  }
  JSX_CUDA(launch_kernel(k_verify_sum<E, false>, grid, dim3(kVfThreads), 0, s, a));
  const unsigned n = cut(B);
  JSX_CUDA(launch_kernel(k_verify_weigh<E>, dim3(n, B), dim3(kVfThreads), 0, s, a));
  return JSX_OK;
}

}  // namespace jsx

using namespace jsx;

// steps of a row: the 32-bit form has the most
static int64_t vf_steps(int V) { return (V + 6) / 4 / 32 + 1; }

extern "C" int jsx_verify_workspace_size(int B, int T, int V, size_t* bytes) {
  JSX_REQUIRE(bytes && B >= 1 && T >= 0 && T <= kVfMaxDraft && V >= 1 && V <= kVfMaxVocab, "bad arguments");
  *bytes = (size_t)B * (T + 1) * sizeof(VfRow) + (size_t)B * (T + 1) * vf_steps(V) * 8;
  return JSX_OK;
}

extern "C" int jsx_verify_drafts(const void* logits, int logits_f32, int64_t row_stride, const int32_t* draft_ids,
                                 const float* draft_probs, const int32_t* n_draft, const float* uniforms,
                                 float temperature, int32_t* accepted, int32_t* tokens, float* accept_prob, int B,
                                 int T, int V, void* workspace, size_t workspace_bytes, void* stream) {
  JSX_REQUIRE(B >= 1 && T >= 0 && T <= kVfMaxDraft && (int64_t)B * (T + 1) <= 65535, "B=%d T=%d (T in 0..%d, B (T + 1) up to 65535)", B,
              T, kVfMaxDraft);
  JSX_REQUIRE(V >= 1 && V <= kVfMaxVocab && row_stride >= V, "V=%d (1..%d) row_stride=%lld", V, kVfMaxVocab,
              (long long)row_stride);
  JSX_REQUIRE(logits && accepted && tokens, "null pointer argument");
  JSX_REQUIRE(T == 0 || (draft_ids && accept_prob), "null draft_ids or accept_prob");
  JSX_REQUIRE(temperature >= 0.f && temperature <= 3.4e38f, "temperature must be finite and not negative");
  JSX_REQUIRE(uniforms || temperature == 0.f, "null uniforms");
  JSX_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (logits_f32 ? 3u : 1u)) == 0, "unaligned logits");
  size_t need = 0;
  const int st = jsx_verify_workspace_size(B, T, V, &need);
  if (st) return st;
  JSX_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, "workspace of %zu bytes, %zu needed",
              workspace_bytes, need);
  VfArgs a;
  a.logits = logits;
  a.ids = draft_ids;
  a.probs = draft_probs;
  a.n_draft = n_draft;
  a.u = uniforms;
  a.rows = (VfRow*)workspace;
  a.steps = (unsigned long long*)((char*)workspace + (size_t)B * (T + 1) * sizeof(VfRow));
  a.step_stride = (int)vf_steps(V);
  a.accepted = accepted;
  a.tokens = tokens;
  a.accept_prob = accept_prob;
  a.row_stride = row_stride;
  a.T = T;
  a.V = V;
  a.inv_temp = temperature == 0.f ? 0.f : 1.f / temperature;
  JSX_REQUIRE(temperature == 0.f || (a.inv_temp > 0.f && a.inv_temp <= 3.4e38f), "temperature %g out of range",
              (double)temperature);
  return logits_f32 ? verify_launch<float>(a, B, (cudaStream_t)stream) : verify_launch<bf16>(a, B, (cudaStream_t)stream);
}
