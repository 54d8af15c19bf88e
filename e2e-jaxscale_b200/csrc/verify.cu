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
// Two launches, each one cluster of 8 CTAs per row (stats: every row; draw: one
// row per sequence): a row of 151552 bf16 logits is 303 KB, an eighth of it is read
// from memory once and the second pass (the sum after the maximum) hits L1.
// Temperature 0 is greedy: p is 1 at the lowest index of the maximum.
// NaN logits and a row's -inf entries have no mass; a row with no mass at all, or
// with +inf, accepts nothing and draws token -1 (greedy takes +inf as the maximum).
#include <math.h>

#include "common.cuh"
#include "launch.cuh"

namespace jsx {

constexpr int kVfCtas = 8;
constexpr int kVfThreads = 512;
constexpr int kVfMaxDraft = 31;
constexpr int kVfMaxVocab = 1 << 20;

struct VfRow {  // per (sequence, position), written by the first kernel
  unsigned long long sum;  // Z; 0: no distribution
  float max;
  int best;  // temperature 0: argmax, -1 none
  int ok;    // draft accepted (positions < n_draft)
  int pad;
};

struct VfArgs {
  const void* logits;
  const int32_t* ids;
  const float* probs;  // [B][T][V] or null
  const int32_t* n_draft;
  const float* u;  // [B][T + 1]
  VfRow* rows;
  int32_t* accepted;
  int32_t* tokens;
  float* accept_prob;
  int64_t row_stride;  // of logits, elements
  int T, V;
  float inv_temp;  // 0: greedy
};

__device__ __forceinline__ uint32_t vf_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void vf_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned long long vf_peer(const unsigned long long* p, uint32_t rank) {
  uint32_t a;
  unsigned long long v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}

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
  // elements outside the row read as `fill`
  __device__ void load(int j, float (&x)[N], float fill) const {
    const int e = first(j);
    if (e >= 0 && e + N <= V) {
      const uint4 w = *reinterpret_cast<const uint4*>(base + e);
      if constexpr (sizeof(E) == 2) {
        unpack8(w, x);
      } else {
        x[0] = __uint_as_float(w.x);
        x[1] = __uint_as_float(w.y);
        x[2] = __uint_as_float(w.z);
        x[3] = __uint_as_float(w.w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = e + i >= 0 && e + i < V ? (float)base[e + i] : fill;
    }
  }
};

// floor(e 2^40) for e in [0, 1] as hi 2^20 + lo; NaN gives 0.  Adding 2^23 with
// rounding towards zero leaves the integer part in the low mantissa bits.
__device__ __forceinline__ void vf_fix(float e, uint32_t& hi, uint32_t& lo) {
  e = e > 0.f ? e : 0.f;
  const float t = e * 1048576.f;
  const float f = __fadd_rz(t, 8388608.f);
  hi = __float_as_uint(f) & 0x7fffffu;
  const float r = (t - (f - 8388608.f)) * 1048576.f;
  lo = __float_as_uint(__fadd_rz(r, 8388608.f)) & 0x7fffffu;
}
__device__ __forceinline__ unsigned long long vf_join(uint32_t hi, uint32_t lo) {
  return ((unsigned long long)hi << 20) + lo;
}
// The product is rounded before the subtraction (no fused multiply-add): the row's
// maximum is the maximum of rounded products, and its own weight is exactly 2^40.
__device__ __forceinline__ float vf_exp(float logit, float inv_temp, float mx) {
  return expf(__fsub_rn(__fmul_rn(logit, inv_temp), mx));
}
__device__ __forceinline__ unsigned long long vf_weight(float logit, float inv_temp, float mx) {
  uint32_t hi, lo;
  vf_fix(vf_exp(logit, inv_temp, mx), hi, lo);
  return vf_join(hi, lo);
}

__device__ __forceinline__ unsigned long long vf_warp_sum(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// sum (or maximum) over the CTA, for every thread
template <bool kMax>
__device__ __forceinline__ unsigned long long vf_block(unsigned long long v, unsigned long long* sh) {
  v = kMax ? warp_max_u64(v) : vf_warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long w = (threadIdx.x & 31) < kVfThreads / 32 ? sh[threadIdx.x & 31] : 0ull;
  return kMax ? warp_max_u64(w) : vf_warp_sum(w);
}

template <typename E>
__global__ void __cluster_dims__(kVfCtas, 1, 1) __launch_bounds__(kVfThreads) k_verify_stats(VfArgs a) {
  __shared__ unsigned long long sh[32];
  __shared__ unsigned long long mine[2];
  pdl_wait();
  const uint32_t cta = vf_rank();
  const int row = blockIdx.x / kVfCtas, b = row / (a.T + 1), i = row % (a.T + 1), tid = threadIdx.x;
  const E* lg = (const E*)a.logits + (int64_t)row * a.row_stride;
  const VfVec<E> vec(lg, a.V);
  constexpr int N = VfVec<E>::N;
  const int per = (vec.count + kVfCtas - 1) / kVfCtas;
  const int j0 = min((int)cta * per, vec.count), j1 = min(j0 + per, vec.count);
  const bool greedy = a.inv_temp == 0.f;
  const float scale = greedy ? 1.f : a.inv_temp;

  unsigned long long key = 0;
  float top = -INFINITY;
  for (int j = j0 + tid; j < j1; j += kVfThreads) {
    float x[N];
    vec.load(j, x, -INFINITY);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (greedy) {
        if (x[e] > top) {  // ascending indexes within a thread: the first one stays
          top = x[e];
          key = argmax_key(x[e], (uint32_t)(vec.first(j) + e));
        }
      } else {
        top = fmaxf(top, __fmul_rn(x[e], scale));  // (ignores NaN)
      }
    }
  }
  if (!greedy) key = argmax_key(top, 0u);
  key = vf_block<true>(key, sh);
  if (tid == 0) mine[0] = key;
  vf_sync();
  for (int r = 0; r < kVfCtas; ++r) {
    const unsigned long long k = vf_peer(&mine[0], r);
    key = k > key ? k : key;
  }
  const uint32_t ord = (uint32_t)(key >> 32);
  const float mx = key == 0 ? -INFINITY : __uint_as_float((ord & 0x80000000u) ? (ord & 0x7fffffffu) : ~ord);
  VfRow out = {0ull, mx, -1, 0, 0};
  if (greedy) {
    if (key != 0) out.best = (int)argmax_key_index(key);
  } else if (fabsf(mx) < INFINITY) {
    uint32_t hi = 0, lo = 0;  // at most 2^20 / 4096 elements per thread: 2^28 each
    for (int j = j0 + tid; j < j1; j += kVfThreads) {
      float x[N];
      vec.load(j, x, -INFINITY);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        uint32_t h, l;
        vf_fix(vf_exp(x[e], scale, mx), h, l);
        hi += h;
        lo += l;
      }
    }
    const unsigned long long s = vf_block<false>(vf_join(hi, lo), sh);
    if (tid == 0) mine[1] = s;
  }
  if (tid == 0 && (greedy || !(fabsf(mx) < INFINITY))) mine[1] = 0;
  vf_sync();
  if (cta == 0 && tid == 0) {
    for (int r = 0; r < kVfCtas; ++r) out.sum += vf_peer(&mine[1], r);
    if (i < a.T) {
      const int n = a.n_draft ? min(max(a.n_draft[b], 0), a.T) : a.T;
      float prob = 0.f;
      if (i < n) {
        const int id = a.ids[(int64_t)b * a.T + i];
        if (id >= 0 && id < a.V) {
          if (greedy) {
            out.ok = id == out.best;
            prob = out.ok ? 1.f : 0.f;
          } else {
            const float p = out.sum ? __fdiv_rn((float)vf_weight((float)lg[id], scale, mx), (float)out.sum) : 0.f;
            const float q = a.probs ? a.probs[((int64_t)b * a.T + i) * a.V + id] : 1.f;
            out.ok = __fmul_rn(a.u[(int64_t)b * (a.T + 1) + i], q) < p;
            prob = q > 0.f ? fminf(__fdiv_rn(p, q), 1.f) : p > 0.f ? 1.f : 0.f;
          }
        }
      }
      a.accept_prob[(int64_t)b * a.T + i] = prob;
    }
    a.rows[row] = out;
  }
  vf_sync();  // no CTA leaves while its shared memory may be read
}

// floor(total u) with u taken to 24 bits; total < 2^63
__device__ __forceinline__ unsigned long long vf_threshold(unsigned long long total, float u) {
  float t = u * 16777216.f;
  t = t > 0.f ? fminf(t, 16777215.f) : 0.f;
  const unsigned long long f = (unsigned long long)t;
  return (total >> 32) * f * 256ull + (((total & 0xffffffffull) * f) >> 24);
}

template <typename E>
__global__ void __cluster_dims__(kVfCtas, 1, 1) __launch_bounds__(kVfThreads) k_verify_draw(VfArgs a) {
  __shared__ unsigned long long sh[32];
  __shared__ unsigned long long mine[2];
  __shared__ int found;
  pdl_wait();
  const uint32_t cta = vf_rank();
  const int b = blockIdx.x / kVfCtas, tid = threadIdx.x, lane = tid & 31;
  const int T = a.T;
  const int nd = a.n_draft ? min(max(a.n_draft[b], 0), T) : T;
  const VfRow* rows = a.rows + (int64_t)b * (T + 1);
  const uint32_t no = __ballot_sync(0xffffffffu, lane >= nd || !rows[min(lane, T)].ok);
  const int n = __ffs((int)no) - 1;  // nd <= 31, so a bit is set
  const VfRow row = rows[n];
  const bool greedy = a.inv_temp == 0.f;
  int extra = greedy ? row.best : -1;

  if (!greedy && row.sum != 0) {
    const E* lg = (const E*)a.logits + ((int64_t)b * (T + 1) + n) * a.row_stride;
    const VfVec<E> vec(lg, a.V);
    constexpr int N = VfVec<E>::N;
    const int per = (vec.count + kVfCtas - 1) / kVfCtas;
    const int j0 = min((int)cta * per, vec.count), j1 = min(j0 + per, vec.count);
    const bool refused = n < nd;
    const int id = refused ? a.ids[(int64_t)b * T + n] : -1;
    const float* q = refused && a.probs ? a.probs + ((int64_t)b * T + n) * a.V : nullptr;
    const float z = (float)row.sum;
    bool residual = refused;
    auto weights = [&](int j, unsigned long long (&w)[N]) {
      float x[N];
      vec.load(j, x, -INFINITY);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int v = vec.first(j) + e;
        w[e] = vf_weight(x[e], a.inv_temp, row.max);
        if (residual) {
          if (!q) {
            if (v == id) w[e] = 0;
          } else if (v >= 0 && v < a.V) {
            const float p = __fdiv_rn((float)w[e], z), d = q[v];
            uint32_t hi, lo;
            vf_fix(p > d ? p - d : 0.f, hi, lo);
            w[e] = vf_join(hi, lo);
          }
        }
      }
    };
    unsigned long long total, before;
    for (int pass = 0;; ++pass) {
      unsigned long long s = 0;
      for (int j = j0 + tid; j < j1; j += kVfThreads) {
        unsigned long long w[N];
        weights(j, w);
#pragma unroll
        for (int e = 0; e < N; ++e) s += w[e];
      }
      s = vf_block<false>(s, sh);
      if (tid == 0) mine[pass] = s;
      vf_sync();
      total = before = 0;
      for (int r = 0; r < kVfCtas; ++r) {
        const unsigned long long x = vf_peer(&mine[pass], r);
        if (r < (int)cta) before += x;
        total += x;
      }
      if (total != 0 || !residual) break;
      residual = false;  // p nowhere above q (rounding): the target's own distribution
    }
    const unsigned long long k = vf_threshold(total, a.u[(int64_t)b * (T + 1) + T]);
    // the CTA whose slice holds the running sum's crossing looks for it, 512 vectors at a time
    if (tid == 0) found = -1;
    __syncthreads();
    if (k >= before) {
      unsigned long long run = before;
      for (int js = j0; js < j1; js += kVfThreads) {
        const int j = js + tid;
        unsigned long long w[N], s = 0;
        if (j < j1) {
          weights(j, w);
#pragma unroll
          for (int e = 0; e < N; ++e) s += w[e];
        }
        // inclusive scan over the CTA
        unsigned long long x = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) sh[tid >> 5] = x;
        __syncthreads();
        unsigned long long low = run, all = run;
        for (int r = 0; r < kVfThreads / 32; ++r) {
          if (r < (tid >> 5)) low += sh[r];
          all += sh[r];
        }
        const unsigned long long hi_ = low + x, lo_ = hi_ - s;
        if (j < j1 && lo_ <= k && k < hi_) {
          unsigned long long c = lo_;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            if (c <= k && k < c + w[e]) found = vec.first(j) + e;
            c += w[e];
          }
        }
        if (all > k) break;
        run = all;
      }
    }
    __syncthreads();
    extra = found;
    vf_sync();  // peers have read this CTA's sums
    if (extra < 0) return;  // another CTA has the token
  } else if (cta != 0) {
    return;
  }
  if (tid <= T) {
    int t = -1;
    if (tid < n) t = a.ids[(int64_t)b * T + tid];
    if (tid == n) t = extra;
    a.tokens[(int64_t)b * (T + 1) + tid] = t;
  }
  if (tid == 0) a.accepted[b] = n;
}

template <typename E>
static int verify_launch(const VfArgs& a, int B, cudaStream_t s) {
  JSX_CUDA(launch_kernel(k_verify_stats<E>, dim3((unsigned)(B * (a.T + 1) * kVfCtas)), dim3(kVfThreads), 0, s, a));
  JSX_CUDA(launch_kernel(k_verify_draw<E>, dim3((unsigned)(B * kVfCtas)), dim3(kVfThreads), 0, s, a));
  return JSX_OK;
}

}  // namespace jsx

using namespace jsx;

extern "C" int jsx_verify_workspace_size(int B, int T, int V, size_t* bytes) {
  JSX_REQUIRE(bytes && B >= 1 && T >= 0 && T <= kVfMaxDraft && V >= 1 && V <= kVfMaxVocab, "bad arguments");
  *bytes = (size_t)B * (T + 1) * sizeof(VfRow);
  return JSX_OK;
}

extern "C" int jsx_verify_drafts(const void* logits, int logits_f32, int64_t row_stride, const int32_t* draft_ids,
                                 const float* draft_probs, const int32_t* n_draft, const float* uniforms,
                                 float temperature, int32_t* accepted, int32_t* tokens, float* accept_prob, int B,
                                 int T, int V, void* workspace, size_t workspace_bytes, void* stream) {
  JSX_REQUIRE(B >= 1 && B <= (1 << 20) && T >= 0 && T <= kVfMaxDraft, "B=%d T=%d (T in 0..%d)", B, T, kVfMaxDraft);
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
