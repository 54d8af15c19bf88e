// Attention over the 4-bit key/value pages (kv4.cuh), causal, with an optional
// sliding window and first tokens that stay visible.
//
// Row (b, i) of T tokens per sequence is at position p = positions[b] + i and sees
// cache row j when j <= p, (no window or j > p - window or j < sinks) and j's page is
// present; o = sum_j softmax_j(scale q . k_j) v_j, and 0 when it sees nothing.
//
// One CTA of 128 threads per query row and head: a thread scores one key of each
// block of 128, then accumulates one output dimension over the block (online
// softmax, fp32).
#include <math.h>

#include "common.cuh"
#include "kv4.cuh"
#include "launch.cuh"

namespace jsx {

struct KaArgs {
  const bf16* q;
  bf16* out;
  int64_t q_stride, out_stride;  // per token, elements
  const uint8_t* pool;
  const int32_t* table;
  const int32_t* positions;
  const int32_t* n_tokens;
  int num_pages, slots, B, T, nq, nkv, pt, window, sinks;
  float scale;
};

template <int D>
__device__ __forceinline__ float ka_value(const uint8_t* block, int pt, int t, int d, bool v) {
  uint32_t h[4];
  e2m1x8_to_h2(*reinterpret_cast<const uint32_t*>(block + (v ? kv4_off_v(pt, D) : 0) + t * (D / 2) + d / 8 * 4), h);
  const uint32_t sc = block[(v ? kv4_off_vs(pt, D) : kv4_off_ks(pt, D)) + t * (D / 16) + d / 16];
  const uint32_t y = hmul2_u(d & 4 ? (d & 2 ? h[3] : h[2]) : (d & 2 ? h[1] : h[0]), e4m3x2_to_h2(sc | (sc << 8)));
  const __half2 x = *reinterpret_cast<const __half2*>(&y);
  return d & 1 ? __high2float(x) : __low2float(x);
}

template <int D>
__global__ void __launch_bounds__(128) k_kv4_attn(KaArgs a) {
  __shared__ float qs[D], ps[128], red[4];
  __shared__ const uint8_t* blocks[128];
  pdl_wait();
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int b = row / a.T, i = row % a.T, kvh = h / (a.nq / a.nkv);
  const int pos = a.positions[b] + i;
  const bool used = !a.n_tokens || i < a.n_tokens[b];
  if (tid < D) qs[tid] = __bfloat162float(a.q[row * a.q_stride + h * D + tid]);
  const int first = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int j0 = 0; used && j0 <= pos; j0 += 128) {
    if (j0 >= a.sinks && j0 + 127 < first) continue;
    __syncthreads();
    const int j = j0 + tid, slot = j / a.pt;
    const uint8_t* block = nullptr;
    if (j <= pos && (j >= first || j < a.sinks) && slot < a.slots) {
      const int page = a.table[(int64_t)b * a.slots + slot];
      if (page >= 0 && page < a.num_pages)
        block = a.pool + ((int64_t)page * a.nkv + kvh) * kv4_block_bytes(a.pt, D);
    }
    float s = -INFINITY;
    if (block) {
      s = 0.f;
      for (int d = 0; d < D; ++d) s += qs[d] * ka_value<D>(block, a.pt, j % a.pt, d, false);
      s *= a.scale;
    }
    blocks[tid] = block;
    float mx = warp_max(s);
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    if (mx == -INFINITY && __syncthreads_or(s != s) == 0) continue;
    const float mn = fmaxf(m, mx);
    const float f = m == -INFINITY ? 0.f : expf(m - mn);
    const float p = block ? expf(s - mn) : 0.f;
    ps[tid] = p;
    const float sum = warp_sum(p);
    if ((tid & 31) == 0) red[tid >> 5] = sum;
    __syncthreads();
    l = l * f + red[0] + red[1] + red[2] + red[3];
    m = mn;
    o *= f;
    if (tid < D)
      for (int k = 0; k < 128; ++k)
        if (blocks[k]) o += ps[k] * ka_value<D>(blocks[k], a.pt, (j0 + k) % a.pt, tid, true);
  }
  if (tid < D) a.out[row * a.out_stride + h * D + tid] = __float2bfloat16_rn(l == 0.f ? 0.f : o / l);
}

}  // namespace jsx

using namespace jsx;

extern "C" int jsx_kv4_attn_workspace_size(int B, int T, int nq, int nkv, int head_dim, size_t* bytes) {
  JSX_REQUIRE(bytes && B >= 1 && T >= 1 && nq >= 1 && nkv >= 1 && nq % nkv == 0, "bad arguments");
  *bytes = 256;
  return JSX_OK;
}

extern "C" int jsx_kv4_attn(const void* q, int64_t q_stride, const void* pool, int num_pages, const int32_t* table,
                            int table_slots, const int32_t* positions, const int32_t* n_tokens, void* out,
                            int64_t out_stride, int B, int T, int nq, int nkv, int head_dim, int page_tokens,
                            int window, int sinks, float scale, void* workspace, size_t workspace_bytes,
                            void* stream) {
  JSX_REQUIRE(q && out && positions, "null pointer argument");
  JSX_KV4_REQUIRE(pool, num_pages, table, table_slots, nkv, head_dim, page_tokens);
  JSX_REQUIRE(B >= 1 && T >= 1 && (int64_t)B * T <= INT32_MAX, "B=%d T=%d", B, T);
  JSX_REQUIRE(nq >= 1 && nq % nkv == 0, "nq=%d is not a multiple of nkv=%d", nq, nkv);
  JSX_REQUIRE(aligned16(q) && aligned16(out) && q_stride % 8 == 0 && out_stride % 8 == 0 &&
                  q_stride >= (int64_t)nq * head_dim && out_stride >= (int64_t)nq * head_dim,
              "q and out must be 16-byte aligned, with token strides of at least nq * head_dim in multiples of 8");
  JSX_REQUIRE(window >= 0 && sinks >= 0, "window=%d sinks=%d", window, sinks);
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
  a.num_pages = num_pages;
  a.slots = table_slots;
  a.B = B;
  a.T = T;
  a.nq = nq;
  a.nkv = nkv;
  a.pt = page_tokens;
  a.window = window;
  a.sinks = sinks;
  a.scale = scale;
  auto kern = head_dim == 128 ? k_kv4_attn<128> : k_kv4_attn<64>;
  JSX_CUDA(launch_kernel(kern, dim3(B * T, nq), dim3(128), 0, (cudaStream_t)stream, a));
  return JSX_OK;
}
