// Verification of drafted tokens against the model's own distribution, from random numbers that the caller drew (speculative sampling:
// the tokens that come out are distributed as if the model had been sampled token by token).  For sequence b with n drafts x_0 .. x_{n-1}:
//   p_t = softmax(logits[b][t] / temperature);  x_t stands while  u_t q_t(x_t) < p_t(x_t)   (q_t: the draft's own probabilities, or 1 at x_t)
//   at the first refusal a the next token is drawn from r = max(p_a - q_a, 0), without a refusal from r = p_n:
//   the lowest v with r(v) > 0 and  sum_{w <= v} r(w) > u_last * sum r.     temperature 0: x_t stands while it is the argmax (lowest index).
// What comes out are whole numbers decided by comparisons, so the weights exp((x - max) / temperature) and their sums are held in 64 bits: over
// 150 000 tokens the running sum in 32 bits would pick a neighbour in about one draw of fifty.  The bytes are those of the logits.
//   verify_stats_kernel   (chunk, row, sequence): max, sum of weights, argmax of a chunk of kChunk logits
//   verify_rest_kernel    (chunk, sequence), only with draft probabilities: sum of the refused row's max(p - q, 0)
//   verify_pick_kernel    (sequence): which drafts stand, the chunk the draw falls into, the token in it
// No atomics: the same call gives the same result.
#include "qp_common.h"

namespace {

constexpr int kChunk = 4096, kThreads = 256, kPer = kChunk / kThreads;
constexpr int kMaxDrafts = 255, kMaxChunks = 1024;

struct VerifyParams {
  const void* logits; int64_t seq_stride, row_stride;          // elements
  const int64_t* drafts; const int* n_draft;
  const float* probs; int64_t probs_seq_stride, probs_row_stride;
  const float* u;
  int batch, T, nc; int64_t V;
  double inv_temp;
  double* sum; double* rest; float* top; int* arg;             // [batch][T + 1][nc] (rest: [batch][nc])
  int* accepted; int64_t* tokens;
};

__device__ __forceinline__ int drafts_of(const VerifyParams& p, int b) {      // -1: an idle place of the batch
  if (!p.n_draft) return p.T;
  const int n = p.n_draft[b];
  return n < 0 ? -1 : (n > p.T ? p.T : n);
}
template <bool kF32>
__device__ __forceinline__ float logit(const VerifyParams& p, int64_t row, int64_t v) {          // NaN is never chosen: like -infinity
  const float x = kF32 ? ((const float*)p.logits)[row + v] : bf16_bits_to_f32(((const uint16_t*)p.logits)[row + v]);
  return x == x ? x : -INFINITY;
}
__device__ __forceinline__ double weight(float x, float top, double inv_temp) {
  return x == top ? 1.0 : exp(((double)x - (double)top) * inv_temp);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ __forceinline__ double block_sum_f64(double v, double* red) {       // red: 4 doubles; all threads get the sum
  v = wave_sum_f64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <bool kF32>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyParams p) {
  __shared__ double red[4];
  __shared__ float red_m[4];
  __shared__ int red_i[4];
  const int ch = blockIdx.x, t = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  if (t > drafts_of(p, b)) return;
  const int64_t row = (int64_t)b * p.seq_stride + (int64_t)t * p.row_stride, v0 = (int64_t)ch * kChunk;
  float x[kPer], m = -INFINITY;
  int arg = INT32_MAX;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t v = v0 + tid + i * kThreads;
    x[i] = v < p.V ? logit<kF32>(p, row, v) : -INFINITY;
    if (x[i] > m) { m = x[i]; arg = (int)v; }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const float om = __shfl_xor(m, d, 64);
    const int oa = __shfl_xor(arg, d, 64);
    if (om > m || (om == m && oa < arg)) { m = om; arg = oa; }
  }
  if ((tid & 63) == 0) { red_m[tid >> 6] = m; red_i[tid >> 6] = arg; }
  __syncthreads();
  m = red_m[0]; arg = red_i[0];
#pragma unroll
  for (int w = 1; w < 4; ++w)
    if (red_m[w] > m || (red_m[w] == m && red_i[w] < arg)) { m = red_m[w]; arg = red_i[w]; }
  double s = 0.0;
  if (p.inv_temp != 0.0 && m != -INFINITY) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (x[i] != -INFINITY) s += weight(x[i], m, p.inv_temp);
  }
  s = block_sum_f64(s, red);
  if (tid == 0) {
    const int64_t at = ((int64_t)b * (p.T + 1) + t) * p.nc + ch;
    p.sum[at] = s; p.top[at] = m; p.arg[at] = arg;
  }
}

// Which drafts stand: every workgroup that asks finds it again from the chunks' statistics (a few KB) instead of waiting for another launch.
struct Decision { int n, a; float top; double z; int arg; };   // row a: the refused one, or n; its maximum, sum of weights, argmax

template <bool kF32>
__device__ Decision decide(const VerifyParams& p, int b, int n) {
  __shared__ int ok[kMaxDrafts + 1];
  __shared__ float tops[kMaxDrafts + 1];
  __shared__ double zs[kMaxDrafts + 1];
  __shared__ int args[kMaxDrafts + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int t = wave; t <= n; t += kThreads / 64) {
    const int64_t at = ((int64_t)b * (p.T + 1) + t) * p.nc;
    float m = -INFINITY;
    int arg = INT32_MAX;
    for (int c = lane; c < p.nc; c += 64) {
      const float cm = p.top[at + c];
      const int ca = p.arg[at + c];
      if (cm > m || (cm == m && ca < arg)) { m = cm; arg = ca; }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const float om = __shfl_xor(m, d, 64);
      const int oa = __shfl_xor(arg, d, 64);
      if (om > m || (om == m && oa < arg)) { m = om; arg = oa; }
    }
    double z = 0.0;
    if (p.inv_temp != 0.0)
      for (int c = lane; c < p.nc; c += 64) {
        const float cm = p.top[at + c];
        if (cm != -INFINITY) z += p.sum[at + c] * weight(cm, m, p.inv_temp);
      }
    z = wave_sum_f64(z);
    if (lane == 0) {
      bool stands = false;
      if (t < n && m != -INFINITY) {
        const int64_t x = p.drafts[(int64_t)b * p.T + t];
        if (x >= 0 && x < p.V) {
          if (p.inv_temp == 0.0) {
            stands = x == arg;
          } else {
            const float lx = logit<kF32>(p, (int64_t)b * p.seq_stride + (int64_t)t * p.row_stride, x);
            const double px = lx == -INFINITY ? 0.0 : weight(lx, m, p.inv_temp);
            const double q = p.probs ? (double)p.probs[(int64_t)b * p.probs_seq_stride + (int64_t)t * p.probs_row_stride + x] : 1.0;
            stands = (double)p.u[(int64_t)b * (p.T + 1) + t] * q * z < px;
          }
        }
      }
      ok[t] = stands; tops[t] = m; zs[t] = z; args[t] = arg;
    }
  }
  __syncthreads();
  Decision d;
  d.n = n; d.a = 0;
  while (d.a < n && ok[d.a]) ++d.a;
  d.top = tops[d.a]; d.z = zs[d.a]; d.arg = args[d.a];
  return d;
}

enum { FROM_ROW = 0, WITHOUT_DRAFT = 1, LESS_DRAFT = 2 };      // what the next token is drawn from: p, p without x, max(p - q, 0)

// weight of token v in the draw, in units of the row's exp((x - max) / temperature)
template <bool kF32>
__device__ __forceinline__ double draw_weight(const VerifyParams& p, int64_t row, int64_t q_row, int64_t v, int kind, int64_t x, const Decision& d) {
  if (v >= p.V || (kind == WITHOUT_DRAFT && v == x)) return 0.0;
  const float l = logit<kF32>(p, row, v);
  double w = l == -INFINITY ? 0.0 : weight(l, d.top, p.inv_temp);
  if (kind == LESS_DRAFT) w = fmax(w - (double)p.probs[q_row + v] * d.z, 0.0);
  return w;
}

template <bool kF32>
__global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyParams p) {
  __shared__ double red[4];
  const int ch = blockIdx.x, b = blockIdx.y, n = drafts_of(p, b);
  if (n < 0) return;
  const Decision d = decide<kF32>(p, b, n);
  if (d.a == n || d.top == -INFINITY) return;
  const int64_t row = (int64_t)b * p.seq_stride + (int64_t)d.a * p.row_stride, q_row = (int64_t)b * p.probs_seq_stride + (int64_t)d.a * p.probs_row_stride;
  double s = 0.0;
  for (int i = 0; i < kPer; ++i) s += draw_weight<kF32>(p, row, q_row, (int64_t)ch * kChunk + threadIdx.x + i * kThreads, LESS_DRAFT, -1, d);
  s = block_sum_f64(s, red);
  if (threadIdx.x == 0) p.rest[(int64_t)b * p.nc + ch] = s;
}

template <bool kF32>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyParams p) {
  __shared__ double red[4], share[kMaxChunks], before[kThreads];
  __shared__ int found[2];
  const int b = blockIdx.x, tid = threadIdx.x, n = drafts_of(p, b);
  int64_t* out = p.tokens + (int64_t)b * (p.T + 1);
  if (n < 0) {
    for (int t = tid; t <= p.T; t += kThreads) out[t] = -1;
    if (tid == 0) p.accepted[b] = 0;
    return;
  }
  const Decision d = decide<kF32>(p, b, n);
  for (int t = tid; t <= p.T; t += kThreads)
    if (t != d.a) out[t] = t < d.a ? p.drafts[(int64_t)b * p.T + t] : -1;
  if (tid == 0) p.accepted[b] = d.a;
  if (d.top == -INFINITY || p.inv_temp == 0.0) {               // greedy, or a row that offers nothing
    if (tid == 0) out[d.a] = d.top == -INFINITY ? -1 : d.arg;
    return;
  }
  const int64_t row = (int64_t)b * p.seq_stride + (int64_t)d.a * p.row_stride, q_row = (int64_t)b * p.probs_seq_stride + (int64_t)d.a * p.probs_row_stride;
  const int64_t at = ((int64_t)b * (p.T + 1) + d.a) * p.nc;
  int kind = d.a == n ? FROM_ROW : (p.probs ? LESS_DRAFT : WITHOUT_DRAFT);
  int64_t x = -1;
  if (kind == WITHOUT_DRAFT) x = p.drafts[(int64_t)b * p.T + d.a];
  double total = 0.0;
  for (;;) {                                                   // twice at most: nothing left of p - q (they are equal) -> p itself
    double mine = 0.0;
    for (int c = tid; c < p.nc; c += kThreads) {
      double w;
      if (kind == LESS_DRAFT) w = p.rest[(int64_t)b * p.nc + c];
      else { const float cm = p.top[at + c]; w = cm == -INFINITY ? 0.0 : p.sum[at + c] * weight(cm, d.top, p.inv_temp); }
      share[c] = w;
    }
    __syncthreads();
    if (kind == WITHOUT_DRAFT && x >= 0 && x < p.V) {          // summed again without x: its share may be nearly all there is
      const int64_t c = x / kChunk;
      double s = 0.0;
      for (int i = 0; i < kPer; ++i) s += draw_weight<kF32>(p, row, q_row, c * kChunk + tid + i * kThreads, kind, x, d);
      s = block_sum_f64(s, red);
      if (tid == 0) share[c] = s;
      __syncthreads();
    }
    for (int c = tid; c < p.nc; c += kThreads) mine += share[c];
    total = block_sum_f64(mine, red);
    if (total > 0.0 || kind == FROM_ROW) break;
    kind = FROM_ROW;
    __syncthreads();
  }
  const double want = (double)p.u[(int64_t)b * (p.T + 1) + p.T] * total;
  if (tid == 0) {
    double run = 0.0, base = 0.0;
    int hit = -1, last = 0;
    double last_base = 0.0;
    for (int c = 0; c < p.nc; ++c) {
      const double w = share[c];
      if (!(w > 0.0)) continue;
      last = c; last_base = run;
      if (run + w > want) { hit = c; base = run; break; }
      run += w;
    }
    found[0] = hit >= 0 ? hit : last;
    before[0] = hit >= 0 ? base : last_base;
  }
  __syncthreads();
  const int c = found[0];
  const double base = before[0];
  __syncthreads();
  double w[kPer], sum = 0.0;
  const int64_t v0 = (int64_t)c * kChunk + (int64_t)tid * kPer;
#pragma unroll
  for (int i = 0; i < kPer; ++i) { w[i] = draw_weight<kF32>(p, row, q_row, v0 + i, kind, x, d); sum += w[i]; }
  double incl = sum;                                           // running sum over the workgroup's threads
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const double o = __shfl_up(incl, s, 64);
    if ((tid & 63) >= s) incl += o;
  }
  if ((tid & 63) == 63) red[tid >> 6] = incl;
  if (tid < 2) found[tid] = tid == 0 ? INT32_MAX : -1;
  __syncthreads();
  double run = base + (incl - sum);
  for (int k = 0; k < (tid >> 6); ++k) run += red[k];
  int first = INT32_MAX, last = -1;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    run += w[i];
    if (w[i] > 0.0) {
      last = (int)(v0 + i);
      if (first == INT32_MAX && run > want) first = last;
    }
  }
  if (first != INT32_MAX) atomicMin(&found[0], first);
  if (last >= 0) atomicMax(&found[1], last);
  __syncthreads();
  if (tid == 0) out[d.a] = found[0] != INT32_MAX ? found[0] : found[1];
}

template <bool kF32>
int launch(const VerifyParams& p, hipStream_t s) {
  verify_stats_kernel<kF32><<<dim3((unsigned)p.nc, (unsigned)(p.T + 1), (unsigned)p.batch), kThreads, 0, s>>>(p);
  int rc = qp_check_launch("verify_drafts(stats)");
  if (rc) return rc;
  if (p.probs && p.inv_temp != 0.0) {
    verify_rest_kernel<kF32><<<dim3((unsigned)p.nc, (unsigned)p.batch), kThreads, 0, s>>>(p);
    if ((rc = qp_check_launch("verify_drafts(rest)"))) return rc;
  }
  verify_pick_kernel<kF32><<<(unsigned)p.batch, kThreads, 0, s>>>(p);
  return qp_check_launch("verify_drafts(pick)");
}

}  // namespace

int64_t qp_verify_max_vocab() { return (int64_t)kChunk * kMaxChunks; }
int qp_verify_max_drafts() { return kMaxDrafts; }

size_t qp_verify_workspace_bytes_impl(int batch, int t_max, int64_t vocab) {
  const size_t nc = (size_t)((vocab + kChunk - 1) / kChunk), rows = (size_t)batch * (t_max + 1);
  return rows * nc * (sizeof(double) + sizeof(float) + sizeof(int)) + (size_t)batch * nc * sizeof(double);
}

int qp_launch_verify_drafts(const void* logits, int logits_f32, int64_t seq_stride, int64_t row_stride, const int64_t* drafts, const int32_t* n_draft,
                            const float* probs, int64_t probs_seq_stride, int64_t probs_row_stride, const float* uniforms, int batch, int t_max,
                            int64_t vocab, float temperature, int32_t* n_accepted, int64_t* tokens, void* workspace, hipStream_t s) {
  VerifyParams p;
  p.logits = logits; p.seq_stride = seq_stride; p.row_stride = row_stride;
  p.drafts = drafts; p.n_draft = n_draft;
  p.probs = t_max > 0 ? probs : nullptr; p.probs_seq_stride = probs_seq_stride; p.probs_row_stride = probs_row_stride;
  p.u = uniforms; p.batch = batch; p.T = t_max; p.V = vocab;
  p.nc = (int)((vocab + kChunk - 1) / kChunk);
  p.inv_temp = temperature > 0.f ? 1.0 / (double)temperature : 0.0;
  const size_t rows = (size_t)batch * (t_max + 1) * p.nc;
  p.sum = (double*)workspace;
  p.rest = p.sum + rows;
  p.top = (float*)(p.rest + (size_t)batch * p.nc);
  p.arg = (int*)(p.top + rows);
  p.accepted = n_accepted; p.tokens = tokens;
  return logits_f32 ? launch<true>(p, s) : launch<false>(p, s);
}
