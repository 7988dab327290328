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
  double scale;                                                // log2(e) / temperature; 0: greedy
  double *sum, *rest, *others; float* top; int* arg;           // [batch][T + 1][nc] (rest: [batch][nc], others: [batch][T])
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
// 2^y, y <= 0, in 64 bits: y = k + f with |f| <= 1/2 (k by adding 1.5 * 2^52, whose last bits then are k), the series of 2^f = e^(f ln 2) up to
// f^11 (what is left out is (ln 2 / 2)^12 / 12! < 7e-15), k added to the exponent.  16 operations at the full rate of 64-bit arithmetic, where the
// library's exp takes twice the time with its special cases; 0 below 2^-1020.
__device__ __forceinline__ double exp2_neg(double y) {
  constexpr double L = 0.693147180559945309417;                // ln 2
  constexpr double c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6, c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9,
                   c10 = c9 * L / 10, c11 = c10 * L / 11;
  constexpr double shift = 6755399441055744.0;                 // 1.5 * 2^52
  const double in = fmax(y, -1021.0), t = in + shift, f = in - (t - shift);
  double r = fma(c11, f, c10);
  r = fma(r, f, c9); r = fma(r, f, c8); r = fma(r, f, c7); r = fma(r, f, c6); r = fma(r, f, c5); r = fma(r, f, c4); r = fma(r, f, c3); r = fma(r, f, c2);
  r = fma(r, f, L); r = fma(r, f, 1.0);
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, r) + (__builtin_bit_cast(unsigned long long, t) << 52);
  return y < -1020.0 ? 0.0 : __builtin_bit_cast(double, bits);
}
// weight of a logit against the row's maximum (above -infinity): 1 at the maximum, also an infinite one; 0 for -infinity
__device__ __forceinline__ double weight(float x, float top, double scale) {
  return exp2_neg(x == top ? 0.0 : ((double)x - (double)top) * scale);
}
template <int kStep = 0>
__device__ __forceinline__ double wave_sum_f64(double v) {     // the same bits in every lane
  if constexpr (kStep < 6) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    unsigned lo, hi;
    const unsigned olo = swap_lanes<kStep>((unsigned)b, lo), ohi = swap_lanes<kStep>((unsigned)(b >> 32), hi);
    return wave_sum_f64<kStep + 1>(__builtin_bit_cast(double, (unsigned long long)hi << 32 | lo) + __builtin_bit_cast(double, (unsigned long long)ohi << 32 | olo));
  } else {
    return v;
  }
}
// the largest value and, where several lanes hold it, the lowest number (kArg)
template <bool kArg, int kStep = 0>
__device__ __forceinline__ void wave_max(float& m, int& arg) {
  if constexpr (kStep < 6) {
    unsigned am, aa = 0, om, oa = 0;
    om = swap_lanes<kStep>(__builtin_bit_cast(unsigned, m), am);
    if (kArg) oa = swap_lanes<kStep>((unsigned)arg, aa);
    const float a = __builtin_bit_cast(float, am), b = __builtin_bit_cast(float, om);
    if (kArg) arg = b > a || (b == a && (int)oa < (int)aa) ? (int)oa : (int)aa;
    m = fmaxf(a, b);
    wave_max<kArg, kStep + 1>(m, arg);
  }
}
// sum of this lane's and all lower lanes'
template <int kCtrl, int kRows>
__device__ __forceinline__ double from_below(double v) {       // 0 where nothing is below
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, kCtrl, kRows, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), kCtrl, kRows, 0xf, false);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan_f64(double v) {
  v += from_below<0x111, 0xf>(v);                              // row_shr 1, 2, 4, 8
  v += from_below<0x112, 0xf>(v);
  v += from_below<0x114, 0xf>(v);
  v += from_below<0x118, 0xf>(v);
  v += from_below<0x142, 0xa>(v);                              // the last lane of rows 0 and 2 to rows 1 and 3
  v += from_below<0x143, 0xc>(v);                              // lane 31 to the upper half
  return v;
}
__device__ __forceinline__ double lane_f64(double v, int lane) {               // (lane: the same for all)
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)b, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(b >> 32), lane);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
template <int kWaves>
__device__ __forceinline__ double block_sum_f64(double v, double* red) {       // red: a double per wave; all threads get the sum
  v = wave_sum_f64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s += red[w];
  return s;
}

// 16 logits of a chunk per thread: 16 B a load where the row lies on a 16-B boundary, one by one where it does not or ends.  place(i) = the i-th one's token
template <bool kF32>
struct Chunk {
  static constexpr int W = kF32 ? 4 : 8;                       // logits in 16 B
  float x[kPer];
  bool wide;
  __device__ __forceinline__ int place(int i) const { return wide ? ((i / W) * kThreads + (int)threadIdx.x) * W + i % W : i * kThreads + (int)threadIdx.x; }
  __device__ __forceinline__ void load(const VerifyParams& p, int64_t row, int64_t v0) {
    const char* at = (const char*)p.logits + (row + v0) * (kF32 ? 4 : 2);
    wide = ((uintptr_t)at & 15) == 0;
    if (wide && v0 + kChunk <= p.V) {
#pragma unroll
      for (int j = 0; j < kPer / W; ++j) {
        const uint4 u = reinterpret_cast<const uint4*>(at)[j * kThreads + threadIdx.x];
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (kF32) x[j * W + e] = __uint_as_float(w[e]);
          else { x[j * W + 2 * e] = __uint_as_float(w[e] << 16); x[j * W + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
        }
      }
    } else {
      wide = false;
#pragma unroll
      for (int i = 0; i < kPer; ++i) { const int64_t v = v0 + place(i); x[i] = v < p.V ? logit<kF32>(p, row, v) : -INFINITY; }
    }
  }
};

// What bounds it in a large batch is about half the logits' bytes and half the 64-bit exponentials: 32 x 5 rows of 152064 fp32 logits take 21 us (23 in the
// first calls, before the clocks have risen; 14 then with the 32-bit exponential instead).  More or fewer workgroups on a CU, or several chunks per workgroup with the next one's loads ahead, gained nothing.
// A small call is a chain of latencies: maxima and sums per wave, which meet once, instead of a maximum of the whole chunk first (4 rows: 7.2 -> 5.3 us).
template <bool kF32>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyParams p) {
  __shared__ double red[4], red_o[4];
  __shared__ float red_m[4];
  __shared__ int red_i[4];
  const int ch = blockIdx.x, t = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, wave = tid >> 6;
  if (t > drafts_of(p, b)) return;
  const int64_t row = (int64_t)b * p.seq_stride + (int64_t)t * p.row_stride, v0 = (int64_t)ch * kChunk;
  // a certain draft: the sum without it as well, which may be next to nothing of the whole
  const bool certain = p.scale != 0.0 && !p.probs && t < p.T;
  const int64_t draft = certain ? p.drafts[(int64_t)b * p.T + t] : -1;
  Chunk<kF32> c;
  c.load(p, row, v0);
  float m = -INFINITY;
  int arg = INT32_MAX;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {                             // (a thread's places ascend; NaN is never chosen)
    if (!(c.x[i] == c.x[i])) c.x[i] = -INFINITY;
    if (c.x[i] > m) { m = c.x[i]; arg = (int)v0 + c.place(i); }
  }
  // Every wave against its own maximum; they meet once, at the end.
  double s = 0.0, o = 0.0;
  if (p.scale == 0.0) {
    wave_max<true>(m, arg);
  } else {
    wave_max<false>(m, arg);
    if (m != -INFINITY) {
      bool holds = false;
#pragma unroll
      for (int i = 0; i < kPer; ++i) s += weight(c.x[i], m, p.scale);
      o = s;
      if (draft >= v0 && draft < v0 + kChunk) {                // (uniform)
#pragma unroll
        for (int i = 0; i < kPer; ++i) holds |= v0 + c.place(i) == draft;
        if (holds) {                                           // one thread sums again
          o = 0.0;
#pragma unroll
          for (int i = 0; i < kPer; ++i) o += v0 + c.place(i) == draft ? 0.0 : weight(c.x[i], m, p.scale);
        }
        o = wave_sum_f64(o);
      }
      s = wave_sum_f64(s);
    }
  }
  if ((tid & 63) == 0) { red_m[wave] = m; red_i[wave] = arg; red[wave] = s; red_o[wave] = o; }
  __syncthreads();
  if (tid != 0) return;
  m = red_m[0]; arg = red_i[0];
#pragma unroll
  for (int w = 1; w < 4; ++w)
    if (red_m[w] > m || (red_m[w] == m && red_i[w] < arg)) { m = red_m[w]; arg = red_i[w]; }
  s = o = 0.0;
  if (p.scale != 0.0 && m != -INFINITY) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const double f = weight(red_m[w], m, p.scale);
      s += red[w] * f; o += red_o[w] * f;
    }
  }
  if (draft >= v0 && draft < v0 + kChunk) p.others[(int64_t)b * p.T + t] = o;              // (0 of a chunk that offers nothing)
  const int64_t at = ((int64_t)b * (p.T + 1) + t) * p.nc + ch;
  p.sum[at] = s; p.top[at] = m; p.arg[at] = arg;
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
  for (int t = wave; t <= n; t += (int)blockDim.x / 64) {
    const int64_t at = ((int64_t)b * (p.T + 1) + t) * p.nc;
    // the draft's own numbers are on their way while the chunks are joined
    const int64_t x = t < n ? p.drafts[(int64_t)b * p.T + t] : -1;
    const bool inside = x >= 0 && x < p.V;
    float lx = -INFINITY, qx = 1.f, u = 0.f;
    if (inside && p.scale != 0.0) {
      u = p.u[(int64_t)b * (p.T + 1) + t];
      lx = logit<kF32>(p, (int64_t)b * p.seq_stride + (int64_t)t * p.row_stride, x);
      if (p.probs) qx = p.probs[(int64_t)b * p.probs_seq_stride + (int64_t)t * p.probs_row_stride + x];
    }
    float m = -INFINITY, cm = -INFINITY;                       // cm, cs: of the lane's first chunk (mostly its only one)
    double cs = 0.0;
    int arg = INT32_MAX;
    for (int c = lane; c < p.nc; c += 64) {
      const float om = p.top[at + c];
      const int oa = p.arg[at + c];
      if (c == lane) { cm = om; cs = p.sum[at + c]; }
      if (om > m || (om == m && oa < arg)) { m = om; arg = oa; }
    }
    wave_max<true>(m, arg);
    double z = 0.0, px = 0.0;
    if (p.scale != 0.0 && m != -INFINITY) {
      z = cs * weight(cm, m, p.scale);
      for (int c = lane + 64; c < p.nc; c += 64) z += p.sum[at + c] * weight(p.top[at + c], m, p.scale);
      z = wave_sum_f64(z);
      px = weight(lx, m, p.scale);
    }
    if (lane == 0) {
      bool stands = inside && m != -INFINITY;
      if (stands) stands = p.scale == 0.0 ? x == arg : (double)u * (double)qx * z < px;
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

// weight of a token in the draw, in units of the row's exp((x - max) / temperature): l its logit, q the draft's probability of it
__device__ __forceinline__ double draw_weight(float l, float q, int kind, const Decision& d, double scale) {
  const double w = weight(l, d.top, scale);
  return kind == LESS_DRAFT ? fmax(w - (double)q * d.z, 0.0) : w;
}

// (512 threads: the five rows of a four-draft sequence are joined by eight waves at once; when that was chosen 32 sequences took 46.8 us in all, with 256
// threads 49.6 - 51.5, with 1024 52.5; 43 now)
constexpr int kRestThreads = 512, kRestPer = kChunk / kRestThreads, kRestWaves = kRestThreads / 64;
template <bool kF32>
__global__ __launch_bounds__(kRestThreads) void verify_rest_kernel(VerifyParams p) {
  __shared__ double red[kRestWaves];
  const int ch = blockIdx.x, b = blockIdx.y, n = drafts_of(p, b);
  if (n < 0) return;
  const Decision d = decide<kF32>(p, b, n);
  if (d.a == n || d.top == -INFINITY) return;
  const int64_t row = (int64_t)b * p.seq_stride + (int64_t)d.a * p.row_stride, q_row = (int64_t)b * p.probs_seq_stride + (int64_t)d.a * p.probs_row_stride;
  float l[kRestPer], q[kRestPer];
#pragma unroll
  for (int i = 0; i < kRestPer; ++i) {
    const int64_t v = (int64_t)ch * kChunk + threadIdx.x + i * kRestThreads;
    l[i] = v < p.V ? logit<kF32>(p, row, v) : -INFINITY;
    q[i] = v < p.V ? p.probs[q_row + v] : 0.f;
  }
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kRestPer; ++i) s += draw_weight(l[i], q[i], LESS_DRAFT, d, p.scale);
  s = block_sum_f64<kRestWaves>(s, red);
  if (threadIdx.x == 0) p.rest[(int64_t)b * p.nc + ch] = s;
}

constexpr int kPickThreads = 1024, kPickPer = kChunk / kPickThreads, kPickWaves = kPickThreads / 64;

template <bool kF32>
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(VerifyParams p) {
  __shared__ double red[kPickWaves], start, target;
  __shared__ int first, last, at_chunk, draw_kind;
  __shared__ int64_t draft;
  const int b = blockIdx.x, tid = threadIdx.x, n = drafts_of(p, b);
  int64_t* out = p.tokens + (int64_t)b * (p.T + 1);
  if (n < 0) {
    for (int t = tid; t <= p.T; t += kPickThreads) out[t] = -1;
    if (tid == 0) p.accepted[b] = 0;
    return;
  }
  const Decision d = decide<kF32>(p, b, n);
  for (int t = tid; t <= p.T; t += kPickThreads)
    if (t != d.a) out[t] = t < d.a ? p.drafts[(int64_t)b * p.T + t] : -1;
  if (tid == 0) p.accepted[b] = d.a;
  if (d.top == -INFINITY || p.scale == 0.0) {               // greedy, or a row that offers nothing
    if (tid == 0) out[d.a] = d.top == -INFINITY ? -1 : d.arg;
    return;
  }
  const int64_t row = (int64_t)b * p.seq_stride + (int64_t)d.a * p.row_stride, q_row = (int64_t)b * p.probs_seq_stride + (int64_t)d.a * p.probs_row_stride;
  if (tid < 64) {                                              // one wave finds the chunk that the draw falls into
    const int64_t at = ((int64_t)b * (p.T + 1) + d.a) * p.nc;
    int kind = d.a == n ? FROM_ROW : (p.probs ? LESS_DRAFT : WITHOUT_DRAFT);
    int64_t x = -1;
    if (kind == WITHOUT_DRAFT) {
      x = p.drafts[(int64_t)b * p.T + d.a];
      if (x < 0 || x >= p.V) { x = -1; kind = FROM_ROW; }
    }
    const int cx = x >= 0 ? (int)(x / kChunk) : -1;
    auto share = [&](int c) {
      if (c >= p.nc) return 0.0;
      if (kind == LESS_DRAFT) return p.rest[(int64_t)b * p.nc + c];
      const double* s = kind == WITHOUT_DRAFT && c == cx ? p.others + (int64_t)b * p.T + d.a : p.sum + at + c;
      return *s * weight(p.top[at + c], d.top, p.scale);
    };
    const float u = p.u[(int64_t)b * (p.T + 1) + p.T];
    double total, held;                                        // held: this lane's share of the first 64 chunks (mostly all there are)
    for (;;) {                                                 // twice at most: nothing left of p - q (they are equal) -> p itself
      double mine = held = share(tid);
      for (int c = tid + 64; c < p.nc; c += 64) mine += share(c);
      total = wave_sum_f64(mine);
      if (total > 0.0 || kind == FROM_ROW) break;
      kind = FROM_ROW; x = -1;
    }
    const double want = (double)u * total;
    double run = 0.0, base = 0.0;                              // run: of the chunks before this round's 64
    int chunk = 0;                                             // the last one with a share so far
    for (int c0 = 0; c0 < p.nc; c0 += 64) {
      const double w = c0 ? share(c0 + tid) : held;
      const double incl = wave_scan_f64(w);
      const double before = run + (incl - w);
      const unsigned long long has = __ballot(w > 0.0), over = __ballot(w > 0.0 && run + incl > want);
      const unsigned long long pick = over ? (over & -over) : has;
      if (pick) {
        const int l = over ? __ffsll((long long)pick) - 1 : 63 - __clzll((long long)pick);
        chunk = c0 + l;
        base = lane_f64(before, __builtin_amdgcn_readfirstlane(l));
      }
      if (over) break;
      run += lane_f64(incl, 63);
    }
    if (tid == 0) { at_chunk = chunk; start = base; target = want; draw_kind = kind; draft = x; first = INT32_MAX; last = -1; }
  }
  __syncthreads();
  const int kind = draw_kind;
  const int64_t x = draft;
  float l[kPickPer], q[kPickPer];
  const int64_t v0 = (int64_t)at_chunk * kChunk + (int64_t)tid * kPickPer;
#pragma unroll
  for (int i = 0; i < kPickPer; ++i) {
    const bool in = v0 + i < p.V && v0 + i != x;               // (x: the refused certain draft, or -1)
    l[i] = in ? logit<kF32>(p, row, v0 + i) : -INFINITY;
    q[i] = in && kind == LESS_DRAFT ? p.probs[q_row + v0 + i] : 0.f;
  }
  double w[kPickPer], sum = 0.0;
#pragma unroll
  for (int i = 0; i < kPickPer; ++i) { w[i] = draw_weight(l[i], q[i], kind, d, p.scale); sum += w[i]; }
  const double incl = wave_scan_f64(sum);
  if ((tid & 63) == 63) red[tid >> 6] = incl;
  __syncthreads();
  double run = start + (incl - sum);
#pragma unroll
  for (int k = 0; k < kPickWaves - 1; ++k) run += k < (tid >> 6) ? red[k] : 0.0;
  int hit = INT32_MAX, able = -1;
#pragma unroll
  for (int i = 0; i < kPickPer; ++i) {
    run += w[i];
    if (w[i] > 0.0) {
      able = (int)(v0 + i);
      if (hit == INT32_MAX && run > target) hit = able;
    }
  }
  const unsigned long long hits = __ballot(hit != INT32_MAX), ables = __ballot(able >= 0);        // (one LDS atomic per wave: 1024 of them take 5 us)
  const int wave_hit = __builtin_amdgcn_readlane(hit, __builtin_amdgcn_readfirstlane(hits ? __ffsll((long long)hits) - 1 : 0));
  const int wave_able = __builtin_amdgcn_readlane(able, __builtin_amdgcn_readfirstlane(ables ? 63 - __clzll((long long)ables) : 0));
  if ((tid & 63) == 0) {
    if (hits) atomicMin(&first, wave_hit);
    if (ables) atomicMax(&last, wave_able);
  }
  __syncthreads();
  if (tid == 0) out[d.a] = first != INT32_MAX ? first : last;
}

template <bool kF32>
int launch(const VerifyParams& p, hipStream_t s) {
  verify_stats_kernel<kF32><<<dim3((unsigned)p.nc, (unsigned)(p.T + 1), (unsigned)p.batch), kThreads, 0, s>>>(p);
  int rc = qp_check_launch("verify_drafts(stats)");
  if (rc) return rc;
  if (p.probs && p.scale != 0.0) {
    verify_rest_kernel<kF32><<<dim3((unsigned)p.nc, (unsigned)p.batch), kRestThreads, 0, s>>>(p);
    if ((rc = qp_check_launch("verify_drafts(rest)"))) return rc;
  }
  verify_pick_kernel<kF32><<<(unsigned)p.batch, kPickThreads, 0, s>>>(p);
  return qp_check_launch("verify_drafts(pick)");
}

}  // namespace

int64_t qp_verify_max_vocab() { return (int64_t)kChunk * kMaxChunks; }
int qp_verify_max_drafts() { return kMaxDrafts; }

size_t qp_verify_workspace_bytes_impl(int batch, int t_max, int64_t vocab) {
  const size_t nc = (size_t)((vocab + kChunk - 1) / kChunk), rows = (size_t)batch * (t_max + 1);
  return rows * nc * (sizeof(double) + sizeof(float) + sizeof(int)) + (size_t)batch * (nc + t_max) * sizeof(double);
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
  p.scale = temperature > 0.f ? 1.4426950408889634074 / (double)temperature : 0.0;
  const size_t rows = (size_t)batch * (t_max + 1) * p.nc;
  p.sum = (double*)workspace;
  p.rest = p.sum + rows;
  p.others = p.rest + (size_t)batch * p.nc;
  p.top = (float*)(p.others + (size_t)batch * t_max);
  p.arg = (int*)(p.top + rows);
  p.accepted = n_accepted; p.tokens = tokens;
  return logits_f32 ? launch<true>(p, s) : launch<false>(p, s);
}
