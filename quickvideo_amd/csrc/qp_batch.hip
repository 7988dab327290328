// Decoding a BATCH of sequences over one prefilled video (beams, sampled answers, several questions, drafted tokens).  All sequences
// share the video's keys (the layer's arena, contiguous, frozen); what a sequence adds - its question, its generated tokens - lives in
// pages of its own: pages [n_pages][n_kv][page_size][128], page_table int32 [batch][max_pages], key row j of sequence b = slot j % page_size
// of page page_table[b][j / page_size].  seq_len[b] = rows stored before this step, n_new[b] <= t_max = rows of this step; both are read on
// the device, so a captured step replays with new lengths.  A page number outside [0, n_pages) is never followed.
//
//   batch_rope_append_kernel   rotates the step's q and k rows and stores k / v into the pages
//   batch_attn_kernel          attention of (batch x t_max) query rows over (shared prefix, own pages): partial results per key range
//   batch_combine_kernel       joins the partial results of a row
//   batch_attn_direct_kernel   both in one launch, for few keys
#include "qp_attn.h"

namespace {

using qpattn::lds_read_b128;
using qpattn::lds_read_tr16;
using qpattn::s16x8_t;
using qpattn::xhalf_max;
using qpattn::xhalf_sum;

struct Pages {
  const int* table;               // [batch][max_pages]
  const int* seq_len;             // [batch]
  const int* n_new;               // [batch] or NULL (= t_max for all)
  int max_pages, n_pages, page_size;
  int64_t page_stride16;          // uint4 between consecutive pages
};

__device__ __forceinline__ int rows_new(const Pages& p, int b, int t_max) {
  if (!p.n_new) return t_max;
  const int n = p.n_new[b];
  return n < 0 ? 0 : (n > t_max ? t_max : n);
}
// uint4 offset of key row j of sequence b, kv head h; -1 when the row has no page
__device__ __forceinline__ int64_t page_row16(const Pages& p, int b, int h, int j) {
  if ((unsigned)j >= (unsigned)p.max_pages * (unsigned)p.page_size) return -1;
  const unsigned pi = (unsigned)j / (unsigned)p.page_size, slot = (unsigned)j - pi * (unsigned)p.page_size;
  const int page = p.table[(int64_t)b * p.max_pages + pi];
  if ((unsigned)page >= (unsigned)p.n_pages) return -1;
  return (int64_t)page * p.page_stride16 + ((int64_t)h * p.page_size + slot) * 16;
}

// y[d] = x[d] cos[d] - x[d + 64] sin[d],  y[d + 64] = x[d + 64] cos[d] + x[d] sin[d],  d < 64.
// 16 lanes per head row (16 B each), the partner half comes from lane ^ 8.  A product of two bf16 is exact in fp32, so each output is
// two exact products, one fp32 sum and ONE rounding to bf16 (qp_rope_append rounds after every step because the reference's bf16 tensors
// do; a page's keys are never compared bit for bit with the reference's, and the nearer value costs nothing).
// Bytes bound: every row of qkv is read once and written once.
__global__ __launch_bounds__(256) void batch_rope_append_kernel(const uint4* __restrict__ qkv, const uint4* __restrict__ cos_t,
                                                                const uint4* __restrict__ sin_t, Pages pg, int t_max, int hq, int hkv,
                                                                int head_blocks, uint4* __restrict__ q_out, uint4* __restrict__ k_pages,
                                                                uint4* __restrict__ v_pages) {
  const int c = threadIdx.x & 15;
  const int64_t row = blockIdx.x / head_blocks;                // b * t_max + t (uniform)
  const int hr = (int)(blockIdx.x % head_blocks) * 16 + (threadIdx.x >> 4);
  const int b = (int)(row / t_max), t = (int)(row % t_max);
  if (t >= rows_new(pg, b, t_max)) return;
  const int heads = hq + 2 * hkv;
  if (hr >= heads) return;                                     // whole 16-lane groups
  const uint4 x = qkv[(row * heads + hr) * 16 + c];
  const int64_t row_to = (int64_t)pg.seq_len[b] + t;
  const int j = row_to > INT32_MAX ? -1 : (int)row_to;
  if (hr >= hq + hkv) {
    const int64_t at = page_row16(pg, b, hr - hq - hkv, j);
    if (at >= 0) v_pages[at + c] = x;
    return;
  }
  const uint4 ct = cos_t[row * 8 + (c & 7)], st = sin_t[row * 8 + (c & 7)];
  uint4 p;
  auto across = [](unsigned v) { return (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true); };         // row_ror 8: lane i ^ 8 of 16
  p.x = across(x.x); p.y = across(x.y); p.z = across(x.z); p.w = across(x.w);
  const float sign = (c < 8) ? -1.f : 1.f;
  const unsigned xw[4] = {x.x, x.y, x.z, x.w}, pw[4] = {p.x, p.y, p.z, p.w}, cw[4] = {ct.x, ct.y, ct.z, ct.w}, sw[4] = {st.x, st.y, st.z, st.w};
  unsigned o[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float lo = __uint_as_float(xw[w] << 16) * __uint_as_float(cw[w] << 16) + (sign * __uint_as_float(pw[w] << 16)) * __uint_as_float(sw[w] << 16);
    const float hi = __uint_as_float(xw[w] & 0xffff0000u) * __uint_as_float(cw[w] & 0xffff0000u) +
                     (sign * __uint_as_float(pw[w] & 0xffff0000u)) * __uint_as_float(sw[w] & 0xffff0000u);
    o[w] = (unsigned)f32_to_bf16_bits(lo) | ((unsigned)f32_to_bf16_bits(hi) << 16);
  }
  const uint4 y = make_uint4(o[0], o[1], o[2], o[3]);
  if (hr < hq) {
    q_out[(row * hq + hr) * 16 + c] = y;
  } else {
    const int64_t at = page_row16(pg, b, hr - hq, j);
    if (at >= 0) k_pages[at + c] = y;
  }
}

// ---- attention ------------------------------------------------------------------------------------------------------------------------
// Query rows of kv head h: r = (b * t_max + t) * G + g, g < G = hq / hkv, R = batch * t_max * G of them.  All R rows attend every prefix key, so
// the prefix is ONE R-row problem per kv head and is read once for the batch; the pages of a sequence are attended by its own t_max * G rows,
// row (t, g) seeing keys j <= seq_len + t.  Both kinds of work are cut into key ranges; every range leaves (max, sum, o[128]) per row, in
// 32 bits, and batch_combine_kernel joins them:  out = sum_p 2^((m_p - M) c) o_p / sum_p 2^((m_p - M) c) l_p,  c = scale * log2(e).
struct BatchAttnParams {
  const uint4* q; uint16_t* out;
  const uint4* k_pre; const uint4* v_pre; int64_t pre_hs16; int64_t P;
  const uint4* k_pages; const uint4* v_pages;
  Pages pg;
  int batch, t_max, hq, hkv, G; float c;
  int64_t R;
  // prefix: at most `prefix_wgs` workgroups share (row blocks of the batch's live rows) x (key ranges); see key_ranges()
  unsigned prefix_wgs, once, slots; int ns_max; bool compact;
  int ns;                         // without `compact`: the ranges, 0 = no prefix
  float* pre_o; float2* pre_ml;   // [hkv][ns][live rows] rows of 128 floats / (max, sum)
  int* starts;                    // with `compact`: [batch + 1] live tokens before a sequence, then the ranges, left for the joining kernel
  // pages: ns2 key ranges, nrb2 row blocks per sequence and kv head
  int ns2, nrb2; unsigned page_wgs;
  float* part_o; float2* part_ml; // [hkv][ns2][R]
};

// A padded batch (n_new given) is computed without its padding: the live tokens are numbered through, row = (live token) * G + g, and the workgroups are
// dealt over as many row blocks as that makes, so that with few live rows every block's keys are cut into more ranges.
constexpr int kMaxCompact = 512;  // sequences whose counts fit in LDS (a larger padded batch is computed with its padding)
struct Blocks { int64_t rows; unsigned nrb; };
__host__ __device__ inline Blocks row_blocks(int64_t tokens, int G, int block_rows) {
  const unsigned rows = (unsigned)tokens * (unsigned)G;        // (batch * t_max * hq <= 2^26)
  return {(int64_t)rows, (rows + block_rows - 1) / (unsigned)block_rows};
}
// Few row blocks: ranges so many that `once` workgroups, one for each place on the card, are busy (multiples of 8: see the mapping to XCDs).
constexpr unsigned kFewBlocks = 4;
__host__ __device__ inline int ranges_of_few(unsigned nrb, unsigned once, int hkv, int ns_max) {
  const int ns = (int)(once / nrb / 8 * 8 / (unsigned)hkv);
  return ns < 1 ? 1 : (ns < ns_max ? ns : ns_max);
}
// Many row blocks do not divide the card so neatly: the number of ranges, up to 64, that costs least, in tiles of one workgroup - rounds over an XCD's
// places x (tiles of a range + about 3 for its start and end) + writing and reading its partial results.  14 blocks of 256 rows over 32785 keys and 4
// heads: 548 us with the two ranges of the rule above, 340 with the four found here.
__host__ __device__ inline float ranges_cost(unsigned ns, unsigned nrb, unsigned prefix_wgs, unsigned slots, int hkv, int ns_max, unsigned block_rows, unsigned tiles) {
  const unsigned on_xcd = (hkv * ns + 7) / 8 * nrb;
  if (ns > 1 && (ns > (unsigned)ns_max || on_xcd * 8 > prefix_wgs)) return 3e38f;
  const unsigned rounds = (on_xcd + slots / 8 - 1) / (slots / 8);
  return (float)rounds * (float)((tiles + ns - 1) / ns + 3) + (float)nrb * (float)(block_rows * ns * hkv) * (1.0f / 10240.0f);
}
// live token -> b * t_max + t
__device__ __forceinline__ int64_t token_place(const BatchAttnParams& p, const int* starts, int64_t tok) {
  if (!p.compact) return tok;
  int lo = 0, hi = p.batch;                                    // starts[lo] <= tok < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= (int)tok) lo = mid; else hi = mid;
  }
  return (int64_t)lo * p.t_max + (tok - starts[lo]);
}

constexpr float kTiny = 1e-38f;   // least weight of an infinite value that is seen: it shows however small its probability
// A range's partial result o joins with its weight a.  Where a underflows, a finite o adds nothing, however large it is; only an infinite one needs the
// floor.  kFaint: such weights are among the row's; the others do without the choice (40 sequences over 4000 keys 20.3 us, with it 20.6).
template <bool kFaint>
__device__ __forceinline__ void add_part(float4& acc, float4 o, float a) {
  auto weight = [&](float x) { return kFaint && !(fabsf(x) < INFINITY) ? fmaxf(a, kTiny) : a; };
  acc.x = __builtin_fmaf(o.x, weight(o.x), acc.x); acc.y = __builtin_fmaf(o.y, weight(o.y), acc.y);
  acc.z = __builtin_fmaf(o.z, weight(o.z), acc.z); acc.w = __builtin_fmaf(o.w, weight(o.w), acc.w);
}
constexpr int kMaxKeys = 1 << 30; // of the prefix, and of a sequence's table: key numbers and their sums fit in 32 bits

// largest of eight bf16 as 15-bit patterns (even and odd places apart); is_odd: an exponent of all ones among them (infinity, NaN)
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2_t magnitude(uint4 x) {
  auto mag = [](unsigned w) { return __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu); };
  return __builtin_elementwise_max(__builtin_elementwise_max(mag(x.x), mag(x.y)), __builtin_elementwise_max(mag(x.z), mag(x.w)));
}
__device__ __forceinline__ bool is_odd(u16x2_t m) { return m.x >= 0x7f80 || m.y >= 0x7f80; }
__device__ __forceinline__ void make_finite(uint4& x) {       // such numbers to zero
  unsigned* w = reinterpret_cast<unsigned*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
    if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0x0000ffffu;
  }
}

// The rare end of a range: every value that is not finite is added, times its probability, to the rows that see it, where their partial results
// lie (one thread per row: it wrote none of them itself, the barrier before the call orders the writes).
template <bool kPaged>
__device__ __forceinline__ void add_odd_values(const BatchAttnParams& p, int kvh, int b, int64_t row0, int64_t row_end, int k0, int k1, float* part_o,
                                               const float2* part_ml, const int* starts) {
  for (int key = k0; key < k1; ++key) {
    const int64_t at = kPaged ? page_row16(p.pg, b, kvh, key) : (int64_t)kvh * p.pre_hs16 + (int64_t)key * 16;
    if (at < 0) continue;
    const uint4* vrow = (kPaged ? p.v_pages : p.v_pre) + at;
    bool odd = false;
    for (int i = 0; i < 16; ++i) odd |= is_odd(magnitude(vrow[i]));
    if (!odd) continue;                                        // (the same for all threads)
    const uint16_t* krow = reinterpret_cast<const uint16_t*>((kPaged ? p.k_pages : p.k_pre) + at);
    for (int64_t r = row0 + threadIdx.x; r < row_end; r += blockDim.x) {
      const int64_t bt = kPaged ? r / p.G : token_place(p, starts, r / p.G);
      if (kPaged && key > (int64_t)p.pg.seq_len[b] + (bt - (int64_t)b * p.t_max)) continue;
      const uint16_t* qrow = reinterpret_cast<const uint16_t*>(p.q) + ((bt * p.hq) + (int64_t)kvh * p.G + r % p.G) * 128;
      float s = 0.f;
      for (int d = 0; d < 128; ++d) s = __builtin_fmaf(bf16_bits_to_f32(qrow[d]), bf16_bits_to_f32(krow[d]), s);
      const float pe = fmaxf(__builtin_amdgcn_exp2f(__builtin_fmaf(s, p.c, -part_ml[r].x * p.c)), kTiny);
      for (int d = 0; d < 128; ++d) {
        const uint16_t w = reinterpret_cast<const uint16_t*>(vrow)[d];
        if ((w & 0x7f80u) == 0x7f80u) part_o[r * 128 + d] += pe * bf16_bits_to_f32(w);
      }
    }
  }
}

// A workgroup of WR x WK waves takes a block of 32 * WR rows over one key range, a tile of 64 keys at a time, staged in LDS (K row-major with
// XOR-swizzled 16-B slots; V as [key / 4][d / 32][key % 4][32] for the transposing LDS reads).  Wave (wr, wk) owns rows [32 wr, 32 wr + 32) and, for
// WK = 2, half of the tile's keys: S^T = K.Q^T (rows are the columns of v_mfma_f32_32x32x16_bf16: a lane owns one row), online softmax,
// O^T += V^T.P, all sums in fp32.  The prefix goes straight into LDS (walk_prefix), the pages, whose rows lie apart, through registers (walk_keys).
// A value that is not finite would spoil rows that do not see it (0 * infinity is NaN) and the sum of the two products below.  walk_keys puts zero in
// its place, and the range ends with add_odd_values; walk_prefix does not look, but such a value leaves no result of its range finite, which is then
// computed again with walk_keys.
// What bounds it: two waves a SIMD (200 registers each) whose matrix instructions are 60 % of a tile's time with all eight row tiles filled (3100 of
// 5164 clocks: 448 live rows of 1708 over 32785 keys, 62 us), the rest is the barrier and the loads' issue; with fewer rows the bytes: 56 rows over 504015 keys
// 186 us, 5.5 TB/s.  Tried and slower: staging the prefix through registers, one tile ahead (448 rows 64.5 us, 72 rows over 30737 keys 44.4 against
// 39.5); the loads issued between the products (64.1, 40.6); two tiles of 64 keys in LDS instead of three for 8 waves (61.8, 41.6); four (63.0, 40.5);
// wave priorities (no effect).
// P goes into the product as TWO bf16 numbers, bf16(p) and bf16(p - bf16(p)): 2^-16 of p is lost at most instead of 2^-8.  Rounded once, as the prefill
// and decode kernels do it, the result's error against 64 bits is 0.0021 - 0.0027 of it, with two terms 0.0017, which is its own rounding; the second
// product reuses the V fragments, and a step that waits for the prefix's bytes has the matrix pipe free.  Every form does so, also that of many tokens,
// for which the prefill kernel with its one rounding is faster in part (28 and 4 heads, 4 x 61 tokens over 32785 keys 135 against 175 us, 96 x 1 76
// against 89, 4 x 128 over 4096 keys 70 against 73, over 2048 52 both; 4 and 2 heads, 2 x 130 tokens over 8200 keys 47 against 26).
template <int WR, int WK>
struct Shape {
  static constexpr int NT = 64 * WR * WK, KB = WK == 1 ? 2 : 1, TILE = 32 * WK * KB, PT = TILE * 16 / NT;   // PT: 16-B pieces a thread stages of K and of V
  static constexpr int kBuffers = NT == 512 ? 3 : 2;           // of the prefix: one workgroup of 8 waves fits on a CU, two of 4
};
struct Rows {                      // what a lane keeps of its row (both halves of a wave: the same row, other keys)
  f32x16_t o[4];                   // [d / 32], unscaled
  float m, l;
};
// p = hi + lo with both in bf16, two probabilities at a time (one conversion instruction per pair and term)
__device__ __forceinline__ void split_pair(float a, float b, unsigned& hi, unsigned& lo) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  const bf2 h = {(__bf16)a, (__bf16)b};
  hi = __builtin_bit_cast(unsigned, h);
  const bf2 l = {(__bf16)(a - __uint_as_float(hi << 16)), (__bf16)(b - __uint_as_float(hi & 0xffff0000u))};
  lo = __builtin_bit_cast(unsigned, l);
}
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

struct Shared {                    // LDS besides the tile
  unsigned long long holes[2];     // by parity of the tile: its rows without a page
  int odd;                         // a value that is not finite was met
};

#define QP_BATCH_FENCE() __builtin_amdgcn_sched_barrier(0)

// The matrix work of one wave on KB 32-key blocks (kb0 ...) of a staged tile.  `hidden`: some key of the tile is not seen by some row; then this lane's
// row sees rows up to last_row of the tile, without those of hole_bits.  kBeside (two blocks): the first one's products run beside the second one's
// exponentials; otherwise block after block.
template <int KB, bool kBeside>
__device__ __forceinline__ void take_tile(float c, const unsigned char* kl, const unsigned char* vl, int koff, int voff, int kb0, const bf16x8_t (&qf)[8],
                                          bool hidden, int last_row, unsigned long long hole_bits, int hi, float& m_run, float& l_run, f32x16_t (&o)[4]) {
  // LDS reads run ahead of the products that need them: hipcc left to itself reads each fragment just before its use and waits for it
  auto read_k = [&](int kb, bf16x8_t (&f)[8]) {
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) f[kk] = lds_read_b128(kl, kb * 32 * 256 + (koff ^ (kk << 5)));
  };
  auto read_v = [&](int kb, int cc, s16x8_t (&v)[4]) {       // the 16 keys of chunk cc, all 128 dimensions
#pragma unroll
    for (int db = 0; db < 4; ++db) {
      const int off = voff + (((kb * 8 + cc * 4) * 4 + db) << 8);
      const s16x4_t v0 = lds_read_tr16(vl, off);
      const s16x4_t v1 = lds_read_tr16(vl, off + (2 * 4 << 8));
      v[db] = (s16x8_t){v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
    }
  };
  auto scores = [&](const bf16x8_t (&f)[8]) {
    f32x16_t s = (f32x16_t){0};
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[kk], qf[kk], s, 0, 0, 0);
    return s;
  };
  auto hide = [&](int kb, f32x16_t& s) {                     // scores of keys this lane's row does not see
    if (hidden) {
      const int last = last_row - 4 * hi;                    // (seen from this lane's rows)
      const unsigned have = (unsigned)((~hole_bits >> (4 * hi)) >> ((kb & 1) * 32));
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int row = (e & 3) + 8 * (e >> 2);
        s[e] = kb * 32 + row <= last && ((have >> row) & 1) ? s[e] : -INFINITY;
      }
    }
  };
  auto largest = [&](const f32x16_t& s) {
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    return xhalf_max(mx);
  };
  auto outgrown = [&](float mx) { return !__all((mx - m_run) * c <= 8.0f); };       // the reference moves only when a row outgrows it by 2^8
  auto move_reference = [&](float mx) {
    const float m_new = fmaxf(m_run, mx);
    const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * c);
    m_run = m_new;
    l_run *= alpha;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
  };
  auto exponentials = [&](const f32x16_t& s, u32x4_t (&pf)[2], u32x4_t (&pr)[2]) {
    const float mc = m_run * c;
    float rs = 0.f;
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[cc * 8 + 2 * e], c, -mc));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[cc * 8 + 2 * e + 1], c, -mc));
        rs += p0 + p1;
        unsigned h, l;
        split_pair(p0, p1, h, l);
        pf[cc][e] = h; pr[cc][e] = l;
      }
    return rs;                                               // (this half's keys)
  };
  auto product = [&](int i, const s16x8_t (&va)[4], const s16x8_t (&vb)[4], const u32x4_t (&pf)[2], const u32x4_t (&pr)[2]) {       // i-th of a block's 16
    const int db = i & 3;
    const s16x8_t v = i < 8 ? va[db] : vb[db];
    const u32x4_t pp = ((i >> 2) & 1 ? pr : pf)[i >> 3];
    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, pp), o[db], 0, 0, 0);
  };
  // exponentials() dealt among the 16 matrix instructions mfma(0) ... mfma(15): a wave issues in order, so what is to run beside a matrix instruction
  // has to stand behind it, and the fences keep it there (left to itself hipcc puts all of one kind first)
  auto exponentials_beside = [&](auto&& mfma, const f32x16_t& s, u32x4_t (&pf)[2], u32x4_t (&pr)[2]) {
    const float mc = m_run * c;
    float rs = 0.f, pe[16];
    auto pack = [&](int q) {                                   // the q-th pair
      rs += pe[2 * q] + pe[2 * q + 1];
      unsigned h, l;
      split_pair(pe[2 * q], pe[2 * q + 1], h, l);
      pf[q >> 2][q & 3] = h; pr[q >> 2][q & 3] = l;
    };
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      mfma(i);
      pe[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -mc));
      if (i >= 2 && i % 2 == 0) pack(i / 2 - 1);
      QP_BATCH_FENCE();
    }
    pack(7);
    asm volatile("" : "+v"(pf[0]), "+v"(pf[1]), "+v"(pr[0]), "+v"(pr[1]));      // (made here, not sunk to their use)
    return rs;
  };
  if constexpr (!kBeside) {
#pragma unroll
    for (int n = 0; n < KB; ++n) {
      const int kb = kb0 + n;
      bf16x8_t kf[8];
      s16x8_t va[4], vb[4];
      u32x4_t pf[2], pr[2];
      read_k(kb, kf);
      QP_BATCH_FENCE();
      f32x16_t s = scores(kf);
      read_v(kb, 0, va);
      QP_BATCH_FENCE();
      hide(kb, s);
      const float mx = largest(s);
      if (outgrown(mx)) move_reference(mx);
      l_run += xhalf_sum(exponentials(s, pf, pr));
      QP_BATCH_FENCE();
      read_v(kb, 1, vb);
      QP_BATCH_FENCE();
#pragma unroll
      for (int i = 0; i < 16; ++i) product(i, va, vb, pf, pr);
      QP_BATCH_FENCE();
    }
  } else {
    // Both blocks' scores, then the first one's products beside the second one's exponentials.
    const int kb = kb0;
    s16x8_t va[4], vb[4];
    u32x4_t pf0[2], pr0[2], pf1[2], pr1[2];
    f32x16_t s0, s1;
    {
      bf16x8_t f[8];
      read_k(kb, f);
      QP_BATCH_FENCE();
      s0 = scores(f);
    }
    QP_BATCH_FENCE();
    {
      bf16x8_t f[8];
      read_k(kb + 1, f);
      QP_BATCH_FENCE();
      hide(kb, s0);
      s1 = scores(f);
    }
    QP_BATCH_FENCE();
    read_v(kb, 0, va);
    QP_BATCH_FENCE();
    hide(kb + 1, s1);
    float mx = fmaxf(largest(s0), largest(s1));
    if (outgrown(mx)) move_reference(mx);
    float rs = exponentials(s0, pf0, pr0);
    QP_BATCH_FENCE();
    rs += exponentials_beside([&](int i) { if (i == 4) read_v(kb, 1, vb); product(i, va, vb, pf0, pr0); }, s1, pf1, pr1);
    read_v(kb + 1, 0, va);
    read_v(kb + 1, 1, vb);
    QP_BATCH_FENCE();
    l_run += xhalf_sum(rs);
#pragma unroll
    for (int i = 0; i < 16; ++i) product(i, va, vb, pf1, pr1);
  }
}

template <int WR, int WK, bool kPaged>
__device__ __forceinline__ void walk_keys(const BatchAttnParams& p, int kvh, int b, int64_t r, bool row_live, bool wave_live, const bf16x8_t (&qf)[8], int k0,
                                          int k1, unsigned char* lds, Shared& sh, Rows& st) {
  using S = Shape<WR, WK>;
  constexpr int NT = S::NT, PT = S::PT, KB = S::KB, TILE = S::TILE;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, l31 = lane & 31;
  const int wk = wave / WR;
  unsigned char* kl = lds;
  unsigned char* vl = lds + TILE * 256;
  int limit = INT32_MAX;                                       // last visible key of this lane's row
  int seen_by_all = INT32_MAX;                                 // keys below this are visible to every row of the sequence
  if (kPaged) {
    const int stored = min(p.pg.seq_len[b], kMaxKeys);        // (a table has no more rows)
    seen_by_all = stored + 1;
    limit = stored + (row_live ? (int)(r / p.G - (int64_t)b * p.t_max) : 0);
  }
  const uint4* kbase = kPaged ? p.k_pages : p.k_pre + (int64_t)kvh * p.pre_hs16;
  const uint4* vbase = kPaged ? p.v_pages : p.v_pre + (int64_t)kvh * p.pre_hs16;
  const int slot16 = tid & 15, srow = tid >> 4;                // this thread stages rows srow + i * (NT / 16), 16-B slot slot16
  uint4 kx[PT], vx[PT];
  unsigned holes = 0;                                          // bit i: staged row i has no page
  auto load = [&](int t0) {                                // rows past the end are zero: their probability is 0, and 0 * 0 stays 0
    if (!kPaged) {
      const uint4* kt = kbase + (int64_t)t0 * 16;              // a tile of the prefix is 16 KB in a row
      const uint4* vt = vbase + (int64_t)t0 * 16;
      if (t0 + TILE <= k1) {
#pragma unroll
        for (int i = 0; i < PT; ++i) { kx[i] = kt[tid + i * NT]; vx[i] = vt[tid + i * NT]; }
      } else {
        const int rows = k1 - t0;
#pragma unroll
        for (int i = 0; i < PT; ++i) {
          kx[i] = vx[i] = make_uint4(0, 0, 0, 0);
          if (srow + i * (NT / 16) < rows) { kx[i] = kt[tid + i * NT]; vx[i] = vt[tid + i * NT]; }
        }
      }
    } else {
      holes = 0;
#pragma unroll
      for (int i = 0; i < PT; ++i) {
        const int key = t0 + srow + i * (NT / 16);
        kx[i] = vx[i] = make_uint4(0, 0, 0, 0);
        if (key < k1) {
          const int64_t at = page_row16(p.pg, b, kvh, key);
          if (at < 0) { holes |= 1u << i; continue; }
          kx[i] = kbase[at + slot16]; vx[i] = vbase[at + slot16];
        }
      }
    }
  };
  const int koff = l31 * 256 + ((hi ^ (l31 & 15)) << 4);       // fragment kk of the lane's key: slot (2 kk + hi) ^ (key % 16)
  const int voff = (((lane & 15) >> 2) << 6) + (((lane >> 4) & 1) << 5) + ((lane & 3) << 3) + (hi << 10);
  f32x16_t (&o)[4] = st.o;
  float m_run = st.m, l_run = st.l;
  int par = 0;
  for (int t0 = k0; t0 < k1; t0 += TILE, par ^= 1) {
    load(t0);
    __syncthreads();                                           // everyone has read the previous tile
    const bool masked = kPaged && t0 + TILE > seen_by_all;    // some row of the sequence does not see some key of this tile
    u16x2_t top = {0, 0};
#pragma unroll
    for (int i = 0; i < PT; ++i) top = __builtin_elementwise_max(top, magnitude(vx[i]));
    if (is_odd(top)) {
#pragma unroll
      for (int i = 0; i < PT; ++i) make_finite(vx[i]);
      sh.odd = 1;
    }
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int row = srow + i * (NT / 16);
      if (kPaged && ((holes >> i) & 1) && slot16 == 0) atomicOr(&sh.holes[par], 1ull << row);
      *reinterpret_cast<uint4*>(kl + row * 256 + ((slot16 ^ (row & 15)) << 4)) = kx[i];
      *reinterpret_cast<uint4*>(vl + (((row >> 2) * 4 + (slot16 >> 2)) << 8) + ((row & 3) << 6) + ((slot16 & 3) << 4)) = vx[i];
    }
    __syncthreads();
    const unsigned long long hole_bits = kPaged ? sh.holes[par] : 0;
    if (kPaged && tid == 0) sh.holes[par ^ 1] = 0;            // last read before the barrier above, next written behind the next one
    if (!wave_live) continue;
    take_tile<KB, false>(p.c, kl, vl, koff, voff, wk * KB, qf, t0 + TILE > k1 || masked || hole_bits, (limit < k1 ? limit : k1 - 1) - t0, hole_bits, hi, m_run,
                         l_run, o);
  }
  st.m = m_run; st.l = l_run;
}

// The prefix's keys k0 .. k1 - 1 without a look at the values: tiles go from memory straight into LDS (buffer_load ... lds: 1 KB, four rows, per wave and
// instruction, lane i's 16 B at 16 i; the images are made by what each lane reads), kBuffers of them, so that the next ones are under way while one is
// computed, with one barrier a tile.  Rows behind k1 read as zero (the buffer's bound).  The loads are asm, each with its own wait before the barrier:
// hipcc would otherwise wait for all of them at the first LDS read.
// m0 is written by name, so it is declared; hipcc warns that it is a reserved register (it keeps no variable there, but has uses of its own).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(unsigned lds_at, int voff, u32x4_t rsrc) {       // (the wait states: rsrc may come from a vector instruction)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds_at), "v"(voff), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }

template <int WR, int WK>
__device__ __forceinline__ void walk_prefix(const BatchAttnParams& p, int kvh, bool wave_live, bf16x8_t (&qf)[8], int k0, int k1, unsigned char* lds, Rows& st) {
  using S = Shape<WR, WK>;
  constexpr int KB = S::KB, TILE = S::TILE, NW = WR * WK, NB = S::kBuffers, PIECES = TILE / 4 / NW;      // 1-KB pieces a wave loads of K and of V
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5, l31 = lane & 31, wk = wave / WR;
  const int koff = l31 * 256 + ((hi ^ (l31 & 15)) << 4);
  const int voff = (((lane & 15) >> 2) << 6) + (((lane >> 4) & 1) << 5) + ((lane & 3) << 3) + (hi << 10);
  const int krow = wave * 4 + (lane >> 4), ksrc = krow * 256 + (((lane & 15) ^ (krow & 15)) << 4);       // piece j: + j * NW * 1024 (NW * 4 rows, a multiple of 16)
  const int vsrc = (wave * 4 + ((lane >> 2) & 3)) * 256 + ((lane >> 4) << 6) + ((lane & 3) << 4);
  static_assert(NW * 4 % 16 == 0, "the swizzle repeats every 16 rows");
  const unsigned lds32 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char*)lds + wave * 1024;
  const unsigned char* kbase = reinterpret_cast<const unsigned char*>(p.k_pre + (int64_t)kvh * p.pre_hs16);
  const unsigned char* vbase = reinterpret_cast<const unsigned char*>(p.v_pre + (int64_t)kvh * p.pre_hs16);
  auto rsrc_of = [&](const unsigned char* base, int t0) {
    const size_t at = (size_t)(base + (int64_t)t0 * 256);
    const int rows = k1 - t0 < TILE ? k1 - t0 : TILE;
    return (u32x4_t){(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)at), (unsigned)__builtin_amdgcn_readfirstlane((int)((unsigned)(at >> 32) & 0xffffu)),
                     (unsigned)__builtin_amdgcn_readfirstlane(rows * 256), 0x00020000u};
  };
  auto load = [&](int t0, int buf) {
    const u32x4_t rk = rsrc_of(kbase, t0), rv = rsrc_of(vbase, t0);
    const unsigned at = lds32 + buf * (TILE * 512);
#pragma unroll
    for (int j = 0; j < PIECES; ++j) load_to_lds(at + j * (NW * 1024), ksrc + j * (NW * 1024), rk);
#pragma unroll
    for (int j = 0; j < PIECES; ++j) load_to_lds(at + TILE * 256 + j * (NW * 1024), vsrc + j * (NW * 1024), rv);
  };
  float m_run = st.m, l_run = st.l;
#pragma unroll
  for (int i = 0; i < NB - 1; ++i)
    if (k0 + i * TILE < k1) load(k0 + i * TILE, i);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) asm volatile("" : "+v"(qf[kk]));      // hipcc waits for the queries here, not in the loop, where its wait would be for the tiles too
  int buf = 0;
  for (int t0 = k0; t0 < k1; t0 += TILE) {
    if (NB > 2 && t0 + TILE < k1) wait_loads<(NB - 2) * 2 * PIECES>(); else wait_loads<0>();             // this wave's part of the tile is there
    __syncthreads();                                           // everyone's, and everyone has read the tile before, whose place is loaded next
    const int ahead = t0 + (NB - 1) * TILE, to = buf + NB - 1 >= NB ? buf - 1 : buf + NB - 1;
    if (ahead < k1) load(ahead, to);
    if (wave_live) {
      const unsigned char* kl = lds + buf * (TILE * 512);
      take_tile<KB, KB == 2>(p.c, kl, kl + TILE * 256, koff, voff, wk * KB, qf, t0 + TILE > k1, k1 - 1 - t0, 0, hi, m_run, l_run, st.o);
    }
    buf = buf + 1 == NB ? 0 : buf + 1;
  }
  st.m = m_run; st.l = l_run;
}

// The same for ONE row tile (WR = 1): nothing is shared, so every wave stages and computes 32-key blocks of its own (block first, first + WK, ... of the
// range) in its own 16 KB of LDS, without a barrier; waves drift apart and hide each other's waiting.
// A block is asked for when the one before is done.  Asking for the next one ahead costs 30 registers and does not pay, because a wave has two blocks here,
// rarely more (us without and with it: one launch, 12 and 2 heads, 417 keys 9.5, 10.0; 28 and 4 heads, 7 rows, 300 keys 9.7, 9.6, 400 10.4, 10.8, 500 11.9,
// 11.7; ranges of 256 keys, 7 rows over 4100 11.3, 11.1, 28 over 4100 11.95, 12.1, over 11535 13.45, 13.45, 64 rows of 8 heads over 2000 12.6, 12.7).
template <int WK, bool kPaged>
__device__ __forceinline__ void walk_alone(const BatchAttnParams& p, int kvh, int b, int64_t r, bool row_live, const bf16x8_t (&qf)[8], int k0, int k1, int first,
                                           unsigned char* lds, Shared& sh, Rows& st) {
  const int lane = threadIdx.x & 63, hi = lane >> 5, l31 = lane & 31, r4 = lane >> 4, slot16 = lane & 15;
  unsigned char* kl = lds + (threadIdx.x >> 6) * 16384;
  unsigned char* vl = kl + 8192;
  int limit = INT32_MAX, seen_by_all = INT32_MAX;              // as in walk_keys
  if (kPaged) {
    const int stored = min(p.pg.seq_len[b], kMaxKeys);
    seen_by_all = stored + 1;
    limit = stored + (row_live ? (int)(r / p.G - (int64_t)b * p.t_max) : 0);
  }
  const uint4* kbase = kPaged ? p.k_pages : p.k_pre + (int64_t)kvh * p.pre_hs16;
  const uint4* vbase = kPaged ? p.v_pages : p.v_pre + (int64_t)kvh * p.pre_hs16;
  uint4 kx[8], vx[8];
  unsigned holes = 0;                                          // bit i: staged row r4 + 4 i has no page
  auto load = [&](int t0) {
    if (!kPaged) {
      const uint4* kt = kbase + (int64_t)t0 * 16;              // 8 KB in a row
      const uint4* vt = vbase + (int64_t)t0 * 16;
      if (t0 + 32 <= k1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) { kx[i] = kt[lane + i * 64]; vx[i] = vt[lane + i * 64]; }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          kx[i] = vx[i] = make_uint4(0, 0, 0, 0);
          if (t0 + r4 + 4 * i < k1) { kx[i] = kt[lane + i * 64]; vx[i] = vt[lane + i * 64]; }
        }
      }
    } else {
      holes = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = t0 + r4 + 4 * i;
        kx[i] = vx[i] = make_uint4(0, 0, 0, 0);
        if (key < k1) {
          const int64_t at = page_row16(p.pg, b, kvh, key);
          if (at < 0) { holes |= 1u << i; continue; }
          kx[i] = kbase[at + slot16]; vx[i] = vbase[at + slot16];
        }
      }
    }
  };
  const int koff = l31 * 256 + ((hi ^ (l31 & 15)) << 4);
  const int voff = (((lane & 15) >> 2) << 6) + (((lane >> 4) & 1) << 5) + ((lane & 3) << 3) + (hi << 10);
  f32x16_t (&o)[4] = st.o;
  float m_run = st.m, l_run = st.l;
  for (int t0 = k0 + first * 32; t0 < k1; t0 += 32 * WK) {
    load(t0);
    u16x2_t top = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __builtin_elementwise_max(top, magnitude(vx[i]));
    if (__any(is_odd(top))) {
#pragma unroll
      for (int i = 0; i < 8; ++i) make_finite(vx[i]);
      sh.odd = 1;
    }
    __builtin_amdgcn_wave_barrier();                           // the last block's fragment reads stay ahead of these writes
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = r4 + 4 * i;
      *reinterpret_cast<uint4*>(kl + row * 256 + ((slot16 ^ (row & 15)) << 4)) = kx[i];
      *reinterpret_cast<uint4*>(vl + (((row >> 2) * 4 + (slot16 >> 2)) << 8) + ((row & 3) << 6) + ((slot16 & 3) << 4)) = vx[i];
    }
    unsigned have = ~0u;                                       // rows of the block that have a page
    if (kPaged && __any(holes)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned long long m = __ballot((holes >> i) & 1);
        have &= ~(((unsigned)(m & 1) | ((unsigned)(m >> 16) & 1) << 1 | ((unsigned)(m >> 32) & 1) << 2 | ((unsigned)(m >> 48) & 1) << 3) << (4 * i));
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x16_t s = (f32x16_t){0};
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      if (kk == 4) __builtin_amdgcn_sched_barrier(0);          // (half of the K fragments at a time: registers)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lds_read_b128(kl, koff ^ (kk << 5)), qf[kk], s, 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t0 + 32 > k1 || t0 + 32 > seen_by_all || have != ~0u) {
      const int last = (limit < k1 ? limit : k1 - 1) - t0 - 4 * hi;
      const unsigned seen = have >> (4 * hi);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int row = (e & 3) + 8 * (e >> 2);
        s[e] = row <= last && ((seen >> row) & 1) ? s[e] : -INFINITY;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = xhalf_max(mx);
    if (!__all((mx - m_run) * p.c <= 8.0f)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * p.c);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
    }
    const float mc = m_run * p.c;
    float rs = 0.f;
    u32x4_t pf[2], pr[2];
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[cc * 8 + 2 * e], p.c, -mc));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[cc * 8 + 2 * e + 1], p.c, -mc));
        rs += p0 + p1;
        unsigned h, l;
        split_pair(p0, p1, h, l);
        pf[cc][e] = h; pr[cc][e] = l;
      }
    l_run += xhalf_sum(rs);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        const int off = voff + (((cc * 4) * 4 + db) << 8);
        const s16x4_t v0 = lds_read_tr16(vl, off);
        const s16x4_t v1 = lds_read_tr16(vl, off + (2 * 4 << 8));
        const s16x8_t av = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
        o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, av), __builtin_bit_cast(bf16x8_t, pf[cc]), o[db], 0, 0, 0);
        o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, av), __builtin_bit_cast(bf16x8_t, pr[cc]), o[db], 0, 0, 0);
      }
  }
  st.m = m_run; st.l = l_run;
}

// Q fragments of the lane's row, an empty running state and cleared flags (ordered by the first barrier behind it)
__device__ __forceinline__ void begin_rows(const BatchAttnParams& p, int kvh, int64_t bt, int g, bool row_live, bf16x8_t (&qf)[8], Shared& sh, Rows& st) {
  const int tid = threadIdx.x, hi = (tid >> 5) & 1;
  const uint4* src = p.q + ((bt * p.hq) + (int64_t)kvh * p.G + g) * 16;
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (row_live) x = src[kk * 2 + hi];
    qf[kk] = __builtin_bit_cast(bf16x8_t, x);
  }
#pragma unroll
  for (int db = 0; db < 4; ++db) st.o[db] = (f32x16_t){0};
  st.m = -1e30f; st.l = 0.f;
  if (tid < 2) sh.holes[tid] = 0;
  if (tid == 0) sh.odd = 0;
}

// Joining the WK waves that took the keys of the same 32 rows: every wave lays its rows out in LDS, scaled to the rows' common maximum (the tiles
// are read by then); joined() adds them up.  kJoinRow: 128 + 4 floats, so that the rows start on different banks.
constexpr int kJoinRow = 132;
template <int WK> constexpr int join_bytes() { return WK * 32 * kJoinRow * 4; }
template <int WK>
__device__ __forceinline__ void lay_out_rows(const Rows& st, float c, bool row_live, float* obuf, float* lds_m, float* lds_l) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hi = lane >> 5, l31 = lane & 31;
  if (hi == 0) lds_m[wave * 32 + l31] = st.m;
  __syncthreads();
  float M = lds_m[l31];
#pragma unroll
  for (int w = 1; w < WK; ++w) M = fmaxf(M, lds_m[w * 32 + l31]);
  const float a = __builtin_amdgcn_exp2f((st.m - M) * c);
  if (hi == 0) lds_l[wave * 32 + l31] = st.l * a;
  if (row_live) {
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<float4*>(obuf + (wave * 32 + l31) * kJoinRow + db * 32 + 8 * q4 + 4 * hi) =
            make_float4(st.o[db][q4 * 4 + 0] * a, st.o[db][q4 * 4 + 1] * a, st.o[db][q4 * 4 + 2] * a, st.o[db][q4 * 4 + 3] * a);
  }
  __syncthreads();
}
template <int WK>
__device__ __forceinline__ float4 joined(const float* obuf, const float* lds_m, const float* lds_l, int row, int d4, float& m, float& l) {
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  m = lds_m[row]; l = 0.f;
#pragma unroll
  for (int w = 0; w < WK; ++w) {
    const float4 v = *reinterpret_cast<const float4*>(obuf + (w * 32 + row) * kJoinRow + d4);
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    m = fmaxf(m, lds_m[w * 32 + row]); l += lds_l[w * 32 + row];
  }
  return acc;
}

// one key range of one row block: partial results of its rows r into part_o[r], part_ml[r].  Rows of the pages are numbered with the batch's padding
// (b * t_max + t) * G + g, those of the prefix without it.
template <int WR, int WK, bool kPaged>
__device__ __forceinline__ void batch_attn_range(const BatchAttnParams& p, int kvh, int b, int64_t row0, int64_t row_end, int k0, int k1, float* part_o,
                                                 float2* part_ml, const int* starts, unsigned char* lds, float* lds_ml, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, l31 = lane & 31;
  const int wr = wave % WR, wk = wave / WR;
  const int64_t r = row0 + wr * 32 + l31;
  const bool row_live = r < row_end, wave_live = row0 + wr * 32 < row_end;
  bf16x8_t qf[8];
  Rows st;
  {
    const int64_t tok = row_live ? r / p.G : 0;
    const int g = row_live ? (int)(r - tok * p.G) : 0;
    begin_rows(p, kvh, row_live && !kPaged ? token_place(p, starts, tok) : tok, g, row_live, qf, sh, st);
  }
  if (WR == 1) {
    __syncthreads();                                           // flags cleared
    walk_alone<WK, kPaged>(p, kvh, b, r, row_live, qf, k0, k1, wave, lds, sh, st);
    __syncthreads();                                           // the blocks are read: their LDS joins the rows
  } else {
    if (!kPaged) {
      walk_prefix<WR, WK>(p, kvh, wave_live, qf, k0, k1, lds, st);
      float z = st.l * 0.f;                                    // a value that is not finite left its mark in every row: 0 * it is NaN
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) z = __builtin_fmaf(st.o[db][e], 0.f, z);
      if (row_live && z != 0.f) {                              // (what the query of a token that is not there holds does not count)
        const unsigned tok = (unsigned)r / (unsigned)p.G, seq = tok / (unsigned)p.t_max;
        if (p.compact || (int)(tok - seq * p.t_max) < rows_new(p.pg, (int)seq, p.t_max)) sh.odd = 1;
      }
      __syncthreads();
    }
    if (kPaged || sh.odd) {
      if (!kPaged) {                                           // the rare case: once more, with such values left out
#pragma unroll
        for (int db = 0; db < 4; ++db) st.o[db] = (f32x16_t){0};
        st.m = -1e30f; st.l = 0.f;
        __syncthreads();
        if (tid == 0) sh.odd = 0;                              // (it may have been a query or a key: walk_keys finds the values)
      }
      walk_keys<WR, WK, kPaged>(p, kvh, b, r, row_live, wave_live, qf, k0, k1, lds, sh, st);
    }
  }
  if (WR == 1) {
    float* obuf = reinterpret_cast<float*>(lds);
    lay_out_rows<WK>(st, p.c, row_live, obuf, lds_ml, lds_ml + WK * 32);
    const int rows = (int)(row_end - row0 < 32 ? row_end - row0 : 32);
    for (int i = tid; i < rows * 32; i += 64 * WK) {
      const int row = i >> 5, d4 = (i & 31) * 4;
      float m, l;
      const float4 acc = joined<WK>(obuf, lds_ml, lds_ml + WK * 32, row, d4, m, l);
      *reinterpret_cast<float4*>(part_o + (row0 + row) * 128 + d4) = acc;
      if (d4 == 0) part_ml[row0 + row] = make_float2(m, l);
    }
  } else {
    f32x16_t (&o)[4] = st.o;
    float m_run = st.m, l_run = st.l;
    if (WK == 2) {                                               // join the two key halves of a row (the tile's LDS is free)
      __syncthreads();
      float* obuf = reinterpret_cast<float*>(lds);               // [WR][32 rows][kJoinRow]
      if (wk == 1) {
        if (hi == 0) { lds_ml[(wr * 32 + l31) * 2] = m_run; lds_ml[(wr * 32 + l31) * 2 + 1] = l_run; }
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<float4*>(obuf + (wr * 32 + l31) * kJoinRow + db * 32 + 8 * q4 + 4 * hi) =
                make_float4(o[db][q4 * 4 + 0], o[db][q4 * 4 + 1], o[db][q4 * 4 + 2], o[db][q4 * 4 + 3]);
      }
      __syncthreads();
      if (wk == 0) {
        const float m1 = lds_ml[(wr * 32 + l31) * 2], l1 = lds_ml[(wr * 32 + l31) * 2 + 1];
        const float m = fmaxf(m_run, m1);
        const float a0 = __builtin_amdgcn_exp2f((m_run - m) * p.c), a1 = __builtin_amdgcn_exp2f((m1 - m) * p.c);
        m_run = m;
        l_run = l_run * a0 + l1 * a1;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const float4 other = *reinterpret_cast<const float4*>(obuf + (wr * 32 + l31) * kJoinRow + db * 32 + 8 * q4 + 4 * hi);
            o[db][q4 * 4 + 0] = o[db][q4 * 4 + 0] * a0 + other.x * a1;
            o[db][q4 * 4 + 1] = o[db][q4 * 4 + 1] * a0 + other.y * a1;
            o[db][q4 * 4 + 2] = o[db][q4 * 4 + 2] * a0 + other.z * a1;
            o[db][q4 * 4 + 3] = o[db][q4 * 4 + 3] * a0 + other.w * a1;
          }
      }
    }
    if (row_live && wk == 0) {
      if (hi == 0) part_ml[r] = make_float2(m_run, l_run);
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          *reinterpret_cast<float4*>(part_o + r * 128 + db * 32 + 8 * q4 + 4 * hi) =
              make_float4(o[db][q4 * 4 + 0], o[db][q4 * 4 + 1], o[db][q4 * 4 + 2], o[db][q4 * 4 + 3]);
    }
  }
  if (k0 < k1 && sh.odd) {                                  // (read behind the loop's barriers)
    __threadfence_block();
    __syncthreads();
    add_odd_values<kPaged>(p, kvh, b, row0, row0 + 32 * WR < row_end ? row0 + 32 * WR : row_end, k0, k1, part_o, part_ml, starts);
  }
}

// A row block that is at most half full (the last one; a padded batch's only one; a sequence's pages) is taken by WR / 2 x 2 waves, which deal the keys of
// a tile among two: no wave is without rows.
template <int WR, int WK, bool kPaged>
__device__ __forceinline__ void batch_attn_block(const BatchAttnParams& p, int kvh, int b, int64_t row0, int64_t row_end, int k0, int k1, float* part_o,
                                                 float2* part_ml, const int* starts, unsigned char* lds, float* lds_ml, Shared& sh) {
  if constexpr (WK == 1) {
    if (row_end - row0 <= 16 * WR) {
      batch_attn_range<WR / 2, 2, kPaged>(p, kvh, b, row0, row_end, k0, k1, part_o, part_ml, starts, lds, lds_ml, sh);
      return;
    }
  }
  batch_attn_range<WR, WK, kPaged>(p, kvh, b, row0, row_end, k0, k1, part_o, part_ml, starts, lds, lds_ml, sh);
}

// range `split` of n keys cut into `ns` ranges of whole 64-key tiles (the last ones may be empty: k0 >= k1)
__device__ __forceinline__ void key_range(int n, int ns, int split, int& k0, int& k1) {
  const int tiles = (n + 63) / 64, per = (tiles + ns - 1) / ns;
  const int64_t at = (int64_t)split * per * 64, to = at + (int64_t)per * 64;
  k0 = (int)(at < n ? at : n);
  k1 = (int)(to < n ? to : n);
}

// rows of sequence b with this step's, as far as its table goes
__device__ __forceinline__ int stored_rows(const Pages& pg, int b, int n_new) {
  const int64_t len = (int64_t)pg.seq_len[b] + n_new, cap = (int64_t)pg.max_pages * pg.page_size;
  return (int)(len < 0 ? 0 : (len > cap ? cap : len));
}

// Grid: first the workgroups of the pages (short), then those of the prefix.  The row blocks that read the same keys are 8 workgroups apart, so that
// they run on the same XCD (workgroups go to the 8 XCDs in turn) and share its L2.
template <int WR, int WK>
constexpr int lds_of() {
  constexpr int tiles = (WR == 1 ? 1 : Shape<WR, WK>::kBuffers) * 2 * Shape<WR, WK>::TILE * 256, join = WR == 1 ? join_bytes<WK>() : (WK == 1 ? WR / 2 : WR) * 32 * kJoinRow * 4;      // (WK = 1: of the narrow form)
  return join > tiles ? join : tiles;
}
template <int WR, int WK>
__global__ __launch_bounds__(64 * WR * WK, 2) void batch_attn_kernel(BatchAttnParams p) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];          // lds_of<WR, WK>()
  __shared__ float lds_ml[WR == 1 ? WK * 64 : WR * 64];
  __shared__ Shared sh;
  __shared__ int starts[kMaxCompact + 2];
  if (blockIdx.x >= p.page_wgs) {
    const unsigned w = blockIdx.x - p.page_wgs;
    Blocks rows = row_blocks((int64_t)p.batch * p.t_max, p.G, 32 * WR);
    int ns = p.ns;
    if (p.compact) {
      if (threadIdx.x < 64) {                                  // running sum of the counts
        int carry = 0;
        for (int b0 = 0; b0 < p.batch; b0 += 64) {
          const int b = b0 + (int)threadIdx.x, v = b < p.batch ? rows_new(p.pg, b, p.t_max) : 0;
          int incl = v;
          incl += __builtin_amdgcn_update_dpp(0, incl, 0x111, 0xf, 0xf, false);        // row_shr 1, 2, 4, 8; the last lanes of rows, of the lower half
          incl += __builtin_amdgcn_update_dpp(0, incl, 0x112, 0xf, 0xf, false);
          incl += __builtin_amdgcn_update_dpp(0, incl, 0x114, 0xf, 0xf, false);
          incl += __builtin_amdgcn_update_dpp(0, incl, 0x118, 0xf, 0xf, false);
          incl += __builtin_amdgcn_update_dpp(0, incl, 0x142, 0xa, 0xf, false);
          incl += __builtin_amdgcn_update_dpp(0, incl, 0x143, 0xc, 0xf, false);
          if (b < p.batch) starts[b] = carry + incl - v;
          carry += __builtin_amdgcn_readlane(incl, 63);
        }
        rows = row_blocks(carry, p.G, 32 * WR);
        int best = 1;
        if (rows.nrb > kFewBlocks) {                           // each lane a number of ranges
          float cost = ranges_cost(threadIdx.x + 1, rows.nrb, p.prefix_wgs, p.slots, p.hkv, p.ns_max, 32 * WR, (unsigned)((p.P + 63) >> 6));
          best = threadIdx.x + 1;
#pragma unroll
          for (int k = 32; k > 0; k >>= 1) {
            const float c2 = __shfl_xor(cost, k, 64);
            const int b2 = __shfl_xor(best, k, 64);
            if (c2 < cost || (c2 == cost && b2 < best)) { cost = c2; best = b2; }
          }
        } else if (rows.nrb) {
          best = ranges_of_few(rows.nrb, p.once, p.hkv, p.ns_max);
        }
        if (threadIdx.x == 0) { starts[p.batch] = carry; starts[p.batch + 1] = best; }
      }
      __syncthreads();
      rows = row_blocks(starts[p.batch], p.G, 32 * WR);
      ns = starts[p.batch + 1];
      if (w == 0)
        for (int b = threadIdx.x; b <= p.batch + 1; b += 64 * WR * WK) p.starts[b] = starts[b];
    }
    if (rows.nrb == 0) return;
    const unsigned turn = 8u * rows.nrb;
    const int item = (int)(w / turn) * 8 + (int)(w % 8), rb = (int)(w % turn) / 8;
    if (item >= p.hkv * ns) return;
    const int kvh = item / ns, split = item - kvh * ns;
    int k0, k1;
    key_range((int)p.P, ns, split, k0, k1);
    const int64_t slot = ((int64_t)kvh * ns + split) * rows.rows;
    batch_attn_block<WR, WK, false>(p, kvh, 0, (int64_t)rb * 32 * WR, rows.rows, k0, k1, p.pre_o + slot * 128, p.pre_ml + slot, starts, lds, lds_ml, sh);
    return;
  }
  const int w = (int)blockIdx.x;
  const int rb = w % p.nrb2, split = (w / p.nrb2) % p.ns2, hb = w / (p.nrb2 * p.ns2);
  const int kvh = hb % p.hkv, b = hb / p.hkv;
  const int n_new = rows_new(p.pg, b, p.t_max);
  if (n_new == 0) return;                                      // nothing of this sequence is written
  int k0, k1;
  key_range(stored_rows(p.pg, b, n_new), p.ns2, split, k0, k1);
  const int64_t seq_row0 = (int64_t)b * p.t_max * p.G, row0 = seq_row0 + (int64_t)rb * 32 * WR, row_end = seq_row0 + (int64_t)n_new * p.G;
  if (row0 >= row_end) return;
  const int64_t slot = ((int64_t)kvh * p.ns2 + split) * p.R;
  batch_attn_block<WR, WK, true>(p, kvh, b, row0, row_end, k0, k1, p.part_o + slot * 128, p.part_ml + slot, nullptr, lds, lds_ml, sh);
}

// Few keys: ONE launch.  The 8 waves of a workgroup deal the prefix's and the pages' 32-key blocks among themselves for the (at most 32) rows of one
// sequence and kv head and join their results; the prefix is read again for every sequence, from L2.
constexpr int kDirectWaves = 8, kDirectLds = join_bytes<kDirectWaves>();
static_assert(kDirectLds >= 2 * Shape<1, kDirectWaves>::TILE * 256, "the tiles fit as well");

__global__ __launch_bounds__(64 * kDirectWaves, 2) void batch_attn_direct_kernel(BatchAttnParams p) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  __shared__ float lds_m[kDirectWaves * 32], lds_l[kDirectWaves * 32];
  __shared__ Shared sh;
  const int tid = threadIdx.x, l31 = tid & 31;
  const int kvh = (int)(blockIdx.x % p.hkv), b = (int)(blockIdx.x / p.hkv);
  const int n_new = rows_new(p.pg, b, p.t_max);
  if (n_new == 0) return;
  const int len = stored_rows(p.pg, b, n_new);
  const int64_t row0 = (int64_t)b * p.t_max * p.G, row_end = row0 + (int64_t)n_new * p.G, r = row0 + l31;
  const bool row_live = r < row_end;
  bf16x8_t qf[8];
  Rows st;
  begin_rows(p, kvh, row_live ? r / p.G : 0, row_live ? (int)(r % p.G) : 0, row_live, qf, sh, st);
  __syncthreads();                                             // flags cleared
  const int wave = tid >> 6, blocks = ((int)p.P + 31) / 32;
  walk_alone<kDirectWaves, false>(p, kvh, b, r, row_live, qf, 0, (int)p.P, wave, lds, sh, st);
  walk_alone<kDirectWaves, true>(p, kvh, b, r, row_live, qf, 0, len, (wave - blocks) & (kDirectWaves - 1), lds, sh, st);   // the pages go on where the prefix ended
  __syncthreads();                                             // the blocks are read: their LDS joins the rows
  float* obuf = reinterpret_cast<float*>(lds);
  lay_out_rows<kDirectWaves>(st, p.c, row_live, obuf, lds_m, lds_l);
  const int64_t slot0 = (int64_t)kvh * p.R;
  const bool odd = sh.odd != 0;
  for (int pass = 0; pass < 2; ++pass) {                       // second pass only behind add_odd_values, from where it left the rows
    for (int i = tid; i < (int)(row_end - row0) * 32; i += 64 * kDirectWaves) {
      const int row = i >> 5, d4 = (i & 31) * 4;
      float m, l;
      float4 acc = joined<kDirectWaves>(obuf, lds_m, lds_l, row, d4, m, l);
      if (pass) acc = *reinterpret_cast<const float4*>(p.part_o + (slot0 + row0 + row) * 128 + d4);
      if (pass == 0 && odd) {
        *reinterpret_cast<float4*>(p.part_o + (slot0 + row0 + row) * 128 + d4) = acc;
        if (d4 == 0) p.part_ml[slot0 + row0 + row] = make_float2(m, l);
        continue;
      }
      uint2 y = make_uint2(0, 0);                              // a row that sees no key is zero
      if (l != 0.f) {
        const float inv = 1.0f / l;
        y.x = (unsigned)f32_to_bf16_bits(acc.x * inv) | ((unsigned)f32_to_bf16_bits(acc.y * inv) << 16);
        y.y = (unsigned)f32_to_bf16_bits(acc.z * inv) | ((unsigned)f32_to_bf16_bits(acc.w * inv) << 16);
      }
      const int64_t bt = (row0 + row) / p.G;
      const int g = (int)(row0 + row - bt * p.G);
      *reinterpret_cast<uint2*>(p.out + ((bt * p.hq) + (int64_t)kvh * p.G + g) * 128 + d4) = y;
    }
    if (!odd) break;
    if (pass == 0) {
      __threadfence_block();
      __syncthreads();
      add_odd_values<false>(p, kvh, b, row0, row_end, 0, (int)p.P, p.part_o + slot0 * 128, p.part_ml + slot0, nullptr);       // (compact is off: rows as they are)
      add_odd_values<true>(p, kvh, b, row0, row_end, 0, len, p.part_o + slot0 * 128, p.part_ml + slot0, nullptr);           // (a row's thread is the same in both)
      __threadfence_block();
      __syncthreads();
    }
  }
}

// Joins the partial results of a row.  kWide: a workgroup per row, 8 groups of 32 lanes walk the parts (16 B of the row per lane), the
// weights are found once, in LDS, so that no load waits for another; otherwise (few parts, many rows) a wave per row.
constexpr int kMaxParts = 1280;
template <bool kWide>
__global__ __launch_bounds__(256) void batch_combine_kernel(BatchAttnParams p) {
  constexpr int GROUPS = kWide ? 8 : 2;
  __shared__ float4 lds_o[4][32];
  __shared__ float red[8];
  __shared__ int red_faint[4];
  __shared__ float lds_a[kWide ? kMaxParts : 1];               // < 0: an empty range, which left no o behind
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lane32 = tid & 31, grp = kWide ? tid >> 5 : (tid >> 5) & 1;
  const int64_t w = kWide ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (w >= p.R * p.hkv) return;                                // (whole waves)
  const int kvh = (int)(w / p.R);
  const int64_t r = w - (int64_t)kvh * p.R, bt = r / p.G;
  const int g = (int)(r - bt * p.G), b = (int)(bt / p.t_max), t = (int)(bt % p.t_max);
  if (t >= rows_new(p.pg, b, p.t_max)) return;                 // rows behind a sequence's last token stay as they are
  // parts 0 .. ns - 1: the prefix, row `live`; parts ns ...: the pages, row r
  int64_t pre_rows = p.R, live = r;
  int ns = p.ns;
  if (p.compact) { pre_rows = (int64_t)p.starts[p.batch] * p.G; live = (int64_t)(p.starts[b] + t) * p.G + g; ns = p.starts[p.batch + 1]; }
  const int np = ns + p.ns2;
  const float2 *ml0 = p.pre_ml + (int64_t)kvh * ns * pre_rows + live, *ml1 = p.part_ml + (int64_t)kvh * p.ns2 * p.R + r;
  const float *po0 = p.pre_o + ((int64_t)kvh * ns * pre_rows + live) * 128 + lane32 * 4, *po1 = p.part_o + ((int64_t)kvh * p.ns2 * p.R + r) * 128 + lane32 * 4;
  auto ml = [&](int i) { return i < ns ? ml0[(int64_t)i * pre_rows] : ml1[(int64_t)(i - ns) * p.R]; };
  auto po = [&](int i) { return *reinterpret_cast<const float4*>(i < ns ? po0 + (int64_t)i * pre_rows * 128 : po1 + (int64_t)(i - ns) * p.R * 128); };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  if (kWide) {
    // eight parts of a group in flight, the first ones asked for before their weights are known (28 rows 15.4 -> 14.9 us in all; the form below,
    // with many rows under way at once, loses by it: 61 -> 62.5)
    float4 v[8];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k * GROUPS < np) v[k] = po(i0 + k * GROUPS);
    };
    fetch(grp);
    float M = -1e30f;
    for (int i = tid; i < np; i += 256) M = fmaxf(M, ml(i).x);
    M = wave_max_f32(M);
    if (lane == 0) red[wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    bool faint = false;
    for (int i = tid; i < np; i += 256) {
      const float2 x = ml(i);
      const float a = __builtin_amdgcn_exp2f((x.x - M) * p.c);
      lds_a[i] = x.y == 0.f ? -1.f : a;
      faint |= x.y != 0.f && a < kTiny;
      l = __builtin_fmaf(x.y, a, l);
    }
    l = wave_sum_f32(l);
    const bool any_faint = __any(faint);
    if (lane == 0) { red[4 + wave] = l; red_faint[wave] = any_faint; }
    __syncthreads();
    l = (red[4] + red[5]) + (red[6] + red[7]);
    auto join = [&](auto faint_ones) {
      for (int i0 = grp; i0 < np; i0 += GROUPS * 8) {
        if (i0 != grp) fetch(i0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int i = i0 + k * GROUPS;
          const float a = i < np ? lds_a[i] : -1.f;
          if (a >= 0.f) add_part<decltype(faint_ones)::value>(acc, v[k], a);           // (what an empty range holds is not looked at)
        }
      }
    };
    if (red_faint[0] | red_faint[1] | red_faint[2] | red_faint[3]) join(std::true_type{}); else join(std::false_type{});
  } else {                                                     // np <= 64: lane i holds part i
    const float2 x = lane < np ? ml(lane) : make_float2(-1e30f, 0.f);
    float M = x.x;
    M = wave_max_f32(M);
    const float a = __builtin_amdgcn_exp2f((x.x - M) * p.c);
    l = wave_sum_f32(x.y * a);
    const unsigned long long seen = __ballot(x.y != 0.f);      // (an empty range left no o behind)
    auto join = [&](auto faint_ones) {
      for (int i0 = 0; i0 < np; i0 += GROUPS * 4) {
        float4 v[4];
        float ak[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = i0 + k * GROUPS + grp;
          const bool has = i < np && ((seen >> (i & 63)) & 1);
          ak[k] = __shfl(a, i & 63, 64);
          if (!has) ak[k] = 0.f;
          v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (has) v[k] = po(i);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) add_part<decltype(faint_ones)::value>(acc, v[k], ak[k]);
      }
    };
    if (__any(x.y != 0.f && a < kTiny)) join(std::true_type{}); else join(std::false_type{});
  }
  acc.x = xhalf_sum(acc.x); acc.y = xhalf_sum(acc.y); acc.z = xhalf_sum(acc.z); acc.w = xhalf_sum(acc.w);
  if (kWide) {
    if (lane < 32) lds_o[wave][lane32] = acc;
    __syncthreads();
    if (tid >= 32) return;
    const float4 v1 = lds_o[1][lane32], v2 = lds_o[2][lane32], v3 = lds_o[3][lane32];
    acc.x = (acc.x + v1.x) + (v2.x + v3.x); acc.y = (acc.y + v1.y) + (v2.y + v3.y);
    acc.z = (acc.z + v1.z) + (v2.z + v3.z); acc.w = (acc.w + v1.w) + (v2.w + v3.w);
  } else if (lane >= 32) {
    return;
  }
  uint2 y = make_uint2(0, 0);                                  // a row that sees no key is zero
  if (l != 0.f) {
    const float inv = 1.0f / l;
    y.x = (unsigned)f32_to_bf16_bits(acc.x * inv) | ((unsigned)f32_to_bf16_bits(acc.y * inv) << 16);
    y.y = (unsigned)f32_to_bf16_bits(acc.z * inv) | ((unsigned)f32_to_bf16_bits(acc.w * inv) << 16);
  }
  *reinterpret_cast<uint2*>(p.out + ((bt * p.hq) + (int64_t)kvh * p.G + g) * 128 + lane32 * 4) = y;
}

struct Plan {
  int wr, ns2, nrb2, ns_max, ns;
  int64_t R;
  unsigned prefix_wgs, once, slots;
  bool direct, compact, many_parts;
};

// kDirectKeys: one launch against two, us, one sequence (sixteen), 28 query and 4 kv heads, up to 96 keys of the pages: 300 keys 9.8 against 11.0 (10.1,
// 11.5), 400 10.5 against 11.0 (10.9, 11.8), 500 11.9 against 11.0 (12.0, 11.9), 600 11.7 against 11.1 (12.7, 12.0), 1000 15.0 against 11.0; 64 and 8
// heads, 3 x 4 padded tokens, 500 keys 12.0 against 13.4, 800 14.9 against 13.2.
// kOneTile, keys x heads x 32-row tiles of the batch below which blocks of one tile win: about a workgroup for each CU and 256 keys.  us with one tile and two:
// 28 rows over 8000 keys of 4 heads 12.6, 12.9, over 11535 13.55, 13.35, over 16000 16.4, 14.6; 56 rows over 4100 12.5, 13.6, over 11535 15.9, 14.8; 448 rows
// over 1000 14.7, 15.6, over 1500 21.3, 16.2; 32 rows over 24000 of 2 heads 14.6 both, over 32000 16.5, 15.3; 64 rows over 3000 of 8 13.3, 14.4, over 6000
// 16.7, 15.6.  Not beyond kOneTileRows: 672 rows over 700 18.6, 16.5, 1400 over 100 26.8, 21.8.  Where a sequence has more rows than a tile its pages are read
// several times, kOneTilePages keys x tiles at most: 3 x 6 padded tokens with 40 keys of their own over 2000 keys 13.0, 14.2, 8 x 6 with 1000 over 700 39.5, 24.4.
// kShort, keys x heads below which a workgroup of many rows has few tiles: see the table at make_plan().
// kLeastKeys of a range, 64 / 128 / 192 / 256 / 384 / 512, us: 28 rows over 11535 keys 16.1 / 15.4 / 13.4 / 13.7 / 14.5 / 16.8, over 4100 14.0 / 12.0 / 11.7 /
// 12.0 / 13.5 / 15.0, 8 x 8 padded tokens over 4100 22.5 / 21.8 / 19.2 / 17.4 / 17.7 / 19.2, 672 rows over 768 keys 20.2 / 20.3 / 18.0 / 17.6 / 19.4 / 19.4:
// fewer parts to join.
// kFewRows, rows x heads up to which a workgroup joins a row, against a wave, us in all: 28 x 4 over 11535 keys 13.6 against 16.6, 56 x 4 over 504015 186
// against 195, 112 x 4 over 32785 28.3 against 30.7, 224 x 4 over 11535 24.2 against 24.7, 336 x 4 33.8 against 31.8, 1008 x 4 over 32785 126 against 119.
constexpr int64_t kDirectKeys = 640, kOneTile = 60 << 10, kOneTileRows = 512, kOneTilePages = 24 << 10, kShort = 65536, kFewRows = 1024, kLeastKeys = 256;

// ranges of a sequence's pages: `keys` each, fewer ranges where sequences fill the card
int page_ranges(int64_t wgs, int64_t seqs, int64_t suffix_cap, int most, int64_t keys) {
  int64_t ns2 = wgs / seqs;
  const int64_t by_keys = (suffix_cap + keys - 1) / keys;
  if (ns2 > by_keys) ns2 = by_keys;
  return (int)(ns2 < 1 ? 1 : (ns2 > most ? most : ns2));
}

// padded: n_new is given, so that tokens may be missing
Plan make_plan(const qp_ctx* ctx, int batch, int t_max, bool padded, int64_t P, int64_t suffix_cap, int hq, int hkv) {
  Plan pl = {};
  const int G = hq / hkv;
  const int64_t tokens = (int64_t)batch * t_max;
  pl.R = tokens * G;
  if (t_max * G <= 32 && (int64_t)hkv * batch <= ctx->cus && P + suffix_cap <= kDirectKeys) {
    pl.direct = true;
    pl.ns2 = 1;
    return pl;
  }
  // Key ranges times row blocks.  Wide row blocks read the keys less often, narrow ones waste less on rows that are not there (the pages' workgroups
  // hold one sequence each) and start faster.  us with row blocks of 32 / 64 / 128 / 256 rows, 28 query and 4 kv heads:
  //                                    4100 keys                      32785 keys
  //     4 x 1 token,   28 rows         12.0 / 12.4 / 12.5 / 14.0      21.9 / 20.3 / 20.3 / 21.9
  //    16 x 1,        112 rows         15.1 / 14.8 / 16.9 / 18.1      33.0 / 28.7 / 31.3 / 28.6
  //    64 x 1,        448 rows         28.1 / 27.0 / 27.1 / 34.4      83.6 / 60.4 / 62.9 / 64.2
  //    32 x 4,        896 rows         38.9 / 34.9 / 33.6 / 38.0     155   / 111  / 101  / 102
  //     8 x 64 padded, 1701, 2135      59.1 / 47.6 / 51.3 / 53.9     373   / 246  / 225  / 221
  //    16 x 24,      2688 rows         86.0 / 62.6 / 57.4 / 56.6     431   / 281  / 259  / 273
  //     8 x 128,     7168 rows          187 / 135  / 119  / 119     1039   / 762  / 697  / 652
  // (77 live rows of 144 over 30737 keys of 8 heads: 43.6 / 39.2 / 40.3 / 36.1; 56 rows over 504015: 219 / 186 / 188 / 198.)
  pl.compact = padded && t_max > 1 && batch <= kMaxCompact && P > 0;
  const int64_t tiles = (pl.R + 31) / 32, seq_rows = (int64_t)t_max * G;
  const bool one_tile = seq_rows <= 32 ? pl.R <= kOneTileRows : pl.R <= 128 && hkv * batch * ((seq_rows + 31) / 32) * suffix_cap <= kOneTilePages;
  if (one_tile && P * hkv * tiles < kOneTile) pl.wr = 1;
  else if (P * hkv < kShort) pl.wr = pl.R <= 2048 ? 2 : 4;
  else pl.wr = pl.R <= 64 || (!pl.compact && pl.R <= 512) ? 2 : 8;
  const int rows = 32 * pl.wr, per_cu = pl.wr == 8 ? 1 : 2;     // resident workgroups (registers: two waves per SIMD)
  const int64_t nrb = (pl.R + rows - 1) / rows, slots = (int64_t)per_cu * ctx->cus;
  pl.nrb2 = (int)(((int64_t)t_max * G + rows - 1) / rows);
  const int64_t seqs = (int64_t)hkv * batch * pl.nrb2;
  // A page's key costs about twice a prefix's (two loads one behind the other, no tile ahead): no workgroup of the pages runs longer than one of the prefix.
  const int64_t even = P * hkv * nrb / slots / 2;
  pl.ns2 = page_ranges(slots / 4, seqs, suffix_cap, 32, even > 256 ? even : 256);
  if (P > 0) {
    const int64_t page_wgs = seqs * pl.ns2, left = page_wgs * 2 < slots ? slots - page_wgs : slots;
    const int64_t most = (P + kLeastKeys - 1) / kLeastKeys, all = (hkv + 7) / 8 * 8 * nrb, places = nrb > kFewBlocks ? 3 * slots : left;
    pl.once = (unsigned)left;
    pl.slots = (unsigned)slots;
    pl.prefix_wgs = (unsigned)(places > all ? places : all);
    pl.many_parts = pl.R * hkv <= kFewRows;                    // a workgroup joins any number of parts, a wave 64 at most
    const int cap = pl.many_parts ? kMaxParts - 32 : 64 - pl.ns2;
    pl.ns_max = (int)(most < cap ? most : cap);
    pl.ns = nrb > kFewBlocks ? 1 : ranges_of_few((unsigned)nrb, pl.once, hkv, pl.ns_max);
    if (nrb > kFewBlocks) {
      auto cost = [&](unsigned ns) { return ranges_cost(ns, (unsigned)nrb, pl.prefix_wgs, pl.slots, hkv, pl.ns_max, (unsigned)rows, (unsigned)((P + 63) / 64)); };
      for (int ns = 2; ns <= 64; ++ns)
        if (cost(ns) < cost(pl.ns)) pl.ns = ns;
    }
  }
  return pl;
}

// where things lie in the workspace
struct Layout { size_t pre_o, pre_ml, part_o, part_ml, starts, end; };
Layout layout_of(const Plan& pl, int batch, int hkv) {
  Layout l;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t a = at; at += (bytes + 255) & ~(size_t)255; return a; };
  const size_t pages = (size_t)hkv * pl.ns2 * pl.R, prefix = (size_t)pl.prefix_wgs * 32 * pl.wr;       // hkv * ns * live rows <= workgroups * block rows
  l.pre_o = take(prefix * 512); l.pre_ml = take(prefix * sizeof(float2));
  l.part_o = take(pages * 512); l.part_ml = take(pages * sizeof(float2));
  l.starts = take(pl.compact ? ((size_t)batch + 2) * sizeof(int) : 0);
  l.end = at;
  return l;
}

// grids x threads below 2^32, as a launch takes them (the direct form has a workgroup per CU at most)
bool launches(const Plan& pl, int batch, int hkv) {
  if (pl.direct) return true;
  const int64_t threads = pl.wr == 8 ? 512 : 256, pages = (int64_t)hkv * batch * pl.nrb2 * pl.ns2, join = pl.many_parts ? pl.R * hkv : (pl.R * hkv + 3) / 4;
  return (pages + pl.prefix_wgs) * threads < (1LL << 32) && join * 256 < (1LL << 32);
}

Pages pages_of(const int32_t* table, const int32_t* seq_len, const int32_t* n_new, int max_pages, int n_pages, int page_size, int64_t page_stride) {
  Pages pg;
  pg.table = table; pg.seq_len = seq_len; pg.n_new = n_new;
  pg.max_pages = max_pages; pg.n_pages = n_pages; pg.page_size = page_size; pg.page_stride16 = page_stride / 8;
  return pg;
}

template <int WR, int WK>
int launch_ranges(const BatchAttnParams& p, unsigned grid, hipStream_t s) {
  constexpr int bytes = lds_of<WR, WK>();
  if (bytes > 60 * 1024) {
    static std::atomic<unsigned long long> opted{0};
    int rc = qp_opt_in_lds(opted, (const void*)batch_attn_kernel<WR, WK>, bytes, "batch_attn");
    if (rc) return rc;
  }
  batch_attn_kernel<WR, WK><<<grid, 64 * WR * WK, bytes, s>>>(p);
  return qp_check_launch("batch_attn");
}

}  // namespace

int qp_launch_batch_rope_append(const void* qkv, const void* cos, const void* sin, int batch, int t_max, const int32_t* seq_len, const int32_t* n_new,
                                int hq, int hkv, void* q_out, void* k_pages, void* v_pages, int64_t page_stride, int n_pages, int page_size,
                                const int32_t* table, int max_pages, hipStream_t s) {
  const int head_blocks = (hq + 2 * hkv + 15) / 16;
  const int64_t grid = (int64_t)batch * t_max * head_blocks;
  batch_rope_append_kernel<<<(unsigned)grid, 256, 0, s>>>((const uint4*)qkv, (const uint4*)cos, (const uint4*)sin,
                                                          pages_of(table, seq_len, n_new, max_pages, n_pages, page_size, page_stride), t_max, hq, hkv,
                                                          head_blocks, (uint4*)q_out, (uint4*)k_pages, (uint4*)v_pages);
  return qp_check_launch("batch_rope_append");
}

// 0: a launch would have 2^32 threads or more
size_t qp_batch_attn_workspace_bytes_impl(const qp_ctx* ctx, int batch, int t_max, int64_t P, int64_t suffix_cap, int hq, int hkv) {
  size_t most = 0;
  for (bool padded : {false, true}) {
    const Plan pl = make_plan(ctx, batch, t_max, padded, P, suffix_cap, hq, hkv);
    if (!launches(pl, batch, hkv)) return 0;
    const size_t bytes = layout_of(pl, batch, hkv).end;
    if (bytes > most) most = bytes;
  }
  return most;
}

int qp_launch_batch_attn(const qp_ctx* ctx, const void* q, const void* k_prefix, const void* v_prefix, int64_t prefix_head_stride, int64_t P,
                         const void* k_pages, const void* v_pages, int64_t page_stride, int n_pages, int page_size, const int32_t* table, int max_pages,
                         const int32_t* seq_len, const int32_t* n_new, int batch, int t_max, int hq, int hkv, float scale, void* out, void* workspace,
                         hipStream_t s) {
  const Plan pl = make_plan(ctx, batch, t_max, n_new != nullptr, P, (int64_t)max_pages * page_size, hq, hkv);
  const Layout l = layout_of(pl, batch, hkv);
  char* ws = (char*)workspace;
  BatchAttnParams p = {};
  p.q = (const uint4*)q; p.out = (uint16_t*)out;
  p.k_pre = (const uint4*)k_prefix; p.v_pre = (const uint4*)v_prefix; p.pre_hs16 = prefix_head_stride / 8; p.P = P;
  p.k_pages = (const uint4*)k_pages; p.v_pages = (const uint4*)v_pages;
  p.pg = pages_of(table, seq_len, n_new, max_pages, n_pages, page_size, page_stride);
  p.batch = batch; p.t_max = t_max; p.hq = hq; p.hkv = hkv; p.G = hq / hkv; p.c = scale * 1.4426950408889634f;
  p.R = pl.R; p.prefix_wgs = pl.prefix_wgs; p.once = pl.once; p.slots = pl.slots; p.ns_max = pl.ns_max; p.ns = pl.ns; p.compact = pl.compact;
  p.pre_o = (float*)(ws + l.pre_o); p.pre_ml = (float2*)(ws + l.pre_ml);
  p.part_o = (float*)(ws + l.part_o); p.part_ml = (float2*)(ws + l.part_ml);
  p.starts = (int*)(ws + l.starts);
  p.ns2 = pl.ns2; p.nrb2 = pl.nrb2;
  p.page_wgs = (unsigned)((int64_t)hkv * batch * pl.nrb2 * pl.ns2);
  int rc;
  if (pl.direct) {
    static std::atomic<unsigned long long> opted{0};
    if ((rc = qp_opt_in_lds(opted, (const void*)batch_attn_direct_kernel, kDirectLds, "batch_attn_direct"))) return rc;
    batch_attn_direct_kernel<<<(unsigned)(hkv * batch), 64 * kDirectWaves, kDirectLds, s>>>(p);
    return qp_check_launch("batch_attn(direct)");
  }
  const unsigned grid = p.page_wgs + pl.prefix_wgs;
  switch (pl.wr) {
    case 1: rc = launch_ranges<1, 4>(p, grid, s); break;
    case 2: rc = launch_ranges<2, 2>(p, grid, s); break;
    case 4: rc = launch_ranges<4, 1>(p, grid, s); break;
    default: rc = launch_ranges<8, 1>(p, grid, s); break;
  }
  if (rc) return rc;
  if (pl.many_parts) batch_combine_kernel<true><<<(unsigned)(pl.R * hkv), 256, 0, s>>>(p);
  else batch_combine_kernel<false><<<(unsigned)((pl.R * hkv + 3) / 4), 256, 0, s>>>(p);
  return qp_check_launch("batch_attn(combine)");
}
