// Attention of one new token of each of many sequences over a paged key-value cache: the pages of sequence b are the entries of its row of
// the block table, its length is on the device, and no two need be alike.  The counterpart for a pool of pages of decode_attn.cu, whose
// sequences share one position (reference ops/decode_attn.go:64-170).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(s_j - max_i s_i),   s_j = scale q . k_j, or cap tanh(scale q . k_j / cap),   max(0, n - window) <= j < n
//
// No key (a row of the batch that no sequence has), or none whose score is above -inf: o = 0.  A key on a page outside the pool counts as
// absent and is reported.
#include "paged.cuh"

namespace lb {
namespace {

__device__ unsigned int g_attn_status = 0;

constexpr float LOG2E = 1.4426950408889634f;

struct PagedArgs {
  const void *q, *k, *v;
  void *out;
  const int *table, *lens;
  long long q_s[2], ks[3], vs[3], table_stride, pages;  // strides in elements: q token, head; cache page, head, row
  int B, NH, KH, G, D, W, window;
  float scale, softcap;
  FastDiv page;
};

// the valid keys of a sequence: [first, n)
__device__ __forceinline__ int length_of(const PagedArgs &a, int b) {
  const int n = a.lens[b];
  return min(max(n, 0), a.W * a.page.d);
}
__device__ __forceinline__ int first_of(const PagedArgs &a, int n) { return a.window > 0 ? max(0, n - a.window) : 0; }

__device__ __forceinline__ float ex2(float x) {  // relative error 2^-22; results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// A score in units of log2 e.  tanh z = 1 - 2 / (e^(2 z) + 1), whose absolute error is a few 2^-24: nothing for a z of the order of 1, but scores far
// below the cap would lose cap 2^-23 of themselves; below 0.35 its Taylor series to z^9 instead (the next term is 2^-22 of z there).
struct Scorer {
  float sc, cap;  // without a cap: scale log2 e; with one, of 1e-20 to 1e20 (neither overflows): scale / cap, and cap log2 e
  __device__ Scorer(float scale, float softcap) : sc(softcap > 0.f ? scale / softcap : scale * LOG2E), cap(softcap * LOG2E) {}
  __device__ __forceinline__ float operator()(float dot) const { return cap > 0.f ? capped(dot * sc) : dot * sc; }
  static constexpr float NEAR = 0.35f;
  __device__ __forceinline__ static float near_of(float z) {
    const float y = z * z;
    return z * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  }
  __device__ __forceinline__ float capped(float z) const {
    const float far = 1.f - 2.f * __fdividef(1.f, ex2(z * (2.f * LOG2E)) + 1.f);
    return cap * (fabsf(z) < NEAR ? near_of(z) : far);
  }
  template <int N>  // (33 sequences with a window and a cap: 20.6 -> 19.7 us, where all of a warp's scores are below 0.35 of the cap)
  __device__ __forceinline__ void cap_all(float (&z)[N][4]) const {  // of the whole warp
    bool small = true;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) small = small && fabsf(z[i][e]) < NEAR;
    if (__all_sync(0xffffffffu, small)) {
#pragma unroll
      for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) z[i][e] = cap * near_of(z[i][e]);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) z[i][e] = capped(z[i][e]);
    }
  }
};

// ------------------------------------------------------------------------------------ any head size, any stride
// What the kernels below do not take: head sizes that are not whole 16s, cache rows off 16 bytes, strides whose offsets do not fit 32 bits.  A
// CTA takes a query head, its four warps every fourth key, a lane every 32nd dim; a chain of a key's latencies bounds it (64 ragged
// sequences to 8192 keys, 8 KV heads of 128 under 32: 2.96 ms, where the kernel below takes 45 us).
constexpr int PL_WARPS = 4, PL_MAX_D = 256;

template <typename T>
__global__ void __launch_bounds__(PL_WARPS * 32) paged_attn_any_kernel(PagedArgs a) {
  constexpr int P = PL_MAX_D / 32;
  __shared__ float part[PL_WARPS][PL_MAX_D + 2];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.x / a.NH, h = blockIdx.x - b * a.NH, kh = h / a.G;
  const int n = length_of(a, b), j0 = first_of(a, n);
  unsigned odd = a.lens[b] != n ? PAGED_LENGTH : 0;
  const T *q = static_cast<const T *>(a.q) + b * a.q_s[0] + h * a.q_s[1];
  const T *k = static_cast<const T *>(a.k) + kh * a.ks[1], *v = static_cast<const T *>(a.v) + kh * a.vs[1];
  const Scorer score(a.scale, a.softcap);
  float qf[P], acc[P], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < P; i++) acc[i] = 0.f, qf[i] = lane + 32 * i < a.D ? to_f32(q[lane + 32 * i]) : 0.f;
  for (int j = j0 + warp; j < n; j += PL_WARPS) {
    const int w = a.page.div(j), r = j - w * a.page.d, pg = a.table[b * a.table_stride + w];
    if (pg < 0 || pg >= a.pages) {
      odd |= PAGED_PAGE;
      continue;
    }
    const T *kr = k + pg * a.ks[0] + r * a.ks[2], *vr = v + pg * a.vs[0] + r * a.vs[2];
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < P; i++)
      if (lane + 32 * i < a.D) d = fmaf(qf[i], to_f32(kr[lane + 32 * i]), d);
    const float s = score(warp_sum(d)), mx = fmaxf(m, s), use = mx == -INFINITY ? 0.f : mx;
    const float corr = ex2(m - use), p = ex2(s - use);
    m = mx, l = fmaf(l, corr, p);
#pragma unroll
    for (int i = 0; i < P; i++)
      if (lane + 32 * i < a.D) acc[i] = fmaf(p, to_f32(vr[lane + 32 * i]), acc[i] * corr);
  }
  if (lane == 0) part[warp][0] = m, part[warp][1] = l;
#pragma unroll
  for (int i = 0; i < P; i++) part[warp][2 + lane + 32 * i] = acc[i];
  if (odd && lane == 0) atomicOr(&g_attn_status, odd);
  __syncthreads();
  float top = -INFINITY, L = 0.f;
#pragma unroll
  for (int w = 0; w < PL_WARPS; w++) top = fmaxf(top, part[w][0]);
  if (top == -INFINITY) top = 0.f;
#pragma unroll
  for (int w = 0; w < PL_WARPS; w++) L = fmaf(ex2(part[w][0] - top), part[w][1], L);
  for (int d = threadIdx.x; d < a.D; d += PL_WARPS * 32) {
    float A = 0.f;
#pragma unroll
    for (int w = 0; w < PL_WARPS; w++) A = fmaf(ex2(part[w][0] - top), part[w][2 + d], A);
    static_cast<T *>(a.out)[(long long)blockIdx.x * a.D + d] = from_f32<T>(L == 0.f ? 0.f : A / L);
  }
}

// ------------------------------------------------------------------------------------ rows on 16 bytes, head sizes of whole 16s
// The caches are read once (2 n KH D elements) and everything else is small, so the kernel is a stream: what it does is keep loads in
// flight on every SM whatever the lengths are.
//   * Work is cut evenly.  A unit is a sequence's KV head (with up to 16 of its query heads); its keys come in blocks of 16 rows (f32: 8).
//     All blocks of all units in order are dealt to the warps in runs of equal cost, a long sequence over many, many short ones to one; what a
//     unit costs beside its blocks counts as UNIT of them.  Every CTA scans the lengths for itself.
//   * A warp is on its own: it copies its blocks of keys and values into a ring of its own by 16-byte asynchronous copies, the next
//     blocks' page numbers being read meanwhile, folds them into a running (max, sum, sum p v), and writes a unit out that it holds whole.  Rows
//     without a key are filled with zeros: a weight of 0 times what lies there must not be NaN.
//   * Pieces of a unit that was cut are joined in their order, first those of a CTA's warps at its end, in shared memory; what goes on
//     over CTAs goes to scratch, at most two pieces a CTA, and a second launch joins those: no atomics, the same bits every time.
// Bound by the memory where sequences are long: one of 131072 keys (537 MB, bf16) 89 us, 6.1 TB/s; eight of 8192 in f32 (537 MB) 90 us.  Of
// shorter ones by what a launch costs beside its stream: 64 ragged ones (232 MB) 45 us, of which about 6 are the chain of lengths,
// schedule, pages and first rows (2000 + 1500 + 2000 + 2500 cycles) and 4 the join.
//   * One wave of CTAs: two, three and four waves of finer runs take 98, 102 and 108 us for the one long sequence, each wave that chain again.
//   * UNIT 3.  1, 2, 3, 5, 8 give (us) 50.8, 44.2, 44.3, 44.9, 45.0 for the 64; 18.3, 17.2, 17.7, 20.5, 23.8 for 200 of 300 keys at most; 22.2, 21.3, 20.9,
//     20.4, 20.3 for 33 in f16 with a window; the same for the long ones.  So 2 is the better by 3 % for short sequences, and worse by 2 % under a window.
//   * All four warps of a CTA on the blocks of one unit in turn, with barriers, took 75 us for the 64: two microseconds a unit.
constexpr int PA_WARPS = 4, PA_THREADS = PA_WARPS * 32, UNIT = 3, CLUSTER_BLOCKS = 4, CLUSTER_WIDE = 8;

struct SplitArgs {
  PagedArgs p;
  int hpg, groups;    // query heads per unit, units per KV head
  uint32_t ku[3], vu[3], unit;  // the cache's strides in units of so many bytes, in which every row's offset has 32 bits
  bool alike;         // ku == vu
  int4 *heads;        // per CTA, of the unit that begins there and goes on: sequence, first query head, heads, pieces (0: none)
  float *ml, *acc;    // [2 CTAs][HEADS][2], [2 CTAs][HEADS][D]
};

// 16-byte chunk c of row r of a block lies at chunk c ^ spread(r): eight rows of one chunk on all banks (ldmatrix)
__device__ __forceinline__ int spread(int r) { return (r & 1) << 2 | (r >> 1 & 3); }

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {  // of an 8 x 8 matrix of 16-bit elements held by the warp
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) { mma16816(d, a[0], a[1], a[2], a[3], b0, b1); }
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two weights as 16-bit elements; a and b become what they were rounded to
__device__ __forceinline__ uint32_t pack(float &a, float &b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  a = f.x, b = f.y;
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack(float &a, float &b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  const uint32_t v = *reinterpret_cast<const uint32_t *>(&h);
  a = __uint_as_float(v << 16), b = __uint_as_float(v & 0xFFFF0000u);
  return v;
}

__device__ __forceinline__ float lds_f16(uint32_t addr) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(v) : "r"(addr) : "memory");
  return __half2float(__ushort_as_half(v));
}

// Two weights, 0 or above, as a high and a low 16-bit element each that sum to them: high is less than the weight by 2^-16 of it or more, so that the
// low one has the same sign and is 0 only with it (a value of infinity keeps its sign under both), and by 2^-7 (f16: 2^-10) at most, of which the low one
// keeps all but 2^-8 (2^-11).  (f16: elements lie 2^-24 apart at least.)
__device__ __forceinline__ void halves(float a, float b, uint32_t &hi, uint32_t &lo, __nv_bfloat16) {
  const uint32_t x = __float_as_uint(a * (1.f - 0x1p-16f)), y = __float_as_uint(b * (1.f - 0x1p-16f));
  hi = __byte_perm(x, y, 0x7632);  // (cut off)
  a -= __uint_as_float(x & 0xFFFF0000u), b -= __uint_as_float(y & 0xFFFF0000u);
  lo = pack(a, b, __nv_bfloat16());
}
__device__ __forceinline__ void halves(float a, float b, uint32_t &hi, uint32_t &lo, __half) {
  const float x = fmaf(a, 1.f - 0x1p-16f, -0x1p-24f), y = fmaf(b, 1.f - 0x1p-16f, -0x1p-24f);
  asm("cvt.rz.relu.f16x2.f32 %0, %1, %2;\n" : "=r"(hi) : "f"(y), "f"(x));
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
  a -= f.x, b -= f.y;
  lo = pack(a, b, __half());
}

// bf16 / f16: a block of 16 keys on mma.sync (m16n8k16, f32 sums).  tcgen05 has no use here: its smallest tile has 128 rows, a unit 1 to 16.
//   S^T = K Q^T: the keys are the rows, the query heads the 8 (or twice 8) columns; O^T += V^T P^T: the dims are the rows.  Both operands come
//   from the ring by ldmatrix, plain and transposed; P^T is S^T with its 8 x 8 tiles turned by movmatrix, in registers.
//   A block of 128 dims is about 380 instructions of a warp (of 400, with a maximum every block, it took 0.65 us by itself); eight warps of an SM
//   fold 8 KB each in 1.4 us, which is the memory's rate.
//   A weight goes in as two elements of the cache's type, as the instruction wants it, right to 2^-15 (bf16; f16: 2^-21, or 2^-25 of 1) of itself: rounded to
//   one, its 2^-8 (2^-11) stood out wherever values cancel, and two products instead of one cost little, the tensor pipe being idle for the most part (64 ragged
//   sequences 44.5 -> 44.8 us; 33 in f16 with a window 20.4 -> 21.7, where the instructions count).
//   The sum below the fraction adds the f32 weights.
//   f16 has them 2^11 times larger (2^15 at most, with a slack of 2^4; numerator and denominator share the factor, in all pieces), so that it keeps them down to
//   2^-25 of the largest to 2^-11 of themselves.  A block with one below that has more products (fold_light): where a key holds nearly all the weight and its
//   value little, the answer is the sum of many that are lighter than any f16.  (16 sequences of 8192 keys: 90 us, with a heavy key in every block 96; by f32
//   products, as fold_plain has them, 193.)
template <typename T_, int DP_, int NT>
struct MmaBlock {
  using T = T_;
  static constexpr int DP = DP_, KB = 16, HEADS = 8 * NT, ROWB = DP * 2, PR = DP + 4, EXTRA = 0;
  static constexpr bool HALF = std::is_same<T, __half>::value;
  // Weights are 2^(score - m) for an m that follows the running maximum only when a score is above it by more than SLACK: one vote a block instead of the
  // maximum's shuffles and the corrections (64 ragged sequences 45.1 -> 44.5 us, 33 with a window 19.6 -> 18.8; f32, whose heads' maxima take three
  // shuffles: 11.2 -> 11.6 for 4 x 1024; all of it before weights had two halves).  Weights reach 2^SLACK, and the largest is 1 or more, as with the maximum
  // itself.  2^4 for f16, which leaves its weights four binades more below the largest.
  static constexpr float SLACK = HALF ? 4.f : 8.f, UP = HALF ? 15.f - SLACK : 0.f;
  uint32_t q[DP / 16][NT][2];
  float o[DP / 16][NT][4], m[NT][2], l[NT][2];

  __device__ __forceinline__ void begin(const SplitArgs &s, int b, int kh, int h0, int count, unsigned char *) {
    const PagedArgs &a = s.p;
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int h = 8 * nt + r;
      const T *p = static_cast<const T *>(a.q) + b * a.q_s[0] + (kh * a.G + h0 + h) * a.q_s[1] + 2 * c;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ks++)
#pragma unroll
        for (int e = 0; e < 2; e++) q[ks][nt][e] = h < count && ks * 16 < a.D ? *reinterpret_cast<const uint32_t *>(p + 16 * ks + 8 * e) : 0u;
#pragma unroll
      for (int e = 0; e < 2; e++) m[nt][e] = -INFINITY, l[nt][e] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / 16; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[t][nt][e] = 0.f;
    }
  }

  __device__ __forceinline__ void block(const Scorer &score, uint32_t kbase, uint32_t valid, unsigned char *) {
    const int lane = threadIdx.x & 31, r = lane >> 2;
    float s[NT][4], s2[NT][4];  // (two sums: half the chain of dependent instructions)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) s[nt][e] = s2[nt][e] = 0.f;
    const int turn = spread(lane & 7);
    const uint32_t krow = kbase + (lane & 15) * ROWB, vrow = kbase + KB * ROWB + ((lane & 7) + (lane >> 4) * 8) * ROWB;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ks++) {
      uint32_t f[4];
      ldm4(f, krow + (((2 * ks + (lane >> 4)) ^ turn) << 4));
#pragma unroll
      for (int nt = 0; nt < NT; nt++) mma(ks & 1 ? s2[nt] : s[nt], f, q[ks][nt][0], q[ks][nt][1], T());
    }
    bool fits = true;  // all scores within SLACK of the maximum at hand
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int e = 0; e < 4; e++) s[nt][e] = (s[nt][e] + s2[nt][e]) * score.sc;
    }
    if (score.cap > 0.f) score.cap_all(s);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      if (valid != 0xFFFFu) {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (!(valid >> (r + 8 * (e >> 1)) & 1)) s[nt][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 2; e++) fits = fits && fmaxf(s[nt][e], s[nt][2 + e]) <= m[nt][e] + SLACK;
    }
    if (!__all_sync(0xffffffffu, fits)) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        float corr[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float mx = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          mx = fmaxf(mx, m[nt][e]);
          corr[e] = ex2(m[nt][e] - (mx == -INFINITY ? 0.f : mx));
          m[nt][e] = mx, l[nt][e] *= corr[e];
        }
#pragma unroll
        for (int t = 0; t < DP / 16; t++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[t][nt][e] *= corr[e & 1];
      }
    }
    uint32_t p[NT][2][2];  // high, low; keys 0 to 7, 8 to 15
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const float use = (m[nt][e] == -INFINITY ? 0.f : m[nt][e]) - UP;  // no key above -inf so far: all weights 0
        s[nt][e] = ex2(s[nt][e] - use), s[nt][2 + e] = ex2(s[nt][2 + e] - use);
        l[nt][e] += s[nt][e] + s[nt][2 + e];
      }
    }
    if constexpr (HALF) {
      float least = 1.f;
      bool any = false;
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) least = fminf(least, s[nt][e]);
      if (__any_sync(0xffffffffu, least < 0x1p-14f)) {  // (0 where there is no key)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) any = any || light(s[nt][e]);
        if (__any_sync(0xffffffffu, any)) {
          fold_light(s, kbase + KB * ROWB, vrow);
          return;
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        halves(s[nt][2 * i], s[nt][2 * i + 1], p[nt][0][i], p[nt][1][i], T());
        p[nt][0][i] = transposed(p[nt][0][i]), p[nt][1][i] = transposed(p[nt][1][i]);
      }
    }
#pragma unroll
    for (int t = 0; t < DP / 16; t++) {
      uint32_t f[4];
      ldm4_trans(f, vrow + (((2 * t + (lane >> 3 & 1)) ^ turn) << 4));
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) mma(o[t][nt], f, p[nt][i][0], p[nt][i][1], T());
    }
  }

  // 0 < w < 2^-14: f16 has fewer than 11 bits for it; 0 < w < 2^-43: not 2^29 times larger either
  __device__ __forceinline__ static bool light(float w) { return __float_as_uint(w) - 1u < 0x38800000u - 1u; }
  __device__ __forceinline__ static bool faint(float w) { return __float_as_uint(w) - 1u < 0x2A000000u - 1u; }

  // O^T += V^T P^T of a block with light weights: those go in 2^29 times larger, as products of their own.  A weight is 0 in one of the two, which an
  // infinite value would make NaN of: where a result is NaN, and where weights are faint, fold_plain gives it.
  __device__ __forceinline__ void fold_light(const float (&w)[NT][4], uint32_t vbase, uint32_t vrow) {
    const int lane = threadIdx.x & 31, turn = spread(lane & 7);
    bool any = false;
    uint32_t p[NT][2][2], x[NT][2][2];  // high, low; keys 0 to 7, 8 to 15
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        float a[2], b[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float v = w[nt][2 * i + e];
          any = any || faint(v), a[e] = light(v) ? 0.f : v, b[e] = light(v) ? v * 0x1p29f : 0.f;
        }
        halves(a[0], a[1], p[nt][0][i], p[nt][1][i], T()), halves(b[0], b[1], x[nt][0][i], x[nt][1][i], T());
#pragma unroll
        for (int k = 0; k < 2; k++) p[nt][k][i] = transposed(p[nt][k][i]), x[nt][k][i] = transposed(x[nt][k][i]);
      }
    uint32_t left = __any_sync(0xffffffffu, any) ? ~0u : 0u;  // what fold_plain has to do, a bit for sixteen dims of eight heads
    if (!left) {
#pragma unroll
      for (int t = 0; t < DP / 16; t++) {
        uint32_t f[4];
        ldm4_trans(f, vrow + (((2 * t + (lane >> 3 & 1)) ^ turn) << 4));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float u[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 2; k++) mma(u, f, p[nt][k][0], p[nt][k][1], T()), mma(y, f, x[nt][k][0], x[nt][k][1], T());
          bool nan = false;
#pragma unroll
          for (int e = 0; e < 4; e++) u[e] = fmaf(y[e], 0x1p-29f, o[t][nt][e] + u[e]), nan = nan || u[e] != u[e];
          nan = __any_sync(0xffffffffu, nan);
          left |= (uint32_t)nan << (t * NT + nt);
#pragma unroll
          for (int e = 0; e < 4; e++) o[t][nt][e] = nan ? o[t][nt][e] : u[e];
        }
      }
    }
    if (left) fold_plain(w, vbase, left);
  }
  // The same by f32 products: a key at a time, its weights from the lanes that have them.
  __device__ __forceinline__ void fold_plain(const float (&p)[NT][4], uint32_t vbase, uint32_t which) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll 1
    for (int j = 0; j < KB; j++) {
      float w[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) w[nt][e] = __shfl_sync(0xffffffffu, j < 8 ? p[nt][e] : p[nt][2 + e], (j & 7) * 4 + c);
      const uint32_t row = vbase + j * ROWB + 2 * r;
#pragma unroll
      for (int t = 0; t < DP / 16; t++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
          if (which >> (t * NT + nt) & 1) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
              const float v = lds_f16(row + (((2 * t + half) ^ spread(j)) << 4));
#pragma unroll
              for (int e = 0; e < 2; e++) o[t][nt][2 * half + e] = fmaf(w[nt][e], v, o[t][nt][2 * half + e]);
            }
          }
    }
  }

  // the result of `count` heads from `out` on
  __device__ __forceinline__ void write(T *out, int count, int D, unsigned char *) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float inv[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float sum = l[nt][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        l[nt][e] = sum, inv[e] = 1.f / sum;
      }
      const bool none0 = l[nt][0] == 0.f, none1 = l[nt][1] == 0.f;
#pragma unroll
      for (int t = 0; t < DP / 16; t++)
        if (t * 16 < D) {
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float x = none0 ? 0.f : o[t][nt][2 * e] * inv[0], y = none1 ? 0.f : o[t][nt][2 * e + 1] * inv[1];
            const uint32_t v = transposed(pack(x, y, T()));  // head 8 nt + r, dims 2 c and 2 c + 1 of eight
            if (8 * nt + r < count) *reinterpret_cast<uint32_t *>(out + (8 * nt + r) * D + 16 * t + 8 * e + 2 * c) = v;
          }
        }
    }
  }

  __device__ __forceinline__ void store(float *part, int D) {  // [HEADS][PR]: max, sum, -, -, D dims
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float sum = l[nt][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        float *row = part + (8 * nt + 2 * c + e) * PR;
        if (r == 0) row[0] = m[nt][e], row[1] = sum;
#pragma unroll
        for (int t = 0; t < DP / 16; t++)
          if (t * 16 < D) row[4 + 16 * t + r] = o[t][nt][e], row[4 + 16 * t + r + 8] = o[t][nt][2 + e];
      }
  }
};

// f32: a block of 8 keys, f32 products, two to an instruction (f32x2).
//   Scores: sixteen lanes take a key, two keys at a time; a lane has DP / 64 chunks of all query heads in registers and multiplies four keys'
//   with them.  (Read from shared memory, as broadcasts, they were half of its traffic, 252 wavefronts a block instead of 123: seconds of
//   calls of eight sequences of 8192 keys, at the clocks that they run at, 101 us each instead of 92.)  The 4 GH partial sums are
//   exchanged until every lane has one score complete (two of 8 heads): at each step it hands half of them to its partner and keeps the other half.
//   Value i = 4 h + t (head h, key 2 t + lane / 16) ends in the lanes with lane % 16 = i (8 heads: i / 2; fewer than 4: several lanes).
//   Values: the weights go through shared memory, twice each, as the f32x2 products want them; SPLIT keys at a time, a lane owns NC chunks of dims.
template <int DP_, int GH>
struct F32Block {
  using T = float;
  static constexpr int DP = DP_, KB = 8, HEADS = GH, ROWB = DP * 4, PR = DP + 4;
  static constexpr int QC = DP / 64, NV = 4 * GH, OWN = NV > 16 ? NV / 16 : 1, SAME = NV < 16 ? 16 / NV : 1;  // chunks of a query; sums; scores of a lane, lanes of a score
  static constexpr int SPLIT = GH > 4 ? (DP == 64 ? 2 : 1) : DP == 64 ? 4 : DP == 128 ? 2 : 1, LANES = 32 / SPLIT, NC = DP / 4 / LANES;
  static constexpr int EXTRA = KB * GH * 8 + (GH * 4 + 15) / 16 * 16;  // of a warp: weights, corrections or sums
  uint64_t q[GH][QC][2], acc[GH][NC][2];
  float m, l;  // of this lane's head

  __device__ __forceinline__ static int head_of(int lane) { return (lane & 15) * OWN / SAME / 4; }
  __device__ __forceinline__ static int t_of(int lane, int i) { return ((lane & 15) * OWN / SAME + i) & 3; }

  __device__ __forceinline__ void begin(const SplitArgs &s, int b, int kh, int h0, int count, unsigned char *) {
    const PagedArgs &a = s.p;
    const int lane = threadIdx.x & 31;
    const float *from = static_cast<const float *>(a.q) + b * a.q_s[0] + (kh * a.G + h0) * a.q_s[1];
#pragma unroll
    for (int h = 0; h < GH; h++)
#pragma unroll
      for (int i = 0; i < QC; i++) {
        const int c = (lane & 15) + 16 * i;
        q[h][i][0] = q[h][i][1] = 0;
        if (h < count && 4 * c < a.D) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(from + h * a.q_s[1] + 4 * c);
          q[h][i][0] = v.x, q[h][i][1] = v.y;
        }
      }
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int h = 0; h < GH; h++)
#pragma unroll
      for (int i = 0; i < NC; i++) acc[h][i][0] = acc[h][i][1] = 0;
  }

  __device__ __forceinline__ void block(const Scorer &score, uint32_t kbase, uint32_t valid, unsigned char *extra) {
    const int lane = threadIdx.x & 31, sub = lane >> 4;
    float2 *ps = reinterpret_cast<float2 *>(extra);
    float *cs = reinterpret_cast<float *>(ps + KB * GH);
    float v[NV];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      uint64_t d[GH];
#pragma unroll
      for (int h = 0; h < GH; h++) d[h] = 0;
      const int key = 2 * t + sub;
#pragma unroll
      for (int i = 0; i < QC; i++) {
        const uint4 w = lds128(kbase + key * ROWB + ((((lane & 15) + 16 * i) ^ spread(key)) << 4));
        const uint64_t k0 = (uint64_t)w.y << 32 | w.x, k1 = (uint64_t)w.w << 32 | w.z;
#pragma unroll
        for (int h = 0; h < GH; h++) d[h] = fma2(q[h][i][0], k0, fma2(q[h][i][1], k1, d[h]));
      }
#pragma unroll
      for (int h = 0; h < GH; h++) v[4 * h + t] = lo(d[h]) + hi(d[h]);
    }
    int cnt = NV;
#pragma unroll
    for (int x = 8; x >= 1; x >>= 1) {
      if (cnt > OWN) {
        const int half = cnt / 2;
        const bool up = lane & x;
#pragma unroll
        for (int i = 0; i < NV / 2; i++)
          if (i < half) {
            const float send = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, x);
          }
        cnt = half;
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], x);
      }
    }
    float mx = m;
#pragma unroll
    for (int i = 0; i < OWN; i++) v[i] = valid >> (2 * t_of(lane, i) + sub) & 1 ? score(v[i]) : -INFINITY, mx = fmaxf(mx, v[i]);
#pragma unroll
    for (int x = 1; x < 4 / OWN; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x * SAME));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
    const float use = mx == -INFINITY ? 0.f : mx, corr = ex2(m - use);
    const bool same = mx == m;
    m = mx, l *= corr;
#pragma unroll
    for (int i = 0; i < OWN; i++) {
      const float p = ex2(v[i] - use);
      l += p;
      ps[(2 * t_of(lane, i) + sub) * GH + head_of(lane)] = make_float2(p, p);
    }
    cs[head_of(lane)] = corr;  // (the same from all lanes of a head)
    __syncwarp();
    if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
      for (int h = 0; h < GH; h++) {
        const uint64_t c = two(cs[h], cs[h]);
#pragma unroll
        for (int i = 0; i < NC; i++) acc[h][i][0] = mul2(acc[h][i][0], c), acc[h][i][1] = mul2(acc[h][i][1], c);
      }
    }
#pragma unroll
    for (int k0 = 0; k0 < KB; k0 += SPLIT) {
      const int k = k0 + lane / LANES;
      uint64_t p[GH];
      if constexpr (GH >= 2) {
#pragma unroll
        for (int h = 0; h < GH; h += 2) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(ps + k * GH + h);
          p[h] = x.x, p[h + 1] = x.y;
        }
      } else {
        p[0] = *reinterpret_cast<const uint64_t *>(ps + k);
      }
#pragma unroll
      for (int i = 0; i < NC; i++) {
        const uint4 w = lds128(kbase + (KB + k) * ROWB + (((lane % LANES + LANES * i) ^ spread(k)) << 4));
        const uint64_t v0 = (uint64_t)w.y << 32 | w.x, v1 = (uint64_t)w.w << 32 | w.z;
#pragma unroll
        for (int h = 0; h < GH; h++) acc[h][i][0] = fma2(p[h], v0, acc[h][i][0]), acc[h][i][1] = fma2(p[h], v1, acc[h][i][1]);
      }
    }
  }

  // the four dims of a chunk, of all lanes that have some of its keys
  __device__ __forceinline__ float4 dims(int h, int i) const {
    float v[4] = {lo(acc[h][i][0]), hi(acc[h][i][0]), lo(acc[h][i][1]), hi(acc[h][i][1])};
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
      for (int x = LANES; x < 32; x <<= 1) v[e] += __shfl_xor_sync(0xffffffffu, v[e], x);
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  __device__ __forceinline__ float sum_of() const {  // over the keys of all lanes of this lane's head
    float sum = l;
#pragma unroll
    for (int x = 1; x < 4 / OWN; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x * SAME);
    return sum + __shfl_xor_sync(0xffffffffu, sum, 16);
  }

  __device__ __forceinline__ void write(float *out, int count, int D, unsigned char *extra) {
    const int lane = threadIdx.x & 31;
    float *cs = reinterpret_cast<float *>(extra) + 2 * KB * GH;
    const float mine = sum_of();
    __syncwarp();
    cs[head_of(lane)] = mine;
    __syncwarp();
#pragma unroll
    for (int h = 0; h < GH; h++) {
      const float sum = cs[h], inv = 1.f / sum;
#pragma unroll
      for (int i = 0; i < NC; i++) {
        const float4 v = dims(h, i);
        const int c = lane % LANES + LANES * i;
        if (lane < LANES && c * 4 < D && h < count)
          *reinterpret_cast<float4 *>(out + h * D + 4 * c) = sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      }
    }
  }

  __device__ __forceinline__ void store(float *part, int D) {
    const int lane = threadIdx.x & 31;
    const float mine = sum_of();
    part[head_of(lane) * PR] = m, part[head_of(lane) * PR + 1] = mine;  // (the same from all lanes of a head)
#pragma unroll
    for (int h = 0; h < GH; h++)
#pragma unroll
      for (int i = 0; i < NC; i++) {
        const float4 v = dims(h, i);
        const int c = lane % LANES + LANES * i;
        if (lane < LANES && c * 4 < D) *reinterpret_cast<float4 *>(part + h * PR + 4 + 4 * c) = v;
      }
  }
};

// shared memory of a CTA with rings of `stages` blocks, and how many CTAs of two blocks or more fit on an SM (three at most: registers)
constexpr int split_smem(int size, int DP, int HEADS, int stages) {
  const int rows = size == 2 ? 16 : 8, extra = size == 2 ? 0 : rows * HEADS * 8 + (HEADS * 4 + 15) / 16 * 16;
  return PA_WARPS * (stages * 2 * rows * DP * size + HEADS * (DP + 4) * 4 + extra);
}
constexpr int split_room(int ctas) { return 228 * 1024 / ctas - 1024 - 512; }  // beside what is static
constexpr int split_ctas(int size, int DP, int HEADS) {
  int n = DP == 64 ? 3 : DP == 128 ? 2 : 1;
  while (n > 1 && split_smem(size, DP, HEADS, 2) > split_room(n)) n--;
  return n;
}
constexpr int split_stages(int size, int DP, int HEADS) {
  int n = 4;
  while (n > 2 && split_smem(size, DP, HEADS, n) > split_room(split_ctas(size, DP, HEADS))) n--;
  return n;
}

template <typename P>
struct SplitCfg {
  static constexpr int SIZE = sizeof(typename P::T), CTAS = split_ctas(SIZE, P::DP, P::HEADS), S = split_stages(SIZE, P::DP, P::HEADS);
  static constexpr int STAGE = 2 * P::KB * P::ROWB, RING = S * STAGE, PART = P::HEADS * P::PR * 4;  // of a warp
  static constexpr int SMEM = PA_WARPS * (RING + PART + P::EXTRA);
  static_assert(SMEM == split_smem(SIZE, P::DP, P::HEADS, S) && SMEM <= split_room(CTAS) && PART <= RING && PA_WARPS * PART >= PA_THREADS * 4, "");
};

struct Cursor {
  int b, kh, hg, block, n, j0, blocks;  // sequence, KV head, unit of that, block; the sequence's length, first key, blocks per unit
  int left;                             // cost of the run from this block on; none left: no block
  template <int KB>
  __device__ __forceinline__ void at(const PagedArgs &a, int b_) {
    b = b_, n = length_of(a, b_), j0 = first_of(a, n), blocks = (n - j0 + KB - 1) / KB;
  }
  __device__ __forceinline__ void unit(int u, int groups) { kh = groups == 1 ? u : u / groups, hg = u - kh * groups; }
  template <int KB>
  __device__ __forceinline__ void next(const SplitArgs &s, int hop) {
    block += hop, left -= hop;
    if (block < blocks) return;
    left -= UNIT;
    if (left <= 0) return;
    block = 0;
    if (++hg < s.groups) return;
    hg = 0;
    if (++kh < s.p.KH) return;
    kh = 0;
    do at<KB>(s.p, b + 1);
    while (blocks == 0);
  }
};

// four neighbouring elements of an output: v / L
template <typename T>
__device__ __forceinline__ void store4(T *out, const float (&v)[4], float L) {
  const float inv = 1.f / L;
  alignas(16) T x[4];
#pragma unroll
  for (int e = 0; e < 4; e++) x[e] = from_f32<T>(L == 0.f ? 0.f : v[e] * inv);
  if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<const uint4 *>(x);
  else *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(x);
}

// What a warp's copies take: the page of its lane's key, then a block of rows into a slot of its ring.
struct Row {
  int pg, row, kh;
  bool valid;
};

template <typename P, int S>
struct Feeder {
  using C = SplitCfg<P>;
  using T = typename P::T;
  static constexpr int E = 16 / (int)sizeof(T), CHUNKS = P::DP / E, LANES = CHUNKS < 32 ? CHUNKS : 32, RPI = 32 / LANES, CPL = CHUNKS / LANES;
  const SplitArgs &s;
  uint32_t *masks;   // [S]: the keys of each slot's block that there are
  uint32_t ring;
  const char *k0, *v0;
  unsigned odd = 0;

  __device__ __forceinline__ Feeder(const SplitArgs &s_, unsigned char *ring_, uint32_t *masks_) : s(s_), masks(masks_), ring(umma::smem_u32(ring_)) {
    const int lane = threadIdx.x & 31;
    k0 = static_cast<const char *>(s.p.k) + lane % LANES * 16, v0 = static_cast<const char *>(s.p.v) + lane % LANES * 16;
    if (s.p.D < P::DP) {  // chunks past the head: nothing is copied there, and the products run over them
      for (int i = lane; i < S * C::STAGE / 16; i += 32) reinterpret_cast<uint4 *>(ring_)[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
    }
  }
  __device__ __forceinline__ Row peek(const Cursor &c) const { return peek(c, c.j0, c.n); }
  __device__ __forceinline__ Row peek(const Cursor &c, int j0, int n) const {  // (lanes from KB on repeat)
    const PagedArgs &a = s.p;
    Row r;
    const int j = j0 + c.block * P::KB + (threadIdx.x & (P::KB - 1)), w = a.page.div(j);
    r.valid = j < n, r.row = j - w * a.page.d, r.kh = c.kh;
    r.pg = r.valid ? a.table[c.b * a.table_stride + w] : -1;
    return r;
  }
  __device__ __forceinline__ void issue(const Row &r, int slot) {
    const PagedArgs &a = s.p;
    constexpr int KB = P::KB;
    const int lane = threadIdx.x & 31;
    const bool ok = r.valid && r.pg >= 0 && r.pg < a.pages;
    if (r.valid && !ok) odd |= PAGED_PAGE;
    const uint32_t mask = __ballot_sync(0xffffffffu, ok) & ((1u << KB) - 1);
    if (lane == 0) masks[slot] = mask;
    const uint32_t ko = ok ? r.pg * s.ku[0] + r.kh * s.ku[1] + r.row * s.ku[2] : 0;
    const uint32_t dst = ring + slot * C::STAGE;
    if (mask == (1u << KB) - 1 && s.alike) {
#pragma unroll
      for (int i = 0; i < KB / RPI; i++) {
        const int row = i * RPI + lane / LANES;
        const uint32_t off = __shfl_sync(0xffffffffu, ko, row);
        const char *kp = k0 + (unsigned long long)off * s.unit, *vp = v0 + (unsigned long long)off * s.unit;
#pragma unroll
        for (int x = 0; x < CPL; x++) {
          const int c = lane % LANES + 32 * x;
          if (c * E < a.D) {
            const uint32_t to = dst + row * P::ROWB + ((c ^ spread(row)) << 4);
            cp_async16(to, kp + x * 512);
            cp_async16(to + KB * P::ROWB, vp + x * 512);
          }
        }
      }
    } else {
      const uint32_t vo = ok ? r.pg * s.vu[0] + r.kh * s.vu[1] + r.row * s.vu[2] : 0;
#pragma unroll 1
      for (int i = 0; i < KB / RPI; i++) {
        const int row = i * RPI + lane / LANES;
        const uint32_t n = mask >> row & 1 ? 16 : 0;
        const char *kp = k0 + (unsigned long long)__shfl_sync(0xffffffffu, ko, row) * s.unit, *vp = v0 + (unsigned long long)__shfl_sync(0xffffffffu, vo, row) * s.unit;
        for (int x = 0; x < CPL; x++) {
          const int c = lane % LANES + 32 * x;
          if (c * E < a.D) {
            const uint32_t to = dst + row * P::ROWB + ((c ^ spread(row)) << 4);
            cp_async16_part(to, kp + x * 512, n);
            cp_async16_part(to + KB * P::ROWB, vp + x * 512, n);
          }
        }
      }
    }
  }
  // the run's first S - 1 blocks on their way, and the next one's page
  __device__ __forceinline__ Row fill(Cursor &far, int hop) {
    Row first[S - 1], next;
    int have = 0;
#pragma unroll
    for (int i = 0; i < S - 1; i++)
      if (far.left > 0) first[i] = peek(far), have = i + 1, far.next<P::KB>(s, hop);
#pragma unroll
    for (int i = 0; i < S - 1; i++) {
      if (i < have) issue(first[i], i);
      cp_async_commit();
    }
    if (far.left > 0) next = peek(far);
    return next;
  }
  __device__ __forceinline__ void more(Cursor &far, Row &next, int hop, int slot) {
    if (far.left > 0) {
      issue(next, slot);
      far.next<P::KB>(s, hop);
      if (far.left > 0) next = peek(far);
    }
    cp_async_commit();
  }
};

template <typename P>
__global__ void __launch_bounds__(PA_THREADS, SplitCfg<P>::CTAS) paged_attn_kernel(SplitArgs s) {
  using C = SplitCfg<P>;
  using T = typename P::T;
  constexpr int KB = P::KB, S = C::S;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int scan[PA_WARPS];
  __shared__ uint32_t masks[PA_WARPS][S];
  __shared__ int open0[PA_WARPS], open1[PA_WARPS];  // pieces: of a unit begun before the run, of the last begun in it: 0 none, 1 ends in it, 2 goes on
  __shared__ int4 piece0[PA_WARPS], piece1[PA_WARPS];  // their sequence, first query head, heads, blocks
  __shared__ long long cost1[PA_WARPS];             // where in cost the latter begins
  pdl_launch_dependents();
  pdl_wait();
  const PagedArgs &a = s.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x, units = a.KH * s.groups;
  unsigned odd = 0;

  // ---- the warps' runs.  Cost: UNIT, then one for each block, unit after unit; run i of r has [total i / r, total (i + 1) / r).
  const int per = (a.B + PA_THREADS - 1) / PA_THREADS, lo = min(tid * per, a.B), hi = min(lo + per, a.B);
  auto blocks_of = [&](int b) {
    const int n = length_of(a, b);
    return (n - first_of(a, n) + KB - 1) / KB;
  };
  auto cost_of = [&](int n) { return n ? n + UNIT : 0; };
  int *const chunk = reinterpret_cast<int *>(smem + PA_WARPS * C::RING);  // (over the parts, until the runs are known)
  int sum = 0;  // of one unit of each of this thread's sequences (the host has seen to it that all of them sum to less than 2^31)
  for (int b = lo; b < hi; b++) {
    if (cta == 0 && a.lens[b] != length_of(a, b)) odd |= PAGED_LENGTH;
    sum += cost_of(blocks_of(b));
  }
  int before = sum;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, x);
    if (lane >= x) before += v;
  }
  if (lane == 31) scan[warp] = before;
  chunk[tid] = before - sum;
  if (tid < PA_WARPS) open0[tid] = open1[tid] = 0;
  __syncthreads();
  int base[PA_WARPS], each = 0;
#pragma unroll
  for (int w = 0; w < PA_WARPS; w++) base[w] = each, each += scan[w];
  const long long total = (long long)each * units;
  // CTAs with work: the first ones, PA_WARPS blocks' cost or more each
  const int dealt = (int)min((long long)gridDim.x, max(total / PA_WARPS, 1ll)), runs = dealt * PA_WARPS;
  const bool small = total <= 0x7fffffffll;  // (the 64-bit division takes four times as long)
  const long long quota = small ? (long long)((unsigned)total / (unsigned)runs) : total / runs, rest = total - quota * runs;
  auto start_of = [&](int i) { return i * quota + min((long long)i, rest); };
  struct Place {
    int b, u, in, n;  // sequence, unit of it, cost of that before the place, blocks of the unit
  };
  auto locate = [&](long long x) {  // (x < total; the whole warp)
    int t = -1;
#pragma unroll
    for (int w = 0; w < PA_WARPS; w++) t += __popc(__ballot_sync(0xffffffffu, (long long)(base[w] + chunk[32 * w + lane]) * units <= x));
    int c = chunk[t];
#pragma unroll
    for (int w = 0; w < PA_WARPS; w++)
      if (t >> 5 == w) c += base[w];
    Place p;
    p.b = t * per, p.n = blocks_of(p.b);
    while ((long long)(c + cost_of(p.n)) * units <= x) c += cost_of(p.n), p.n = blocks_of(++p.b);
    const long long r = x - (long long)c * units;
    p.u = small ? (int)((unsigned)r / (unsigned)(p.n + UNIT)) : (int)(r / (p.n + UNIT)), p.in = (int)(r - (long long)p.u * (p.n + UNIT));
    return p;
  };
  // A CTA inside one unit deals its blocks to the warps in turn, so that they read side by side; else a warp has its own run.
  const bool works = cta < dealt && total > 0;
  bool inside = false;
  int all = 0, first = 0;  // inside: blocks, the first of them
  long long begun = 0;     // where the unit at hand begins in cost
  Cursor now;
  now.left = 0;
  if (works) {
    const long long x0 = start_of(cta * PA_WARPS), x1 = start_of((cta + 1) * PA_WARPS);
    Place p = locate(x0);
    inside = x1 - x0 <= p.n + UNIT - p.in;
    first = max(p.in - UNIT, 0);
    if (inside) {
      all = max((int)(x1 - x0) + p.in - UNIT, 0) - first, begun = x0 - p.in;
      now.block = first + warp, now.left = all - warp;
    } else {
      const long long w0 = start_of(cta * PA_WARPS + warp), w1 = start_of(cta * PA_WARPS + warp + 1);
      if (warp) p = locate(w0);
      now.block = max(p.in - UNIT, 0), now.left = (int)(w1 - w0) - max(UNIT - p.in, 0), begun = w0 - p.in;
    }
    now.at<KB>(a, p.b);
    now.unit(p.u, s.groups);
  }
  const int hop = inside ? PA_WARPS : 1;
  __syncthreads();
  unsigned char *const ring = smem + warp * C::RING, *const extra = smem + PA_WARPS * (C::RING + C::PART) + warp * P::EXTRA;
  float *const part = reinterpret_cast<float *>(smem + PA_WARPS * C::RING + warp * C::PART);
  if (now.left > 0) {
    Cursor far = now;  // what is fetched, ahead of what is folded
    Feeder<P, S> feed(s, ring, masks[warp]);
    Row next = feed.fill(far, hop);
    const Scorer score(a.scale, a.softcap);
    P state;
    bool fresh = true, begins = false;
    int slot = 0, fill = S - 1;
    while (now.left > 0) {
      if (fresh) begins = now.block == 0, fresh = false, state.begin(s, now.b, now.kh, now.hg * s.hpg, min(s.hpg, a.G - now.hg * s.hpg), extra);
      cp_async_wait<S - 2>();
      __syncwarp();  // the block is there for all lanes, and all are done with the one before
      feed.more(far, next, hop, fill);
      state.block(score, feed.ring + slot * C::STAGE, masks[warp][slot], extra);
      slot = slot + 1 == S ? 0 : slot + 1, fill = fill + 1 == S ? 0 : fill + 1;
      const bool last = now.left <= hop;
      // (inside one unit its end belongs to the last warp's piece, whoever has the last block)
      const bool ends = inside ? last && warp == min(PA_WARPS, all) - 1 && first + all == now.blocks : now.block + 1 == now.blocks;
      if (ends || last) {
        const int h0 = now.hg * s.hpg;
        const int4 who = make_int4(now.b, now.kh * a.G + h0, min(s.hpg, a.G - h0), now.blocks);
        if (begins && ends && !inside) {
          state.write(static_cast<T *>(a.out) + ((long long)now.b * a.NH + now.kh * a.G + h0) * a.D, who.z, a.D, extra);
        } else if (begins) {  // (the run's end: its ring is free once the last copies have landed)
          cp_async_wait<0>();
          __syncwarp();
          state.store(reinterpret_cast<float *>(ring), a.D);
          if (lane == 0) open1[warp] = ends ? 1 : 2, piece1[warp] = who, cost1[warp] = begun;
        } else {
          state.store(part, a.D);
          if (lane == 0) open0[warp] = ends ? 1 : 2, piece0[warp] = who;
        }
        fresh = true, begun += now.blocks + UNIT;
      }
      now.next<KB>(s, hop);
    }
    cp_async_wait<0>();
    odd |= feed.odd;
  }
  if (odd) atomicOr(&g_attn_status, odd);
  __syncthreads();

  // ---- the CTA's pieces: a run's first belongs to a unit begun before it, its last to one that goes on in the next warp's first
  int4 head = make_int4(0, 0, 0, 0);
  unsigned kinds = 0;  // two bits a piece: of warp p / 2, the one begun before its run (p even), or the last begun in it
#pragma unroll
  for (int w = 0; w < PA_WARPS; w++) kinds |= (unsigned)(open0[w] | open1[w] << 2) << (4 * w);
#pragma unroll 1
  for (int p = 0; p < 2 * PA_WARPS;) {
    const int w0 = p >> 1, late = p & 1;
    unsigned kind = kinds >> (2 * p) & 3;
    if (kind == 0) {
      p++;
      continue;
    }
    int w1 = w0;  // the last warp that has a piece of the unit
    while (kind == 2 && w1 + 1 < PA_WARPS && (kinds >> (4 * (w1 + 1)) & 3)) kind = kinds >> (4 * ++w1) & 3;
    const int4 who = late ? piece1[w0] : piece0[w0];
    const bool whole = late && kind == 1;
    const float *const row0 = reinterpret_cast<const float *>(late ? smem + w0 * C::RING : smem + PA_WARPS * C::RING + w0 * C::PART);
    const float *const row1 = reinterpret_cast<const float *>(smem + PA_WARPS * C::RING + w0 * C::PART);
    for (int h = warp; h < who.z; h += PA_WARPS) {
      const float *row[PA_WARPS];
      float2 ml[PA_WARPS];
      float top = -INFINITY, L = 0.f, e[PA_WARPS];
#pragma unroll
      for (int i = 0; i < PA_WARPS; i++) {
        row[i] = (i == 0 ? row0 : row1 + i * (C::PART / 4)) + h * P::PR;
        ml[i] = i <= w1 - w0 ? *reinterpret_cast<const float2 *>(row[i]) : make_float2(-INFINITY, 0.f);
        top = fmaxf(top, ml[i].x);
      }
      const float use = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int i = 0; i < PA_WARPS; i++) e[i] = ex2(ml[i].x - use), L = fmaf(e[i], ml[i].y, L);
      const long long at = (2ll * cta + late) * P::HEADS + h;
      if (!whole && lane == 0) *reinterpret_cast<float2 *>(s.ml + 2 * at) = make_float2(top, L);
#pragma unroll
      for (int d = 4 * lane; d < P::DP; d += 128)
        if (d < a.D) {
          float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < PA_WARPS; i++)
            if (i <= w1 - w0) {
              const float4 x = *reinterpret_cast<const float4 *>(row[i] + 4 + d);
              v[0] = fmaf(e[i], x.x, v[0]), v[1] = fmaf(e[i], x.y, v[1]), v[2] = fmaf(e[i], x.z, v[2]), v[3] = fmaf(e[i], x.w, v[3]);
            }
          if (whole) store4(static_cast<T *>(a.out) + ((long long)who.x * a.NH + who.y + h) * a.D + d, v, L);
          else *reinterpret_cast<float4 *>(s.acc + at * a.D + d) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
    if (late && kind == 2) {  // the run that has its last block, and so the CTAs that it goes over
      const long long x = cost1[w0] + UNIT + who.w - 1, wide = rest * (quota + 1);
      const long long run = small ? (x < wide ? (unsigned)x / (unsigned)(quota + 1) : rest + (unsigned)(x - wide) / (unsigned)quota)
                                  : (x < wide ? x / (quota + 1) : rest + (x - wide) / quota);
      head = make_int4(who.x, who.y, who.z, (int)(run / PA_WARPS) - cta + 1);
    }
    p = w1 > w0 ? 2 * w1 + 1 : p + 1;
  }
  if (s.heads && tid == 0) s.heads[cta] = head;
  // sequences without keys
  for (int b = cta; b < a.B; b += gridDim.x)
    if (blocks_of(b) == 0)
      for (int i = tid; i < a.NH * a.D; i += PA_THREADS) static_cast<T *>(a.out)[(long long)b * a.NH * a.D + i] = from_f32<T>(0.f);
}

// Few units of few blocks: a cluster of up to sixteen CTAs takes a unit, its warps the blocks in turn: one launch, no scratch, no schedule to work
// out, which is what counts when there is little to read.  What bounds it is a chain of latencies, so:
//   * the queries, the length and (without a window) the page of a warp's first block are asked for together;
//   * the output is dealt to the CTAs in slices, and each CTA pushes its part of every slice into the shared memory of the one that has it, before
//     the one barrier: what is read after it is at home, and nobody has to stay for others to read from.  (1024 keys by 16 CTAs: 5.35 us with
//     the parts pulled and a barrier at the end, 5.1 us; 32 units by 8: 6.9, 6.4.)
constexpr int CL_MAX = 16;

template <typename P>
struct ClusterCfg {
  using C = SplitCfg<P>;
  static constexpr int PARTS = PA_WARPS * (C::PART + P::EXTRA), TAKE = P::HEADS * P::DP * 4 + CL_MAX * (16 + P::HEADS * 8);  // parts of the slice, maxima and sums
  static constexpr int stages(int n) { return n > 2 && PA_WARPS * n * C::STAGE + PARTS + TAKE > split_room(C::CTAS) ? stages(n - 1) : n; }
  static constexpr int S = stages(C::S), RING = S * C::STAGE, SMEM = PA_WARPS * RING + PARTS + TAKE;
  static_assert(SMEM <= split_room(C::CTAS), "");
};

__device__ __forceinline__ void st_cluster(uint32_t addr, float2 v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};\n" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, const float (&v)[4]) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}

// `slice`: chunks of four dims of a CTA's slice of the unit's heads
template <typename P>
__global__ void __launch_bounds__(PA_THREADS, SplitCfg<P>::CTAS) paged_attn_cluster_kernel(SplitArgs s, int ks, FastDiv slice) {
  using C = ClusterCfg<P>;
  using T = typename P::T;
  constexpr int KB = P::KB, S = C::S, PART = SplitCfg<P>::PART;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint32_t masks[PA_WARPS][S];
  pdl_launch_dependents();
  pdl_wait();
  const PagedArgs &a = s.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, units = a.KH * s.groups, rank = blockIdx.x % ks, unit = blockIdx.x / ks, b = unit / units;
  const int hop = ks * PA_WARPS;
  unsigned char *const ring = smem + warp * C::RING, *const extra = smem + PA_WARPS * (C::RING + PART) + warp * P::EXTRA;
  float *const part = reinterpret_cast<float *>(smem + PA_WARPS * C::RING + warp * PART);
  Cursor far;
  far.b = b, far.unit(unit - b * units, s.groups), far.block = rank * PA_WARPS + warp;
  const int kh = far.kh, h0 = far.hg * s.hpg, count = min(s.hpg, a.G - h0);
  P state;
  Feeder<P, S> feed(s, ring, masks[warp]);
  state.begin(s, b, kh, h0, count, extra);
  Row next;
  const bool early = a.window == 0;
  if (early) next = feed.peek(far, 0, a.W * a.page.d);
  far.at<KB>(a, b);
  const int blocks = far.blocks;
  int left = far.left = blocks - far.block;
  T *const out = static_cast<T *>(a.out) + ((long long)b * a.NH + kh * a.G + h0) * a.D;
  if (tid == 0 && rank == 0 && kh == 0 && far.hg == 0 && a.lens[b] != far.n) atomicOr(&g_attn_status, (unsigned)PAGED_LENGTH);
  if (blocks == 0) {  // (the whole cluster)
    for (int i = rank * PA_THREADS + tid; i < count * a.D; i += ks * PA_THREADS) out[i] = from_f32<T>(0.f);
    return;
  }
  if (ks > 1) umma::cluster_arrive();  // this CTA runs: others may write into its memory
  if (early) next.valid = (rank * PA_WARPS + warp) * KB + (lane & (KB - 1)) < far.n;
  else if (left > 0) next = feed.peek(far);
  // S blocks on their way to begin with; a slot is filled again as soon as it has been folded
#pragma unroll
  for (int i = 0; i < S; i++) {
    if (far.left > 0) {
      feed.issue(next, i);
      far.next<KB>(s, hop);
      if (far.left > 0) next = feed.peek(far);
    }
    cp_async_commit();
  }
  const Scorer score(a.scale, a.softcap);
  for (int slot = 0; left > 0; left -= hop) {
    cp_async_wait<S - 1>();
    __syncwarp();
    state.block(score, feed.ring + slot * SplitCfg<P>::STAGE, masks[warp][slot], extra);
    __syncwarp();
    if (left > hop) feed.more(far, next, hop, slot);
    slot = slot + 1 == S ? 0 : slot + 1;
  }
  if (feed.odd) atomicOr(&g_attn_status, feed.odd);
  state.store(part, a.D);
  __syncthreads();
  const float *const parts = reinterpret_cast<const float *>(smem + PA_WARPS * C::RING);
  // what the CTAs push here: of each its part of this slice, then of each its maxima and sums
  const uint32_t take = umma::smem_u32(smem + PA_WARPS * C::RING + C::PARTS);
  const uint32_t take_ml = take + (uint32_t)ks * slice.d * 16u;
  if (ks > 1) umma::cluster_wait();
  for (int h = warp; h < count; h += PA_WARPS) {
    const float *row = parts + h * P::PR;
    float2 ml[PA_WARPS];
    float top = -INFINITY, L = 0.f, e[PA_WARPS];
#pragma unroll
    for (int w = 0; w < PA_WARPS; w++) ml[w] = *reinterpret_cast<const float2 *>(row + w * P::HEADS * P::PR), top = fmaxf(top, ml[w].x);
    const float use = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < PA_WARPS; w++) e[w] = ex2(ml[w].x - use), L = fmaf(e[w], ml[w].y, L);
    if (ks > 1 && lane < ks) st_cluster(umma::map_to_rank(take_ml, (uint32_t)lane) + (uint32_t)(rank * P::HEADS + h) * 8u, make_float2(top, L));
#pragma unroll
    for (int d = 4 * lane; d < P::DP; d += 128)
      if (d < a.D) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < PA_WARPS; w++) {
          const float4 x = *reinterpret_cast<const float4 *>(row + w * P::HEADS * P::PR + 4 + d);
          v[0] = fmaf(e[w], x.x, v[0]), v[1] = fmaf(e[w], x.y, v[1]), v[2] = fmaf(e[w], x.z, v[2]), v[3] = fmaf(e[w], x.w, v[3]);
        }
        if (ks == 1) {
          store4(out + h * a.D + d, v, L);
        } else {
          const int c = (h * a.D + d) >> 2, to = slice.div(c);
          st_cluster(umma::map_to_rank(take, (uint32_t)to) + (uint32_t)(rank * slice.d + c - to * slice.d) * 16u, v);
        }
      }
  }
  if (ks == 1) return;
  umma::cluster_arrive();
  umma::cluster_wait();
  for (int c = tid; c < slice.d; c += PA_THREADS) {
    const int i = 4 * (rank * slice.d + c), h = i / a.D;
    if (h >= count) break;
    const float2 *ml = reinterpret_cast<const float2 *>(smem + PA_WARPS * C::RING + C::PARTS + ks * slice.d * 16) + h;
    const float4 *v = reinterpret_cast<const float4 *>(smem + PA_WARPS * C::RING + C::PARTS) + c;
    float top = -INFINITY, L = 0.f, A[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int r = 0; r < ks; r++) top = fmaxf(top, ml[r * P::HEADS].x);
    if (top == -INFINITY) top = 0.f;
#pragma unroll 4
    for (int r = 0; r < ks; r++) {
      const float2 x = ml[r * P::HEADS];
      const float4 y = v[r * slice.d];
      const float e = ex2(x.x - top);
      L = fmaf(e, x.y, L), A[0] = fmaf(e, y.x, A[0]), A[1] = fmaf(e, y.y, A[1]), A[2] = fmaf(e, y.z, A[2]), A[3] = fmaf(e, y.w, A[3]);
    }
    store4(out + i, A, L);
  }
}

// The pieces of a unit that was cut, in order: piece 0 is the second of the CTA where it begins, piece i the first of the i-th CTA after it.
// A warp takes a head of it, eight pieces at a time, all of whose loads are on their way together; a CTA's warps have one head of
// neighbouring CTAs' units.  The pieces of a unit over many CTAs are shared out among the warps (no more than one such unit can begin in
// eight neighbouring CTAs) and their results meet in shared memory.
constexpr int PJ_WARPS = 8, PJ_BATCH = 8, PJ_FEW = 2 * PJ_BATCH;

template <typename T, int NV>  // heads of up to 128 NV
__global__ void __launch_bounds__(PJ_WARPS * 32, NV == 1 ? 3 : 2) paged_join_kernel(SplitArgs s, int HEADS, int ctas) {
  __shared__ float part[PJ_WARPS][128 * NV + 4];
  __shared__ int many;  // the CTA whose unit has many pieces, or -1
  pdl_launch_dependents();
  pdl_wait();
  const PagedArgs &a = s.p;
  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) many = -1;
  __syncthreads();
  float top, L, acc[NV][4];
  auto fold = [&](int cta, int n, int from, int step) {  // pieces from, from + 1, .. from + 7, from + step, ..
    top = -INFINITY, L = 0.f;
#pragma unroll
    for (int x = 0; x < NV; x++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[x][e] = 0.f;
#pragma unroll 1
    for (int i0 = from; i0 < n; i0 += step) {
      float2 ml[PJ_BATCH];
      float4 v[PJ_BATCH][NV];
      float mx = top;
#pragma unroll
      for (int j = 0; j < PJ_BATCH; j++) {
        const int i = i0 + j;
        ml[j] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int x = 0; x < NV; x++) v[j][x] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < n) {
          const long long at = (i == 0 ? 2ll * cta + 1 : 2ll * (cta + i)) * HEADS + h;
          ml[j] = *reinterpret_cast<const float2 *>(s.ml + 2 * at);
#pragma unroll
          for (int x = 0; x < NV; x++)
            if (4 * lane + 128 * x < a.D) v[j][x] = *reinterpret_cast<const float4 *>(s.acc + at * a.D + 4 * lane + 128 * x);
        }
      }
#pragma unroll
      for (int j = 0; j < PJ_BATCH; j++) mx = fmaxf(mx, ml[j].x);
      const float use = mx == -INFINITY ? 0.f : mx, corr = ex2(top - use);
      top = mx, L *= corr;
#pragma unroll
      for (int x = 0; x < NV; x++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[x][e] *= corr;
#pragma unroll
      for (int j = 0; j < PJ_BATCH; j++) {
        const float w = ex2(ml[j].x - use);
        L = fmaf(w, ml[j].y, L);
#pragma unroll
        for (int x = 0; x < NV; x++)
          acc[x][0] = fmaf(w, v[j][x].x, acc[x][0]), acc[x][1] = fmaf(w, v[j][x].y, acc[x][1]), acc[x][2] = fmaf(w, v[j][x].z, acc[x][2]), acc[x][3] = fmaf(w, v[j][x].w, acc[x][3]);
      }
    }
  };
  auto out_of = [&](const int4 &head) { return static_cast<T *>(a.out) + ((long long)head.x * a.NH + head.y + h) * a.D; };
  const int cta = blockIdx.x * PJ_WARPS + warp;
  const int4 head = cta < ctas ? s.heads[cta] : make_int4(0, 0, 0, 0);
  if (head.w > PJ_FEW && h < head.z) {
    if (lane == 0) many = cta;
  } else if (head.w > 0 && h < head.z) {
    fold(cta, head.w, 0, PJ_BATCH);
#pragma unroll
    for (int x = 0; x < NV; x++)
      if (4 * lane + 128 * x < a.D) store4(out_of(head) + 4 * lane + 128 * x, acc[x], L);
  }
  __syncthreads();
  if (many < 0) return;
  const int4 big = s.heads[many];
  T *const out = out_of(big);
  fold(many, big.w, warp * PJ_BATCH, PJ_WARPS * PJ_BATCH);
  if (lane == 0) part[warp][0] = top, part[warp][1] = L;
#pragma unroll
  for (int x = 0; x < NV; x++)
    if (4 * lane + 128 * x < a.D) *reinterpret_cast<float4 *>(&part[warp][4 + 4 * lane + 128 * x]) = make_float4(acc[x][0], acc[x][1], acc[x][2], acc[x][3]);
  __syncthreads();
  top = -INFINITY, L = 0.f;
#pragma unroll
  for (int w = 0; w < PJ_WARPS; w++) top = fmaxf(top, part[w][0]);
  if (top == -INFINITY) top = 0.f;
#pragma unroll
  for (int w = 0; w < PJ_WARPS; w++) L = fmaf(ex2(part[w][0] - top), part[w][1], L);
  for (int d = threadIdx.x; d < a.D; d += PJ_WARPS * 32) {
    float A = 0.f;
#pragma unroll
    for (int w = 0; w < PJ_WARPS; w++) A = fmaf(ex2(part[w][0] - top), part[w][4 + d], A);
    out[d] = from_f32<T>(L == 0.f ? 0.f : A / L);
  }
}

// How a call is cut: heads per unit, CTAs, whether a unit can be cut, and the scratch that takes.
struct Cut {
  bool streamed;       // the kernel above, else the one for any stride
  int hpg, groups, DP, HEADS, ctas;
  int ks;              // CTAs of a cluster that takes a unit; 0: the split kernel
  bool joined;
  uint32_t unit;
  size_t ml_at, acc_at, bytes;
};

Cut cut_of(const lb200_paged_attn_args *p) {
  Cut c{};
  const int size = p->dtype == LB200_F32 ? 4 : 2, G = p->NH / p->KH;
  uint64_t off = (uint64_t)(uintptr_t)p->q | (uint64_t)(uintptr_t)p->k | (uint64_t)(uintptr_t)p->v | (uint64_t)(uintptr_t)p->out;
  const long long nq[2] = {p->B, p->NH}, nk[3] = {p->pages, p->KH, p->page_size};
  for (int i = 0; i < 2; i++) off |= nq[i] > 1 ? (uint64_t)p->q_stride[i] * size : 0;  // (the stride of an extent of one moves nothing)
  for (int i = 0; i < 3; i++) off |= nk[i] > 1 ? (uint64_t)p->k_stride[i] * size | (uint64_t)p->v_stride[i] * size : 0;
  // a row's offset in the largest unit that divides all strides has to fit 32 bits: with rows of 32 bytes or more, 128 GB
  uint64_t all = 0, far[2] = {0, 0};
  for (int i = 0; i < 3; i++)
    if (nk[i] > 1) {
      all |= (uint64_t)p->k_stride[i] * size | (uint64_t)p->v_stride[i] * size;
      far[0] += (uint64_t)(nk[i] - 1) * (uint64_t)p->k_stride[i] * size, far[1] += (uint64_t)(nk[i] - 1) * (uint64_t)p->v_stride[i] * size;
      if (p->k_stride[i] < 0 || p->v_stride[i] < 0) off |= 1;
    }
  c.unit = 16;
  while (c.unit < 4096 && !(all & c.unit)) c.unit *= 2;
  c.streamed = p->D % 16 == 0 && !(off & 15) && (far[0] > far[1] ? far[0] : far[1]) / c.unit <= 0xffffffffull;
  if (!c.streamed) return c;
  c.DP = p->D <= 64 ? 64 : p->D <= 128 ? 128 : 256;
  const int most = size == 2 ? 16 : c.DP == 256 ? 4 : 8;  // heads per unit: what the registers hold
  c.groups = (G + most - 1) / most, c.hpg = (G + c.groups - 1) / c.groups, c.groups = (G + c.hpg - 1) / c.hpg;
  c.HEADS = size == 4 ? (c.hpg <= 1 ? 1 : c.hpg <= 2 ? 2 : c.hpg <= 4 ? 4 : 8) : (c.hpg <= 8 ? 8 : 16);
  long long keys = (long long)p->W * p->page_size;
  if (p->window > 0 && p->window < keys) keys = p->window;
  const long long blocks = (keys + (size == 4 ? 7 : 15)) / (size == 4 ? 8 : 16);
  if ((blocks + UNIT) * p->B > 0x7fffffffll) {  // (the schedule counts a unit's blocks over all sequences in 32 bits)
    c.streamed = false;
    return c;
  }
  const long long slots = (long long)split_ctas(size, c.DP, c.HEADS) * sm_count();
  // A cluster to a unit where all are resident at once and a warp has CLUSTER_BLOCKS blocks at most.  Up to there it is the faster one whatever
  // the lengths (bf16, 8 KV heads, us of the split kernel and of this one: 1 x 2048 keys 7.9, 6.2; 4 x 1024 9.2, 6.8; 16 x 512 12.1, 10.6);
  // with more blocks it gains less on sequences of one length (4 x 4096: 18.7, 16.9) than it loses on others (4 x 8192 ragged: 12.5, 21.2).
  // The table's width stands for the lengths here, which the host does not know: under a table for 8192 tokens or more 1 x 1024 keys take 8.2 us instead of
  // 5.1, 4 x 1024 9.2 instead of 6.4, 16 x 512 12.1 instead of 9.0.
  const long long n_units = (long long)p->B * p->KH * c.groups;
  for (c.ks = 1; c.ks < 8 && n_units * (c.ks + 1) <= slots && blocks > c.ks * PA_WARPS;) c.ks++;
  if (c.ks == 8 && n_units <= CLUSTER_WIDE && blocks > 8 * PA_WARPS) c.ks = 16;  // (1 x 2048: 7.2 -> 6.2, 1 x 4096: 10.7 -> 8.4)
  if (n_units * c.ks <= slots && blocks <= (long long)c.ks * PA_WARPS * CLUSTER_BLOCKS) return c;
  c.ks = 0;
  const double most_work = (double)p->B * p->KH * c.groups * (double)(blocks + UNIT) / PA_WARPS;  // CTAs' worth, were every sequence as long as the table
  c.ctas = (int)slots;
  if (most_work < c.ctas) c.ctas = most_work < 1 ? 1 : (int)most_work;
  c.joined = blocks > 1 && c.ctas > 1;
  if (c.joined) {
    c.ml_at = ((size_t)c.ctas * sizeof(int4) + 255) & ~(size_t)255;
    c.acc_at = (c.ml_at + (size_t)c.ctas * 2 * c.HEADS * 2 * 4 + 255) & ~(size_t)255;
    c.bytes = c.acc_at + (size_t)c.ctas * 2 * c.HEADS * p->D * 4;
  }
  return c;
}

template <typename P>
int launch_cluster(const SplitArgs &s, const Cut &c, cudaStream_t st) {
  auto kern = paged_attn_cluster_kernel<P>;
  static DeviceOnce once;
  cudaError_t e = once.ensure([&] {
    const cudaError_t f = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return f != cudaSuccess ? f : cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ClusterCfg<P>::SMEM);
  });
  if (e != cudaSuccess) return fail((int)e, "light_b200: paged_decode_attn: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(s.p.B * s.p.KH * s.groups * c.ks)), cfg.blockDim = dim3(PA_THREADS), cfg.dynamicSmemBytes = ClusterCfg<P>::SMEM, cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)c.ks, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = c.ks > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, s, c.ks, FastDiv((c.hpg * s.p.D / 4 + c.ks - 1) / c.ks));
  if (e != cudaSuccess) return fail((int)e, "light_b200: paged_decode_attn: %s", cudaGetErrorString(e));
  return launched("paged_decode_attn");
}

template <typename P>
int launch_split(const SplitArgs &s, const Cut &c, cudaStream_t st) {
  if (c.ks) return launch_cluster<P>(s, c, st);
  auto kern = paged_attn_kernel<P>;
  static DeviceOnce once;
  cudaError_t e = once.ensure([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SplitCfg<P>::SMEM); });
  if (e != cudaSuccess) return fail((int)e, "light_b200: paged_decode_attn: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)c.ctas), cfg.blockDim = dim3(PA_THREADS), cfg.dynamicSmemBytes = SplitCfg<P>::SMEM, cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, s);
  if (e != cudaSuccess) return fail((int)e, "light_b200: paged_decode_attn: %s", cudaGetErrorString(e));
  if (int rc = launched("paged_decode_attn")) return rc;
  if (!c.joined) return 0;
  const dim3 grid((unsigned)((c.ctas + PJ_WARPS - 1) / PJ_WARPS), (unsigned)c.hpg), block(PJ_WARPS * 32);
  if constexpr (P::DP <= 128) e = launch_early(paged_join_kernel<typename P::T, 1>, grid, block, st, s, c.HEADS, c.ctas);
  else e = launch_early(paged_join_kernel<typename P::T, 2>, grid, block, st, s, c.HEADS, c.ctas);
  if (e != cudaSuccess) return fail((int)e, "light_b200: paged_decode_attn: %s", cudaGetErrorString(e));
  return launched("paged_decode_attn (join)");
}

template <int DP>
int launch_dtype(const SplitArgs &s, const Cut &c, int dtype, cudaStream_t st) {
  if (dtype == LB200_BF16) return c.HEADS == 8 ? launch_split<MmaBlock<__nv_bfloat16, DP, 1>>(s, c, st) : launch_split<MmaBlock<__nv_bfloat16, DP, 2>>(s, c, st);
  if (dtype == LB200_F16) return c.HEADS == 8 ? launch_split<MmaBlock<__half, DP, 1>>(s, c, st) : launch_split<MmaBlock<__half, DP, 2>>(s, c, st);
  switch (c.HEADS) {
    case 1: return launch_split<F32Block<DP, 1>>(s, c, st);
    case 2: return launch_split<F32Block<DP, 2>>(s, c, st);
    case 4: return launch_split<F32Block<DP, 4>>(s, c, st);
  }
  if constexpr (DP < 256) return launch_split<F32Block<DP, 8>>(s, c, st);
  return fail(LB200_E_SHAPE, "light_b200: paged_decode_attn: %d heads per unit", c.HEADS);
}

}  // namespace

unsigned long long paged_attn_scratch_bytes(const lb200_paged_attn_args *p) {
  return p->B > 0 ? cut_of(p).bytes : 0;
}

int paged_attn_check(const lb200_paged_attn_args *p) {
  if (!p) return fail(LB200_E_NULL, "light_b200: paged_decode_attn: null argument block");
  if (p->dtype != LB200_F32 && p->dtype != LB200_BF16 && p->dtype != LB200_F16) return fail(LB200_E_DTYPE, "light_b200: paged_decode_attn: element type %d", p->dtype);
  if (p->B < 0 || p->NH <= 0 || p->KH <= 0 || p->NH % p->KH || p->D <= 0 || p->D > PL_MAX_D || p->page_size <= 0 || p->W <= 0 || p->pages <= 0 || p->window < 0 ||
      p->table_stride < p->W || !(p->softcap == 0.f || (p->softcap >= 1e-20f && p->softcap <= 1e20f)))
    return fail(LB200_E_SHAPE, "light_b200: paged_decode_attn: B %d NH %d KH %d D %d (at most %d) page size %d table %d pages %lld window %d softcap %g", p->B, p->NH, p->KH,
                p->D, PL_MAX_D, p->page_size, p->W, (long long)p->pages, p->window, (double)p->softcap);
  // scale log2 e and scale / softcap are f32: infinite, they make NaN of a score of 0
  if (!(fabsf(p->scale) <= 1e38f) || (p->softcap > 0.f && !(fabsf(p->scale) / p->softcap <= 1e38f)))
    return fail(LB200_E_SHAPE, "light_b200: paged_decode_attn: scale %g, softcap %g: want a scale, and with a softcap its share of it, up to 1e38", (double)p->scale, (double)p->softcap);
  if ((long long)p->W * p->page_size > 0x7ffffc00ll || p->pages > 0x7fffffffll || (long long)p->B * p->NH > 0x7fffffffll)
    return fail(LB200_E_TOO_LARGE, "light_b200: paged_decode_attn: %d pages of %d rows per sequence, %lld pages, %d x %d heads: want fewer than 2^31 of each", p->W,
                p->page_size, (long long)p->pages, p->B, p->NH);
  if (p->B > 0 && (!p->q || !p->k || !p->v || !p->block_table || !p->lens || !p->out)) return fail(LB200_E_NULL, "light_b200: paged_decode_attn: null pointer");
  return 0;
}

int paged_decode_attn(const lb200_paged_attn_args *p, cudaStream_t st) {
  if (p->B == 0) return 0;
  PagedArgs a{};
  a.q = p->q, a.k = p->k, a.v = p->v, a.out = p->out, a.table = p->block_table, a.lens = p->lens;
  for (int i = 0; i < 2; i++) a.q_s[i] = p->q_stride[i];
  for (int i = 0; i < 3; i++) a.ks[i] = p->k_stride[i], a.vs[i] = p->v_stride[i];
  a.table_stride = p->table_stride, a.pages = p->pages, a.B = p->B, a.NH = p->NH, a.KH = p->KH, a.G = p->NH / p->KH, a.D = p->D, a.W = p->W, a.window = p->window;
  a.scale = p->scale, a.softcap = p->softcap, a.page = FastDiv(p->page_size);
  const Cut c = cut_of(p);
  if (c.streamed) {
    if (c.bytes && (!p->scratch || p->scratch_bytes < c.bytes || ((uintptr_t)p->scratch & 255)))
      return fail(p->scratch ? LB200_E_SHAPE : LB200_E_NULL, "light_b200: paged_decode_attn: %llu bytes of scratch, want %llu, 256-byte aligned", p->scratch_bytes,
                  (unsigned long long)c.bytes);
    SplitArgs s{};
    s.p = a, s.hpg = c.hpg, s.groups = c.groups, s.unit = c.unit, s.alike = true;
    const long long nk[3] = {p->pages, p->KH, p->page_size};
    const int size = p->dtype == LB200_F32 ? 4 : 2;
    for (int i = 0; i < 3; i++) {
      s.ku[i] = nk[i] > 1 ? (uint32_t)((uint64_t)p->k_stride[i] * size / c.unit) : 0, s.vu[i] = nk[i] > 1 ? (uint32_t)((uint64_t)p->v_stride[i] * size / c.unit) : 0;
      s.alike = s.alike && s.ku[i] == s.vu[i];
    }
    if (c.joined) {
      s.heads = static_cast<int4 *>(p->scratch);
      s.ml = reinterpret_cast<float *>(static_cast<char *>(p->scratch) + c.ml_at), s.acc = reinterpret_cast<float *>(static_cast<char *>(p->scratch) + c.acc_at);
    }
    return c.DP == 64 ? launch_dtype<64>(s, c, p->dtype, st) : c.DP == 128 ? launch_dtype<128>(s, c, p->dtype, st) : launch_dtype<256>(s, c, p->dtype, st);
  }
  const dim3 grid((unsigned)(p->B * p->NH)), block(PL_WARPS * 32);
  cudaError_t e = p->dtype == LB200_F32    ? launch_early(paged_attn_any_kernel<float>, grid, block, st, a)
                  : p->dtype == LB200_BF16 ? launch_early(paged_attn_any_kernel<__nv_bfloat16>, grid, block, st, a)
                                           : launch_early(paged_attn_any_kernel<__half>, grid, block, st, a);
  if (e != cudaSuccess) return fail((int)e, "light_b200: paged_decode_attn: %s", cudaGetErrorString(e));
  return launched("paged_decode_attn");
}

int paged_attn_status(unsigned int *bits, bool clear) {
  return clear ? taken_status(g_attn_status, bits) : (int)cudaMemcpyFromSymbol(bits, g_attn_status, sizeof(*bits));
}

}  // namespace lb
