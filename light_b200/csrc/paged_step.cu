// What a step of a serving loop does around its attention over a paged key-value cache: pages for the new tokens, their return, and the
// queries and keys of the new tokens normed, rotated and put in their rows.  The reference keeps one contiguous cache per sequence
// (models/llama.go:438-640) and runs norm and rotation as launches of their own (ops/norm.go:69-111, ops/rope.go:30-77).
#include "paged.cuh"

namespace lb {
namespace {

__device__ unsigned int g_step_status = 0;

// ------------------------------------------------------------------------------------ pages
// Request b holds n_b tokens in held_b = ceil(n_b / P) pages and gets m_b more, which take more_b = ceil((n_b + m_b) / P) - held_b pages:
// those at first_b, first_b + 1, .. from the top of the stack of free ones, first_b = sum of more_a over a < b.  A request whose pages
// the stack does not hold gets none, and as first_b never falls, none after it that needs any.  Token i of the batch belongs to the
// request with starts_b <= i < starts_{b + 1}: a binary search in shared memory.
//
// Two dependent reads (the lengths; then the stack or the table) and the stores bound it: latency.  A step of 256 requests 3.6 us, 43000 tokens of
// 48 prompts 5.4, the return of 900 requests' 95000 pages 5.2.  Every CTA scans the lengths for itself and stores its share.  Where lengths and
// counter are updated in place the CTAs are one cluster, with its barrier between the scan and the stores; else any number of them.
constexpr int PG_THREADS = 1024, PG_MAX_B = LB200_PAGED_MAX_REQUESTS, PG_AHEAD = 4;  // entries of a thread that are on their way together

struct PagesArgs {
  int *table;
  long long table_stride;
  const int *lens, *new_lens;
  const unsigned char *done;
  int *free_pages;
  const int *free_count;
  int *lens_out, *granted, *starts, *count_out;
  long long *positions, *slots;
  int B, W, capacity;  // capacity: entries of free_pages
  FastDiv page;
  long long tokens;
};

struct Two {
  long long a, b;
};
// exclusive prefix of v over the CTA's threads, and the total
__device__ __forceinline__ Two block_scan(Two v, Two &total) {
  __shared__ Two part[PG_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Two x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, x.a, o), b = __shfl_up_sync(0xffffffffu, x.b, o);
    if (lane >= o) x.a += a, x.b += b;
  }
  __syncthreads();  // (part may still be read from the call before)
  if (lane == 31) part[warp] = x;
  __syncthreads();
  Two w = lane < (int)blockDim.x / 32 ? part[lane] : Two{0, 0};  // the warps' sums, summed by every warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, w.a, o), b = __shfl_up_sync(0xffffffffu, w.b, o);
    if (lane >= o) w.a += a, w.b += b;
  }
  total = {__shfl_sync(0xffffffffu, w.a, 31), __shfl_sync(0xffffffffu, w.b, 31)};
  const int upto = max(warp - 1, 0);
  const Two before = {__shfl_sync(0xffffffffu, w.a, upto), __shfl_sync(0xffffffffu, w.b, upto)};
  return {(warp ? before.a : 0) + x.a - v.a, (warp ? before.b : 0) + x.b - v.b};
}

// the b with at[b] <= i < at[b + 1], for at[0] = 0 <= i < at[n]
__device__ __forceinline__ int owner_of(const int *at, int n, int i) {
  int lo = 0, hi = n;  // at[lo] <= i < at[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int saturated(long long v) { return (int)(v < 0x7fffffffll ? v : 0x7fffffffll); }

// all CTAs have read what the stores may overwrite
__device__ __forceinline__ void pages_barrier(bool cluster) {
  if (cluster) umma::cluster_sync();
  else __syncthreads();
}

__global__ void __launch_bounds__(PG_THREADS) paged_advance_kernel(PagesArgs a, bool cluster) {
  extern __shared__ int sm[];
  __shared__ int cut;
  int *starts = sm, *first = sm + a.B + 1, *len = first + a.B + 1;  // len: -1 - n for a request that gets nothing
  pdl_launch_dependents();
  pdl_wait();
  const int rank = blockIdx.x, tid = threadIdx.x, P = a.page.d;
  const int free_now = a.free_count[0], avail = min(max(free_now, 0), a.capacity);
  bool odd = free_now != avail;
  if (tid == 0) cut = 0x7fffffff;
  auto held_of = [&](int n) {
    const int q = a.page.div(n);
    return q + (q * P < n);
  };
  Two carry = {0, 0};
  for (int base = 0; base < a.B; base += blockDim.x) {
    const int b = base + tid;
    int n = 0, m = 0, more = 0;
    bool fits = false;
    if (b < a.B) {
      n = a.lens[b], m = a.new_lens[b];
      odd |= n < 0 || m < 0;
      n = max(n, 0), m = max(m, 0), fits = (long long)n + m <= (long long)a.W * P;
      if (fits) more = held_of(n + m) - held_of(n);
    }
    // (A request whose rows pass `tokens` counts in the sums: so do all after it, of which none can have a token, or so a page.)
    Two total, at = block_scan({m, more}, total);
    if (b < a.B) {
      const long long from = carry.a + at.a, f = carry.b + at.b;
      const bool given = fits && from + m <= a.tokens && (more == 0 || f + more <= avail);
      starts[b] = saturated(from), first[b] = saturated(f), len[b] = given ? n : -1 - n;
      odd |= !given;
      if (!given && more > 0) atomicMin(&cut, saturated(f));  // (a minimum: no order)
    }
    carry.a += total.a, carry.b += total.b;
  }
  if (tid == 0) starts[a.B] = saturated(carry.a), first[a.B] = saturated(carry.b);
  pages_barrier(cluster);
  const int taken = min(cut, first[a.B]);  // pages: those of the requests before the first that does not get its own
  if (odd && rank == 0) atomicOr(&g_step_status, (unsigned)PAGED_REFUSED);

  const int gid = rank * blockDim.x + tid, threads = gridDim.x * blockDim.x;
  for (int b = gid; b < a.B; b += threads) {
    const int l = len[b], m = starts[b + 1] - starts[b];
    a.lens_out[b] = l < 0 ? -1 - l : l + m;
    a.granted[b] = l < 0 ? 0 : m;
    a.starts[b] = starts[b];
  }
  if (gid == 0) a.starts[a.B] = starts[a.B], a.count_out[0] = avail - taken;
  const int given_rows = starts[a.B];
  bool hole = false;  // a page below 0 under a token that got its place, or on its way into the table
  for (long long i0 = gid; i0 < a.tokens; i0 += PG_AHEAD * (long long)threads) {
    int pg[PG_AHEAD], in[PG_AHEAD];
    long long pos[PG_AHEAD];
#pragma unroll
    for (int j = 0; j < PG_AHEAD; j++) {
      const long long i = i0 + j * (long long)threads;
      pg[j] = -1, pos[j] = 0, in[j] = -1;
      if (i < given_rows && i < a.tokens) {
        const int b = owner_of(starts, a.B, (int)i), l = len[b], n = l < 0 ? -1 - l : l;
        pos[j] = (long long)n + ((int)i - starts[b]);
        if (l >= 0) {
          const int w = a.page.div((int)pos[j]), x = w - held_of(n);
          in[j] = (int)pos[j] - w * P;
          pg[j] = x >= 0 ? a.free_pages[avail - 1 - first[b] - x] : a.table[(long long)b * a.table_stride + w];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < PG_AHEAD; j++) {
      const long long i = i0 + j * (long long)threads;
      if (i < a.tokens) a.positions[i] = pos[j], a.slots[i] = pg[j] >= 0 ? (long long)pg[j] * P + in[j] : -1;
      hole |= pg[j] < 0 && in[j] >= 0;
    }
  }
  for (unsigned p0 = gid; p0 < (unsigned)taken; p0 += PG_AHEAD * threads) {  // (after the tokens: their first pages are not among these; 2^31 and a step fit)
    int pg[PG_AHEAD];
#pragma unroll
    for (int j = 0; j < PG_AHEAD; j++) {
      const unsigned p = p0 + j * threads;
      if (p < (unsigned)taken) pg[j] = a.free_pages[avail - 1 - (int)p];
    }
#pragma unroll
    for (int j = 0; j < PG_AHEAD; j++) {
      const unsigned p = p0 + j * threads;
      if (p < (unsigned)taken) {
        const int b = owner_of(first, a.B, (int)p), l = len[b];
        a.table[(long long)b * a.table_stride + held_of(l < 0 ? -1 - l : l) + ((int)p - first[b])] = pg[j];
        hole |= pg[j] < 0;
      }
    }
  }
  if (hole) atomicOr(&g_step_status, (unsigned)PAGED_REFUSED);
}

// The pages of the requests marked done, in order, on top of the stack.
__global__ void __launch_bounds__(PG_THREADS) paged_release_kernel(PagesArgs a, bool cluster) {
  extern __shared__ int sm[];
  int *first = sm, *keep = sm + a.B + 1;
  pdl_launch_dependents();
  pdl_wait();
  const int rank = blockIdx.x, tid = threadIdx.x;
  const int free_now = a.free_count[0], avail = min(max(free_now, 0), a.capacity);
  bool odd = free_now != avail;
  long long carry = 0;
  for (int base = 0; base < a.B; base += blockDim.x) {
    const int b = base + tid;
    int held = 0;
    if (b < a.B) {
      const int n = a.lens[b];
      const bool done = a.done[b];
      keep[b] = done ? 0 : n;
      if (done) {
        const int q = a.page.div(max(n, 0));
        odd |= n < 0 || n > a.W * a.page.d;
        held = min(q + (q * a.page.d < n), a.W);
      }
    }
    Two total, at = block_scan({held, 0}, total);
    if (b < a.B) first[b] = saturated(carry + at.a);
    carry += total.a;
  }
  if (tid == 0) first[a.B] = saturated(carry);
  const int total = (int)min(carry, (long long)(a.capacity - avail));
  odd |= total < carry;
  pages_barrier(cluster);
  if (odd && rank == 0) atomicOr(&g_step_status, (unsigned)PAGED_REFUSED);
  const int gid = rank * blockDim.x + tid, threads = gridDim.x * blockDim.x;
  for (int b = gid; b < a.B; b += threads) a.lens_out[b] = keep[b];
  if (gid == 0) a.count_out[0] = avail + total;
  bool hole = false;  // a page below 0
  for (long long p0 = gid; p0 < total; p0 += PG_AHEAD * (long long)threads) {
    int pg[PG_AHEAD];
#pragma unroll
    for (int j = 0; j < PG_AHEAD; j++) {
      const long long p = p0 + j * (long long)threads;
      if (p < total) {
        const int b = owner_of(first, a.B, (int)p);
        pg[j] = a.table[(long long)b * a.table_stride + ((int)p - first[b])];
      }
    }
#pragma unroll
    for (int j = 0; j < PG_AHEAD; j++) {
      const long long p = p0 + j * (long long)threads;
      if (p < total) a.free_pages[avail + p] = pg[j], hole |= pg[j] < 0;
    }
  }
  if (hole) atomicOr(&g_step_status, (unsigned)PAGED_REFUSED);
}

// `work`: entries at most, beside the requests
int launch_pages(void (*kern)(PagesArgs, bool), const PagesArgs &a, size_t smem, long long work, cudaStream_t st, DeviceOnce &once, const char *what) {
  cudaError_t e = once.ensure([&] {
    const cudaError_t f = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return f != cudaSuccess ? f : cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (PG_MAX_B * 3 + 2) * 4);
  });
  if (e != cudaSuccess) return fail((int)e, "light_b200: %s: %s", what, cudaGetErrorString(e));
  // as many threads as there are requests or entries, and CTAs where that is more than one's, up to what one cluster or the GPU holds
  const bool inplace = a.lens_out == a.lens || a.count_out == a.free_count;
  const long long want = work > a.B ? work : a.B;
  const int threads = want >= PG_THREADS ? PG_THREADS : (int)((want + 31) / 32 * 32 < 128 ? 128 : (want + 31) / 32 * 32);
  long long ctas = (work + 2 * PG_THREADS - 1) / (2 * PG_THREADS), most = inplace ? 16 : sm_count();
  ctas = ctas < 1 ? 1 : ctas > most ? most : ctas;
  if (inplace)
    while (ctas & (ctas - 1)) ctas &= ctas - 1;  // (a power of two)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas), cfg.blockDim = dim3((unsigned)threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)ctas, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
  const bool cluster = inplace && ctas > 1;
  cfg.attrs = at, cfg.numAttrs = cluster ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, a, cluster);
  if (e != cudaSuccess) return fail((int)e, "light_b200: %s: %s", what, cudaGetErrorString(e));
  return launched(what);
}

// ------------------------------------------------------------------------------------ norm, rotation, cache rows
// y = x rsqrt(mean x^2 + eps) w over the D elements of a head (no weight: y = x), then the first R of them in pairs (a, b):
//   (a cos t - b sin t, a sin t + b cos t) factor,   t = position * inv_freq[i],   pair i = (i, i + R / 2) or (2 i, 2 i + 1).
// f32 from the operand to the one rounding at the end; t in f64 (200000 positions far, an f32 angle is off by 0.01), reduced there to
// half a turn for the f32 functions, which get what that leaves over as a turn of their own.  The angles are the same for every head of a token, so each is computed once.
struct RotateArgs {
  const void *q, *k, *v, *qw, *kw;
  void *q_out, *k_out, *v_out;            // k_out: dense, or the cache's keys with slots
  long long q_s[2], k_s[2], v_s[2];       // token and head strides, elements
  long long ks[3], vs[3];                 // cache strides: page, head, row, elements
  const long long *positions, *slots;
  const double *inv_freq;
  long long T, rows;                      // rows of the cache
  int NH, KH, D, R, interleaved;
  float eps, factor;
  FastDiv page;
};

__device__ __forceinline__ float2 cos_sin(long long pos, double freq) {
  const double t = (double)pos * freq * 0.15915494309189533577;  // in turns: 10^6 radians keep 2^-35 of one
  const double u = 2. * (t - rint(t));                           // in half turns, exact
  const float x = (float)u, d = 3.14159265358979f * (float)(u - (double)x);
  float s, c;
  sincospif(x, &s, &c);
  return make_float2(fmaf(-s, d, c), fmaf(c, d, s));  // what the f32 angle leaves over, d <= pi 2^-25: it is all of a sine or cosine next to a zero
}

constexpr int RT_THREADS = 256, RT_MAX_D = 256;

// Any addresses: a CTA takes a token, a warp a head, a lane every 32nd element; pairs meet in shared memory.  (8192 tokens of 48 bf16 heads of 128:
// 157 us, where the kernel below takes 36.5.)
template <typename T>
__global__ void __launch_bounds__(RT_THREADS) qk_norm_rope_kernel(RotateArgs a) {
  __shared__ float trig[RT_MAX_D];  // cos, sin of R / 2 angles
  __shared__ float rowbuf[RT_THREADS / 32][RT_MAX_D];
  pdl_launch_dependents();
  pdl_wait();
  const long long t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = a.R >> 1;
  const long long pos = a.positions[t];
  for (int i = threadIdx.x; i < half; i += RT_THREADS) {
    const float2 cs = cos_sin(pos, a.inv_freq[i]);
    trig[i] = cs.x * a.factor, trig[half + i] = cs.y * a.factor;
  }
  __syncthreads();
  long long slot = -1;
  int page = 0, row = 0;
  if (a.slots) {
    slot = a.slots[t];
    if (slot >= a.rows) {
      if (threadIdx.x == 0) atomicOr(&g_step_status, (unsigned)PAGED_SLOT);
      slot = -1;
    }
    if (slot >= 0) page = (int)(slot / a.page.d), row = (int)(slot - (long long)page * a.page.d);
  }
  const int heads = a.NH + a.KH + (a.slots ? a.KH : 0);
  float *buf = rowbuf[warp];
  for (int h = warp; h < heads; h += RT_THREADS / 32) {
    if (h >= a.NH && a.slots && slot < 0) break;  // a row without a place: its query alone
    if (h >= a.NH + a.KH) {
      const int kh = h - a.NH - a.KH;
      const T *x = static_cast<const T *>(a.v) + t * a.v_s[0] + kh * a.v_s[1];
      T *y = static_cast<T *>(a.v_out) + page * a.vs[0] + kh * a.vs[1] + row * a.vs[2];
      for (int d = lane; d < a.D; d += 32) y[d] = x[d];
      continue;
    }
    const bool is_q = h < a.NH;
    const int kh = h - a.NH;
    const T *x = is_q ? static_cast<const T *>(a.q) + t * a.q_s[0] + h * a.q_s[1] : static_cast<const T *>(a.k) + t * a.k_s[0] + kh * a.k_s[1];
    const T *w = static_cast<const T *>(is_q ? a.qw : a.kw);
    T *y = is_q ? static_cast<T *>(a.q_out) + (t * a.NH + h) * a.D
                : static_cast<T *>(a.k_out) + (a.slots ? page * a.ks[0] + kh * a.ks[1] + row * a.ks[2] : (t * a.KH + kh) * a.D);
    float ss = 0.f;
    for (int d = lane; d < a.D; d += 32) {
      const float v = to_f32(x[d]);
      buf[d] = v, ss = fmaf(v, v, ss);
    }
    const float inv = w ? rsqrtf(warp_sum(ss) / (float)a.D + a.eps) : 1.f;
    if (w)
      for (int d = lane; d < a.D; d += 32) buf[d] = buf[d] * inv * to_f32(w[d]);
    __syncwarp();  // a lane's pair is another lane's element
    for (int d = lane; d < a.D; d += 32) {
      float r = buf[d];
      if (d < a.R) {
        const int i = a.interleaved ? d >> 1 : (d < half ? d : d - half);
        const bool second = a.interleaved ? d & 1 : d >= half;
        const float o = buf[a.interleaved ? d ^ 1 : (second ? d - half : d + half)];
        r = second ? o * trig[half + i] + r * trig[i] : r * trig[i] - o * trig[half + i];
      }
      y[d] = from_f32<T>(r);
    }
    __syncwarp();
  }
}

// Rows that can be cut into chunks of CB bytes.  A warp takes a token (or, of few tokens, some of a token's heads), lg lanes a head, two chunks each,
// chosen so that the pairs of the rotation are in one lane: chunk c and the one R / 2 elements on, or any two where the pairs are neighbours.  So
// a head is read and written once, in whole sectors, its mean square is log2(lg) shuffles, and an angle's sine and cosine, times the weights,
// stay in registers for all heads of the token: with f, g the lane's chunks and r = rsqrt(mean square + eps)
//   f' = r (f (w_f cos) - g (w_g sin)),  g' = r (f (w_f sin) + g (w_g cos)),
// two elements to an instruction (f32x2).  Bound by the memory, 2 (NH + 2 KH) D elements per token, and nearly by the issue slots (2800
// instructions per token of 48 heads of 128, 1000 of them whatever the head size): 8192 such tokens in bf16 (201 MB) 36.5 us, 5.5 TB/s; 1037 in f32
// 9.6 us, 5.3 TB/s.  Loads into registers two rounds ahead instead of the ring: 45.7 us; a choice of kind at every head: 69 us; registers
// for five or six CTAs an SM: 43 and 57 us (spills); 16 or 1000 warps an SM instead of RC_SLOTS: 40.6, 38.4 us.
constexpr int RC_WARPS = 4, RC_AHEAD = 6, RC_SLOTS = 32;  // rounds of heads that are on their way together; warps on an SM

struct Chunks {
  int lg, split, first, count;  // lanes per head, warps per token; chunks that a lane's second lies behind its first; chunks per head
  int q_parts, k_parts;         // where a warp takes heads of one kind: warps of the queries, and of the keys and of the values
  float over_d;                 // 1 / D
};

template <int CB>
struct Raw {
  uint32_t w[CB / 4];
};
template <int CB>
__device__ __forceinline__ Raw<CB> ld_raw(const void *p) {
  Raw<CB> r;
  if constexpr (CB == 16) {
    const uint4 v = *static_cast<const uint4 *>(p);
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else if constexpr (CB == 8) {
    const uint2 v = *static_cast<const uint2 *>(p);
    r.w[0] = v.x, r.w[1] = v.y;
  } else {
    r.w[0] = *static_cast<const uint32_t *>(p);
  }
  return r;
}
template <int CB>
__device__ __forceinline__ void st_raw(void *p, const Raw<CB> &r) {
  if constexpr (CB == 16) *static_cast<uint4 *>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  else if constexpr (CB == 8) *static_cast<uint2 *>(p) = make_uint2(r.w[0], r.w[1]);
  else *static_cast<uint32_t *>(p) = r.w[0];
}
template <int CB>
__device__ __forceinline__ void cp_chunk(uint32_t dst, const void *src) {
  if constexpr (CB == 16) cp_async16(dst, src);
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(dst), "l"(src), "n"(CB) : "memory");
}
template <int CB>
__device__ __forceinline__ Raw<CB> lds_raw(uint32_t addr) {
  Raw<CB> r;
  if constexpr (CB == 16) {
    const uint4 v = lds128(addr);
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else if constexpr (CB == 8) {
    const uint2 v = lds64(addr);
    r.w[0] = v.x, r.w[1] = v.y;
  } else {
    r.w[0] = lds32(addr);
  }
  return r;
}
template <typename T, int CB>
__device__ __forceinline__ void unpack(const Raw<CB> &r, uint64_t (&f)[CB / sizeof(T) / 2]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < CB / 8; i++) f[i] = (uint64_t)r.w[2 * i + 1] << 32 | r.w[2 * i];
  } else {
#pragma unroll
    for (int i = 0; i < CB / 4; i++) {
      const T *h = reinterpret_cast<const T *>(&r.w[i]);
      f[i] = two(to_f32(h[0]), to_f32(h[1]));
    }
  }
}
__device__ __forceinline__ uint32_t rounded(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t rounded(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T, int CB>
__device__ __forceinline__ Raw<CB> packed(const uint64_t (&f)[CB / sizeof(T) / 2]) {
  Raw<CB> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < CB / 8; i++) r.w[2 * i] = (uint32_t)f[i], r.w[2 * i + 1] = (uint32_t)(f[i] >> 32);
  } else {
#pragma unroll
    for (int i = 0; i < CB / 4; i++) r.w[i] = rounded(lo(f[i]), hi(f[i]), T());
  }
  return r;
}

template <typename T, int CB, bool BETWEEN>
__global__ void __launch_bounds__(RC_WARPS * 32) qk_norm_rope_chunks_kernel(RotateArgs a, Chunks ch) {
  constexpr int E = CB / (int)sizeof(T), V = E / 2;
  __shared__ __align__(16) unsigned char ring[RC_WARPS][RC_AHEAD][2][32][CB];
  __shared__ float2 trig[RC_WARPS][RT_MAX_D / 2];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = a.R >> 1;
  const long long id = (long long)blockIdx.x * RC_WARPS + warp, stride = (long long)gridDim.x * RC_WARPS / ch.split;  // (the host makes it whole)
  long long t = ch.split == 1 ? id : id / ch.split;
  if (t >= a.T) return;
  const int gl = lane & (ch.lg - 1), per = 32 / ch.lg, hl = lane / ch.lg;
  // the kinds (queries, keys, values) of this warp and its part of their heads: every kind, or with many warps per token one
  int part = (int)(id - t * ch.split), parts = ch.split, kind0 = 0, kinds = a.slots ? 3 : 2;
  if (ch.q_parts > 0) {
    kind0 = part < ch.q_parts ? 0 : part < ch.q_parts + ch.k_parts ? 1 : 2, kinds = kind0 + 1, parts = kind0 == 0 ? ch.q_parts : ch.k_parts;
    part -= kind0 == 0 ? 0 : kind0 == 1 ? ch.q_parts : ch.q_parts + ch.k_parts;
  }
  // this lane's chunks, -1 for none
  int c0, c1;
  bool turns = false;  // BETWEEN false: the lane's two chunks are pairs
  if constexpr (BETWEEN) {
    c0 = gl < ch.first ? gl : -1, c1 = gl < ch.first && gl + ch.first < ch.count ? gl + ch.first : -1;
  } else {
    turns = gl < ch.first;
    c0 = turns ? gl : 2 * ch.first + 2 * (gl - ch.first), c1 = turns ? gl + ch.first : c0 + 1;
    if (c0 >= ch.count) c0 = -1;
    if (c1 >= ch.count) c1 = -1;
  }
  // Rounds of `per` heads of a kind, this warp has every parts-th: where this lane's head of the next of them lies, elements from one to the next, and
  // the heads from this lane's on (it has one while left > 0).
  struct Walk {
    T *at;
    long long step;
    int left;
  };
  const int hop = per * parts, h0 = part * per + hl;
  auto source = [&](int kind, long long t) {
    const long long *st = kind == 0 ? a.q_s : kind == 1 ? a.k_s : a.v_s;
    return Walk{static_cast<T *>(const_cast<void *>(kind == 0 ? a.q : kind == 1 ? a.k : a.v)) + t * st[0] + h0 * st[1], hop * st[1], (kind == 0 ? a.NH : a.KH) - h0};
  };
  auto target = [&](int kind, int page, int row) {
    const int left = (kind == 0 ? a.NH : a.KH) - h0;
    if (kind == 0) return Walk{static_cast<T *>(a.q_out) + (t * a.NH + h0) * a.D, (long long)hop * a.D, left};
    if (!a.slots) return Walk{static_cast<T *>(a.k_out) + (t * a.KH + h0) * a.D, (long long)hop * a.D, left};
    const long long *cs = kind == 1 ? a.ks : a.vs;
    return Walk{static_cast<T *>(kind == 1 ? a.k_out : a.v_out) + page * cs[0] + h0 * cs[1] + row * cs[2], hop * cs[1], left};
  };
  // a ring of rounds in shared memory, those of the next token behind this one's: every lane copies and reads its own chunks, so nobody waits for anybody
  const uint32_t mine = umma::smem_u32(ring[warp]) + lane * CB;
  for (int i = 0; i < RC_AHEAD; i++) {  // no chunk: zeros, in the mean square
    if (c0 < 0) *reinterpret_cast<Raw<CB> *>(ring[warp][i][0][lane]) = Raw<CB>{};
    if (c1 < 0) *reinterpret_cast<Raw<CB> *>(ring[warp][i][1][lane]) = Raw<CB>{};
  }
  int far_kind = kind0, slot_far = 0, slot_now = 0;
  long long far_t = t;
  Walk far = source(kind0, t);
  // Past kinds of which this warp has no round (more): a slot of the ring is a round's.  With two warps per token and few query heads, its first kind may
  // be one of those.
  auto settle = [&]() {
    while (far.left + hl <= 0 && far_t < a.T) {  // (the same for the whole warp)
      if (++far_kind == kinds) far_kind = kind0, far_t += stride;
      if (far_t < a.T) far = source(far_kind, far_t);
    }
  };
  auto fetch = [&]() {  // the next round, if there is one
    if (far_t < a.T) {
      if (far.left > 0) {
        const uint32_t dst = mine + slot_far * (64 * CB);
        if (c0 >= 0) cp_chunk<CB>(dst, far.at + c0 * E);
        if (c1 >= 0) cp_chunk<CB>(dst + 32 * CB, far.at + c1 * E);
      }
      far.at += far.step, far.left -= hop;
      settle();
    }
    cp_async_commit();
    slot_far = slot_far + 1 == RC_AHEAD ? 0 : slot_far + 1;
  };
  long long pos = a.positions[t], slot = a.slots ? a.slots[t] : 0;
  settle();
#pragma unroll
  for (int i = 0; i < RC_AHEAD; i++) fetch();  // on their way while the angles are worked out
  Walk to;
  auto take = [&](Raw<CB> &x, Raw<CB> &y) {  // (its copies have been waited for)
    x = lds_raw<CB>(mine + slot_now * (64 * CB)), y = lds_raw<CB>(mine + slot_now * (64 * CB) + 32 * CB);
    slot_now = slot_now + 1 == RC_AHEAD ? 0 : slot_now + 1;
  };
  bool kept = true;
  auto put = [&](const Raw<CB> &u, const Raw<CB> &z) {
    if (to.left > 0 && kept) {
      if (c0 >= 0) st_raw<CB>(to.at + c0 * E, u);
      if (c1 >= 0) st_raw<CB>(to.at + c1 * E, z);
    }
    to.at += to.step, to.left -= hop;
  };
#pragma unroll 1
  for (; t < a.T; t += stride) {
    int page = 0, row = 0;
    if (slot >= a.rows && a.slots) {
      if (lane == 0) atomicOr(&g_step_status, (unsigned)PAGED_SLOT);
      slot = -1;
    }
    if (slot >= 0 && a.slots) page = a.rows <= 0x7fffffffll ? a.page.div((int)slot) : (int)(slot / a.page.d), row = (int)(slot - (long long)page * a.page.d);
    if (kind0 < 2) {
      __syncwarp();  // (the token before is done with its angles)
      for (int i = lane; i < half; i += 32) {
        const float2 cs = cos_sin(pos, a.inv_freq[i]);
        trig[warp][i] = make_float2(cs.x * a.factor, cs.y * a.factor);
      }
      __syncwarp();
    }
    const bool placed = slot >= 0;
    if (t + stride < a.T) pos = a.positions[t + stride], slot = a.slots ? a.slots[t + stride] : 0;
#pragma unroll 1
    for (int kind = kind0; kind < kinds; kind++) {
      to = target(kind, page, row), kept = kind == 0 || placed;
      const T *const w = static_cast<const T *>(kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr);
      if (kind == 2 || !kept) {  // copied as they are, or passed over
        while (to.left + hl > 0) {
          Raw<CB> x, y;
          cp_async_wait<RC_AHEAD - 1>();
          take(x, y);
          put(x, y);
          fetch();
        }
        continue;
      }
      if (to.left + hl <= 0) continue;
      // what f and g are multiplied by: f' = f ff + g gf, g' = f fg + g gg (halves); per chunk x' = x ff + swapped x gf (neighbours: chunk g has fg, gg)
      uint64_t ff[V], gf[V], fg[V], gg[V];
      unsigned turned = 0;  // BETWEEN: bit j: pair j of the first chunk turns; V + j: of the second
      {
        Raw<CB> w0{}, w1{};
        uint64_t wf[V], wg[V];
        if (w && c0 >= 0) w0 = ld_raw<CB>(w + c0 * E);
        if (w && c1 >= 0) w1 = ld_raw<CB>(w + c1 * E);
        unpack<T, CB>(w0, wf), unpack<T, CB>(w1, wg);
#pragma unroll
        for (int j = 0; j < V; j++) {
          if (!w) wf[j] = wg[j] = two(1.f, 1.f);
          if constexpr (BETWEEN) {
            const int i0 = c0 * V + j, i1 = c1 * V + j;
            const bool on0 = c0 >= 0 && i0 < half, on1 = c1 >= 0 && i1 < half;
            const float2 p = on0 ? trig[warp][i0] : make_float2(1.f, 0.f), q = on1 ? trig[warp][i1] : make_float2(1.f, 0.f);
            turned |= (unsigned)on0 << j | (unsigned)on1 << (V + j);
            ff[j] = mul2(wf[j], two(p.x, p.x)), gf[j] = two(-hi(wf[j]) * p.y, lo(wf[j]) * p.y);
            gg[j] = mul2(wg[j], two(q.x, q.x)), fg[j] = two(-hi(wg[j]) * q.y, lo(wg[j]) * q.y);
          } else {
            const float2 p = turns ? trig[warp][c0 * E + 2 * j] : make_float2(1.f, 0.f), q = turns ? trig[warp][c0 * E + 2 * j + 1] : make_float2(1.f, 0.f);
            ff[j] = mul2(wf[j], two(p.x, q.x)), gf[j] = mul2(wg[j], two(-p.y, -q.y)), fg[j] = mul2(wf[j], two(p.y, q.y)), gg[j] = mul2(wg[j], two(p.x, q.x));
          }
        }
      }
      while (to.left + hl > 0) {
        // two rounds side by side, if the kind has two more: a round alone is a chain of some 400 cycles
        const bool both = to.left + hl > hop;
        if (both) cp_async_wait<RC_AHEAD - 2>();
        else cp_async_wait<RC_AHEAD - 1>();
        uint64_t f[2][V], g[2][V];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          Raw<CB> x{}, y{};
          if (i == 0 || both) take(x, y);
          unpack<T, CB>(x, f[i]), unpack<T, CB>(y, g[i]);
        }
        if (w) {
          float ss[2];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            uint64_t s0 = mul2(f[i][0], f[i][0]), s1 = mul2(g[i][0], g[i][0]);
#pragma unroll
            for (int j = 1; j < V; j++) s0 = fma2(f[i][j], f[i][j], s0), s1 = fma2(g[i][j], g[i][j], s1);
            ss[i] = (lo(s0) + hi(s0)) + (lo(s1) + hi(s1));
          }
          for (int o = ch.lg >> 1; o > 0; o >>= 1) {
            const float p = __shfl_xor_sync(0xffffffffu, ss[0], o), q = __shfl_xor_sync(0xffffffffu, ss[1], o);
            ss[0] += p, ss[1] += q;
          }
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const float inv = rsqrtf(ss[i] * ch.over_d + a.eps);
            const uint64_t inv2 = two(inv, inv);
#pragma unroll
            for (int j = 0; j < V; j++) f[i][j] = mul2(f[i][j], inv2), g[i][j] = mul2(g[i][j], inv2);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
          uint64_t u[V], z[V];
#pragma unroll
          for (int j = 0; j < V; j++) {
            u[j] = mul2(f[i][j], ff[j]), z[j] = mul2(g[i][j], gg[j]);
            if constexpr (BETWEEN) {
              if (turned >> j & 1) u[j] = fma2(two(hi(f[i][j]), lo(f[i][j])), gf[j], u[j]);
              if (turned >> (V + j) & 1) z[j] = fma2(two(hi(g[i][j]), lo(g[i][j])), fg[j], z[j]);
            } else if (turns) {
              u[j] = fma2(g[i][j], gf[j], u[j]), z[j] = fma2(f[i][j], fg[j], z[j]);
            }
          }
          if (i == 0 || both) {
            put(packed<T, CB>(u), packed<T, CB>(z));
            fetch();
          }
        }
      }
    }
  }
}

}  // namespace

int paged_pages_check(const lb200_paged_pages *p, const char *what, bool release) {
  if (!p) return fail(LB200_E_NULL, "light_b200: %s: null argument block", what);
  if (!p->block_table || !p->lens || !p->free_pages || !p->free_count || !p->lens_out || !p->free_count_out)
    return fail(LB200_E_NULL, "light_b200: %s: null pointer", what);
  if (release ? !p->done : !p->new_lens || !p->granted || !p->starts || (p->tokens > 0 && (!p->positions || !p->slots)))
    return fail(LB200_E_NULL, "light_b200: %s: null pointer", what);
  if (p->B <= 0 || p->W <= 0 || p->page_size <= 0 || p->capacity <= 0 || p->tokens < 0 || p->table_stride < p->W)
    return fail(LB200_E_SHAPE, "light_b200: %s: %d requests, table of %d pages (stride %lld), page size %d, %d free entries, %lld tokens", what, p->B, p->W,
                (long long)p->table_stride, p->page_size, p->capacity, (long long)p->tokens);
  if (p->B > LB200_PAGED_MAX_REQUESTS) return fail(LB200_E_TOO_LARGE, "light_b200: %s: %d requests, at most %d", what, p->B, LB200_PAGED_MAX_REQUESTS);
  if ((long long)p->W * p->page_size > 0x7fffffffll || p->tokens > 0x7fffffffll)
    return fail(LB200_E_TOO_LARGE, "light_b200: %s: %d pages of %d rows, %lld tokens: want fewer than 2^31", what, p->W, p->page_size, (long long)p->tokens);
  return 0;
}

static PagesArgs pages_args(const lb200_paged_pages *p) {
  PagesArgs a{};
  a.table = p->block_table, a.table_stride = p->table_stride, a.lens = p->lens, a.new_lens = p->new_lens, a.done = p->done;
  a.free_pages = p->free_pages, a.free_count = p->free_count, a.lens_out = p->lens_out, a.granted = p->granted, a.starts = p->starts;
  a.count_out = p->free_count_out, a.positions = (long long *)p->positions, a.slots = (long long *)p->slots;
  a.B = p->B, a.W = p->W, a.capacity = p->capacity, a.page = FastDiv(p->page_size), a.tokens = p->tokens;
  return a;
}

int paged_advance(const lb200_paged_pages *p, cudaStream_t st) {
  static DeviceOnce once;
  return launch_pages(paged_advance_kernel, pages_args(p), (size_t)(3 * p->B + 2) * 4, p->tokens, st, once, "paged_advance");
}

int paged_release(const lb200_paged_pages *p, cudaStream_t st) {
  static DeviceOnce once;
  const long long pages = (long long)p->B * p->W;
  return launch_pages(paged_release_kernel, pages_args(p), (size_t)(2 * p->B + 1) * 4, pages < p->capacity ? pages : p->capacity, st, once, "paged_release");
}

int qk_norm_rope_check(const lb200_qk_norm_rope_args *p) {
  if (!p) return fail(LB200_E_NULL, "light_b200: qk_norm_rope: null argument block");
  if (p->T < 0 || p->NH <= 0 || p->KH <= 0 || p->D <= 0 || p->D > RT_MAX_D || p->rotary < 0 || p->rotary % 2 || p->rotary > p->D)
    return fail(LB200_E_SHAPE, "light_b200: qk_norm_rope: T %lld NH %d KH %d D %d (at most %d) rotary %d (even, at most D)", (long long)p->T, p->NH, p->KH, p->D, RT_MAX_D,
                p->rotary);
  if (p->dtype != LB200_F32 && p->dtype != LB200_BF16 && p->dtype != LB200_F16) return fail(LB200_E_DTYPE, "light_b200: qk_norm_rope: element type %d", p->dtype);
  if (p->T > 0x7fffffffll) return fail(LB200_E_TOO_LARGE, "light_b200: qk_norm_rope: %lld tokens", (long long)p->T);
  if (!(p->eps >= 0.f)) return fail(LB200_E_SHAPE, "light_b200: qk_norm_rope: eps %g", (double)p->eps);
  if (p->slots && (p->pages <= 0 || p->page_size <= 0))
    return fail(LB200_E_SHAPE, "light_b200: qk_norm_rope: cache of %lld pages of %d rows", (long long)p->pages, p->page_size);
  if (p->slots && p->pages > 0x7fffffffll) return fail(LB200_E_TOO_LARGE, "light_b200: qk_norm_rope: %lld pages", (long long)p->pages);
  if (p->T > 0 && (!p->q || !p->k || !p->q_out || !p->k_out || !p->positions || (p->rotary && !p->inv_freq) || (p->slots && (!p->v || !p->v_out))))
    return fail(LB200_E_NULL, "light_b200: qk_norm_rope: null pointer (slots come with v and the cache)");
  return 0;
}

template <typename T, int CB>
static cudaError_t launch_as(const RotateArgs &a, const Chunks &ch, unsigned ctas, cudaStream_t st) {
  return a.interleaved ? launch_early(qk_norm_rope_chunks_kernel<T, CB, true>, dim3(ctas), dim3(RC_WARPS * 32), st, a, ch)
                       : launch_early(qk_norm_rope_chunks_kernel<T, CB, false>, dim3(ctas), dim3(RC_WARPS * 32), st, a, ch);
}
template <typename T>
static cudaError_t launch_cb(const RotateArgs &a, const Chunks &ch, int cb, unsigned ctas, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (cb == 4) return launch_as<T, 4>(a, ch, ctas, st);
  return cb == 16 ? launch_as<T, 16>(a, ch, ctas, st) : launch_as<T, 8>(a, ch, ctas, st);
}
static int launch_chunks(const RotateArgs &a, const Chunks &ch, int cb, int dtype, unsigned ctas, cudaStream_t st) {
  const cudaError_t e = dtype == LB200_F32    ? launch_cb<float>(a, ch, cb, ctas, st)
                        : dtype == LB200_BF16 ? launch_cb<__nv_bfloat16>(a, ch, cb, ctas, st)
                                              : launch_cb<__half>(a, ch, cb, ctas, st);
  if (e != cudaSuccess) return fail((int)e, "light_b200: qk_norm_rope: %s", cudaGetErrorString(e));
  return launched("qk_norm_rope");
}

int qk_norm_rope(const lb200_qk_norm_rope_args *p, cudaStream_t st) {
  if (p->T == 0) return 0;
  RotateArgs a{};
  a.q = p->q, a.k = p->k, a.v = p->v, a.qw = p->q_weight, a.kw = p->k_weight, a.q_out = p->q_out, a.k_out = p->k_out, a.v_out = p->v_out;
  for (int i = 0; i < 2; i++) a.q_s[i] = p->q_stride[i], a.k_s[i] = p->k_stride[i], a.v_s[i] = p->v_stride[i];
  for (int i = 0; i < 3; i++) a.ks[i] = p->k_cache_stride[i], a.vs[i] = p->v_cache_stride[i];
  a.positions = (const long long *)p->positions, a.slots = (const long long *)p->slots, a.inv_freq = p->inv_freq;
  a.T = p->T, a.rows = p->slots ? p->pages * p->page_size : 0, a.NH = p->NH, a.KH = p->KH, a.D = p->D, a.R = p->rotary, a.interleaved = p->interleaved;
  a.eps = p->eps, a.factor = p->factor, a.page = FastDiv(p->slots ? p->page_size : 1);
  // chunks as large as the addresses and the distance of a pair's elements allow
  const int size = p->dtype == LB200_F32 ? 4 : 2;
  uint64_t off = (uint64_t)(uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->q_out | (uintptr_t)p->k_out | (uintptr_t)p->q_weight | (uintptr_t)p->k_weight | (uint64_t)p->D * size;
  for (int i = 0; i < 2; i++) off |= (uint64_t)p->q_stride[i] * size | (uint64_t)p->k_stride[i] * size;
  if (p->slots) {
    off |= (uintptr_t)p->v | (uintptr_t)p->v_out;
    for (int i = 0; i < 2; i++) off |= (uint64_t)p->v_stride[i] * size;
    for (int i = 0; i < 3; i++) off |= (uint64_t)p->k_cache_stride[i] * size | (uint64_t)p->v_cache_stride[i] * size;
  }
  if (!p->interleaved) off |= (uint64_t)(p->rotary / 2) * size;
  int cb = off & 15 ? off & 7 ? off & 3 ? 0 : 4 : 8 : 16;
  if (cb < 2 * size) cb = 0;
  if (cb) {
    Chunks ch{};
    ch.count = p->D * size / cb, ch.over_d = 1.f / (float)p->D;
    ch.first = p->interleaved ? (ch.count + 1) / 2 : p->rotary / 2 * size / cb;
    const int lanes = p->interleaved ? ch.first : ch.first + (ch.count - 2 * ch.first + 1) / 2;
    for (ch.lg = 1; ch.lg < lanes;) ch.lg *= 2;
    if (ch.lg <= 32) {
      // Warps per token: one that has its angles for all heads; two, of fewer than twelve tokens for every SM; of fewer than four, as many as have one to four
      // rounds of one kind each, until there are eight for every SM.  Heads of 128, us with one warp and with two: bf16, 1000 tokens of 48 heads 9.9, 7.7, of
      // 8 heads 6.3, 5.3; F32, 1400 of 48 15.7, 12.3, of 24 9.2, 7.3; beyond the rule (2500) bf16 17.0, 19.5, F32 22.4, 22.6.  It is the worse side for 1400 bf16
      // tokens (48 heads 10.2, 12.7; 8 heads 6.6, 9.5: the second warps no longer fit on the SMs), for 600 F32 tokens of 8 heads (4.9, 5.4) and beyond it for
      // 3500 F32 tokens of 48 (35.2, 31.9).
      const int per = 32 / ch.lg, rq = (p->NH + per - 1) / per, rk = (p->KH + per - 1) / per, kinds = p->slots ? 3 : 2;
      ch.split = p->T < 12ll * sm_count() ? 2 : 1, ch.q_parts = ch.k_parts = 0;
      if (p->T < 4ll * sm_count())
        for (int rounds = rk; rounds >= 1 && p->T * (ch.q_parts ? ch.split : 0) < 8ll * sm_count(); rounds = rounds == 1 ? 0 : (rounds + 1) / 2) {
          ch.q_parts = (rq + rounds - 1) / rounds, ch.k_parts = (rk + rounds - 1) / rounds;
          ch.split = ch.q_parts + (kinds - 1) * ch.k_parts;
        }
      // a warp takes a token after the other, where all of them together have more than RC_SLOTS warps for every SM
      long long ctas = (p->T * ch.split + RC_WARPS - 1) / RC_WARPS;
      if (ch.split == 1 && ctas > (long long)RC_SLOTS / RC_WARPS * sm_count()) ctas = (long long)RC_SLOTS / RC_WARPS * sm_count();
      if (ch.split > 1) ctas = (ctas + ch.split - 1) / ch.split * ch.split;  // (a whole number of tokens at a time)
      return launch_chunks(a, ch, cb, p->dtype, (unsigned)ctas, st);
    }
  }
  cudaError_t e;
  if (p->dtype == LB200_F32) e = launch_early(qk_norm_rope_kernel<float>, dim3((unsigned)p->T), dim3(RT_THREADS), st, a);
  else if (p->dtype == LB200_BF16) e = launch_early(qk_norm_rope_kernel<__nv_bfloat16>, dim3((unsigned)p->T), dim3(RT_THREADS), st, a);
  else e = launch_early(qk_norm_rope_kernel<__half>, dim3((unsigned)p->T), dim3(RT_THREADS), st, a);
  if (e != cudaSuccess) return fail((int)e, "light_b200: qk_norm_rope: %s", cudaGetErrorString(e));
  return launched("qk_norm_rope");
}

int paged_step_status(unsigned int *bits, bool clear) {
  return clear ? taken_status(g_step_status, bits) : (int)cudaMemcpyFromSymbol(bits, g_step_status, sizeof(*bits));
}

}  // namespace lb
