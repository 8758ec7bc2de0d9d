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

// A score in units of log2 e.  tanh z = 1 - 2 / (e^(2 z) + 1): absolute error of a few 2^-24, which is what a score's error counts by.
struct Scorer {
  float sc, cap;  // without a cap: scale log2 e; with one: 2 log2 e scale / cap, and cap log2 e
  __device__ Scorer(float scale, float softcap) : sc(softcap > 0.f ? 2.f * LOG2E * scale / softcap : scale * LOG2E), cap(softcap * LOG2E) {}
  __device__ __forceinline__ float operator()(float dot) const {
    const float x = dot * sc;
    return cap > 0.f ? cap - cap * 2.f * __fdividef(1.f, exp2f(x) + 1.f) : x;
  }
};

// ------------------------------------------------------------------------------------ any head size, any stride
// A CTA takes a query head, its four warps every fourth key, a lane every 32nd dim.
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
    const float corr = exp2f(m - use), p = exp2f(s - use);
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
  for (int w = 0; w < PL_WARPS; w++) L = fmaf(exp2f(part[w][0] - top), part[w][1], L);
  for (int d = threadIdx.x; d < a.D; d += PL_WARPS * 32) {
    float A = 0.f;
#pragma unroll
    for (int w = 0; w < PL_WARPS; w++) A = fmaf(exp2f(part[w][0] - top), part[w][2 + d], A);
    static_cast<T *>(a.out)[(long long)blockIdx.x * a.D + d] = from_f32<T>(L == 0.f ? 0.f : A / L);
  }
}

}  // namespace

unsigned long long paged_attn_scratch_bytes(const lb200_paged_attn_args *p) {
  (void)p;
  return 0;
}

int paged_attn_check(const lb200_paged_attn_args *p) {
  if (!p) return fail(LB200_E_NULL, "light_b200: paged_decode_attn: null argument block");
  if (p->dtype != LB200_F32 && p->dtype != LB200_BF16 && p->dtype != LB200_F16) return fail(LB200_E_DTYPE, "light_b200: paged_decode_attn: element type %d", p->dtype);
  if (p->B < 0 || p->NH <= 0 || p->KH <= 0 || p->NH % p->KH || p->D <= 0 || p->D > PL_MAX_D || p->page_size <= 0 || p->W <= 0 || p->pages <= 0 || p->window < 0 ||
      p->table_stride < p->W || !(p->softcap >= 0.f))
    return fail(LB200_E_SHAPE, "light_b200: paged_decode_attn: B %d NH %d KH %d D %d (at most %d) page size %d table %d pages %lld window %d softcap %g", p->B, p->NH, p->KH,
                p->D, PL_MAX_D, p->page_size, p->W, (long long)p->pages, p->window, (double)p->softcap);
  if ((long long)p->W * p->page_size > 0x7fffffffll || p->pages > 0x7fffffffll || (long long)p->B * p->NH > 0x7fffffffll)
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
  const dim3 grid((unsigned)(p->B * p->NH)), block(PL_WARPS * 32);
  cudaError_t e = p->dtype == LB200_F32    ? launch_early(paged_attn_any_kernel<float>, grid, block, st, a)
                  : p->dtype == LB200_BF16 ? launch_early(paged_attn_any_kernel<__nv_bfloat16>, grid, block, st, a)
                                           : launch_early(paged_attn_any_kernel<__half>, grid, block, st, a);
  if (e != cudaSuccess) return fail((int)e, "light_b200: paged_decode_attn: %s", cudaGetErrorString(e));
  return launched("paged_decode_attn");
}

int paged_attn_status(unsigned int *bits) { return (int)cudaMemcpyFromSymbol(bits, g_attn_status, sizeof(*bits)); }

}  // namespace lb
