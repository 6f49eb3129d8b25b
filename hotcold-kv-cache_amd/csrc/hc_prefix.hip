// Attention of a batch behind one shared prompt: host side and C ABI.
#include <algorithm>

#include "hc_common.h"

namespace hc {

int page_shift(int64_t P);   // hc_pages.hip

struct PrefixArgs {
  const void* q;
  int64_t q_sn, q_sh;
  const void* kp;
  int64_t kp_sh, kp_ss;
  const void* vp;
  int64_t vp_sh, vp_ss;
  const int32_t* prefix_lens;
  const void* kg;
  int64_t kg_sp, kg_sh, kg_ss;
  const void* vg;
  int64_t vg_sp, vg_sh, vg_ss;
  const int32_t* tables;
  int64_t t_sb;
  const int32_t* lens;
  const int32_t* cu;
  void* out;
  int64_t o_sn, o_sh;
  float* lse;
  int64_t l_sn, l_sh;
  int64_t num_pages;
  float scaling;
  int N, B, G, D, S, T, lp;
};

// One workgroup per (token, query head): 256 keys at a time, a thread per
// key, then a thread per (dimension, part of the keys).
template <typename T>
__global__ __launch_bounds__(256) void prefix_attn_kernel(PrefixArgs a) {
  __shared__ float s_q[128], s_p[256], s_red[8], s_acc[256];
  __shared__ int64_t s_voff[256];
  const int n = blockIdx.x, h = blockIdx.y, hk = h / a.G, tid = threadIdx.x;
  int b = n, c1 = n + 1;
  if (a.cu) {
    if (n >= min(a.cu[a.B], a.N)) return;
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu[mid] <= n) lo = mid; else hi = mid - 1;
    }
    b = lo;
    c1 = a.cu[lo + 1];
  }
  const int S = a.prefix_lens ? min(max(a.prefix_lens[b], 0), a.S) : a.S;
  const int len = min(max(a.lens[b], 0), a.T << a.lp);
  const int own = max(0, len - (c1 - 1 - n));
  const T* q = (const T*)a.q + n * a.q_sn + h * a.q_sh;
  for (int d = tid; d < a.D; d += 256) s_q[d] = to_f32(q[d]) * a.scaling;
  const int parts = 256 / a.D, d = tid % a.D, part = tid / a.D;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int64_t k0 = 0; k0 < (int64_t)S + own; k0 += 256) {
    __syncthreads();
    const int64_t key = k0 + tid;
    float x = -INFINITY;
    int64_t voff = -1;
    const T* kr = nullptr;
    if (key < S) {
      kr = (const T*)a.kp + hk * a.kp_sh + key * a.kp_ss;
      voff = hk * a.vp_sh + key * a.vp_ss;
    } else if (key < (int64_t)S + own) {
      const int r = (int)(key - S);
      const int64_t page = a.tables[b * a.t_sb + (r >> a.lp)];
      const int row = r & ((1 << a.lp) - 1);
      if (page >= 0 && page < a.num_pages) {
        kr = (const T*)a.kg + page * a.kg_sp + hk * a.kg_sh + row * a.kg_ss;
        voff = page * a.vg_sp + hk * a.vg_sh + row * a.vg_ss;
      }
    }
    if (kr) {
      x = 0.f;
      for (int i = 0; i < a.D; ++i) x += s_q[i] * to_f32(kr[i]);
    }
    s_voff[tid] = voff;
    float t = wave_max(x);
    if ((tid & 63) == 0) s_red[tid >> 6] = t;
    __syncthreads();
    t = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float mn = fmaxf(m, t);
    const float p = kr ? expf(x - mn) : 0.f;
    s_p[tid] = p;
    t = wave_sum(p);
    if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = t;
    __syncthreads();
    const float alpha = mn == -INFINITY ? 1.f : expf(m - mn);
    l = l * alpha + (s_red[4] + s_red[5] + s_red[6] + s_red[7]);
    acc *= alpha;
    m = mn;
    if (part < parts)
      for (int j = part; j < 256; j += parts) {
        const int64_t v = s_voff[j];
        if (v >= 0) {
          const T* base = k0 + j < S ? (const T*)a.vp : (const T*)a.vg;
          acc += s_p[j] * to_f32(base[v + d]);
        }
      }
  }
  __syncthreads();
  s_acc[tid] = acc;
  __syncthreads();
  if (tid < a.D) {
    float t = 0.f;
    for (int j = 0; j < parts; ++j) t += s_acc[j * a.D + tid];
    ((T*)a.out)[n * a.o_sn + h * a.o_sh + tid] = from_f32<T>(l == 0.f ? 0.f : t / l);
  }
  if (tid == 0 && a.lse) a.lse[n * a.l_sn + h * a.l_sh] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace hc

using namespace hc;

extern "C" int64_t hc_prefix_attn_args_size(void) { return (int64_t)sizeof(hc_prefix_attn_args); }

static int check_args(const hc_prefix_attn_args* x) {
  HC_REQUIRE(x != nullptr, "prefix_attention: null argument struct");
  HC_REQUIRE(x->dtype == HC_DTYPE_F32 || x->dtype == HC_DTYPE_F16 || x->dtype == HC_DTYPE_BF16,
             "prefix_attention: bad dtype %lld", (long long)x->dtype);
  HC_REQUIRE(x->N >= 0 && x->N <= (1 << 20) && x->B >= 1 && x->B <= 65536,
             "prefix_attention: N=%lld outside [0, 2^20] or B=%lld outside [1, 65536]", (long long)x->N, (long long)x->B);
  HC_REQUIRE(x->Hk >= 1 && x->Hq >= x->Hk && x->Hq <= 1024, "prefix_attention: Hq=%lld, Hk=%lld", (long long)x->Hq,
             (long long)x->Hk);
  if (x->Hq % x->Hk != 0)
    return set_error(HC_ERR_GROUP, "prefix_attention: Hq (%lld) must be a multiple of Hk (%lld)", (long long)x->Hq,
                     (long long)x->Hk);
  if (x->D != 16 && x->D != 32 && x->D != 64 && x->D != 128)
    return set_error(HC_ERR_UNSUPPORTED, "prefix_attention: head dimension %lld (16, 32, 64 and 128 are supported)",
                     (long long)x->D);
  HC_REQUIRE(x->prefix_rows >= 0 && x->prefix_rows <= ((int64_t)1 << 30), "prefix_attention: %lld prompt rows",
             (long long)x->prefix_rows);
  const int lp = page_shift(x->page_size);
  HC_REQUIRE(lp >= 0, "prefix_attention: page size %lld must be a power of two up to 65536", (long long)x->page_size);
  HC_REQUIRE(x->num_pages >= 1 && x->num_pages <= INT32_MAX, "prefix_attention: %lld pages", (long long)x->num_pages);
  HC_REQUIRE(x->table_width >= 1 && x->table_width <= (((int64_t)1 << 30) >> lp) && x->t_sb >= x->table_width,
             "prefix_attention: table rows of %lld pages of %lld rows, row stride %lld", (long long)x->table_width,
             (long long)x->page_size, (long long)x->t_sb);
  HC_REQUIRE(x->cu_new || x->N == x->B, "prefix_attention: without cu_new every request has one token (N=%lld, B=%lld)",
             (long long)x->N, (long long)x->B);
  HC_REQUIRE(x->max_new >= 1 && (x->cu_new || x->max_new == 1), "prefix_attention: max_new=%lld", (long long)x->max_new);
  HC_REQUIRE(x->N == 0 || (x->q && x->out && x->k_pages && x->v_pages && x->tables && x->lens &&
                 (x->prefix_rows == 0 || (x->k_prefix && x->v_prefix))),
             "prefix_attention: null pointer");
  const int64_t es = dtype_size((int)x->dtype);
  const void* ps[] = {x->q, x->k_prefix, x->v_prefix, x->k_pages, x->v_pages, x->out};
  for (const void* p : ps) HC_REQUIRE((uintptr_t)p % 16 == 0, "prefix_attention: rows must be 16-byte aligned");
  const int64_t st[] = {x->q_sn, x->q_sh, x->kp_sh, x->kp_ss, x->vp_sh, x->vp_ss, x->kg_sp, x->kg_sh, x->kg_ss,
                        x->vg_sp, x->vg_sh, x->vg_ss, x->o_sn, x->o_sh};
  for (const int64_t s : st)
    HC_REQUIRE((s * es) % 16 == 0, "prefix_attention: strides must be multiples of 16 bytes (got %lld elements)",
               (long long)s);
  return HC_OK;
}

extern "C" int64_t hc_prefix_attn_workspace_size(const hc_prefix_attn_args* x) { return check_args(x); }

extern "C" int hc_prefix_attn(const hc_prefix_attn_args* x, void* stream) {
  if (const int rc = check_args(x)) return rc;
  if (x->N == 0) return HC_OK;
  const int dtype = (int)x->dtype, lp = page_shift(x->page_size);
  PrefixArgs a{};
  a.q = x->q; a.q_sn = x->q_sn; a.q_sh = x->q_sh;
  a.kp = x->k_prefix; a.kp_sh = x->kp_sh; a.kp_ss = x->kp_ss;
  a.vp = x->v_prefix; a.vp_sh = x->vp_sh; a.vp_ss = x->vp_ss;
  a.prefix_lens = x->prefix_lens;
  a.kg = x->k_pages; a.kg_sp = x->kg_sp; a.kg_sh = x->kg_sh; a.kg_ss = x->kg_ss;
  a.vg = x->v_pages; a.vg_sp = x->vg_sp; a.vg_sh = x->vg_sh; a.vg_ss = x->vg_ss;
  a.tables = x->tables; a.t_sb = x->t_sb; a.lens = x->lens; a.cu = x->cu_new;
  a.out = x->out; a.o_sn = x->o_sn; a.o_sh = x->o_sh;
  a.lse = x->lse; a.l_sn = x->l_sn; a.l_sh = x->l_sh;
  a.num_pages = x->num_pages; a.scaling = (float)x->scaling;
  a.N = (int)x->N; a.B = (int)x->B; a.G = (int)(x->Hq / x->Hk); a.D = (int)x->D; a.S = (int)x->prefix_rows;
  a.T = (int)x->table_width; a.lp = lp;
  const dim3 grid((unsigned)x->N, (unsigned)x->Hq);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HC_DTYPE_F16) prefix_attn_kernel<half_t><<<grid, 256, 0, s>>>(a);
  else if (dtype == HC_DTYPE_BF16) prefix_attn_kernel<bf16_t><<<grid, 256, 0, s>>>(a);
  else prefix_attn_kernel<float><<<grid, 256, 0, s>>>(a);
  return check_launch("prefix_attention");
}
