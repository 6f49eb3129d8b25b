// Attention of a batch behind one shared prompt: host side and C ABI.
#include <algorithm>
#include <cmath>

#include "hc_prefix_kernels.h"

namespace hc {

int page_shift(int64_t P);   // hc_pages.hip

extern template void launch_prefix<half_t>(const PrefixArgs&, int64_t, hipStream_t);
extern template void launch_prefix<bf16_t>(const PrefixArgs&, int64_t, hipStream_t);
extern template void launch_prefix<float>(const PrefixArgs&, int64_t, hipStream_t);

constexpr int kCus = 256;

// How a call is laid out over workgroups.
struct PrefixPlan {
  int p_rows, p_tiles, p_splits, p_chunk, o_rows, o_tiles, o_splits, m_tiles, m_sub, both;
  int64_t items, slots;
};

// Query rows of a tile: as many as there are, up to 32 for each wave.
int tile_rows(int64_t rows, int waves) {
  int n = 16;
  while (n < 32 * waves && rows > n) n *= 2;
  return n;
}

// Times of a workgroup, in ns, as measured at head dimension 128 and 2-byte
// types: kWgNs of its own (arguments, first loads, the waves' join), and a
// key's; kSweepNs of a second run of keys, kJoinNs of the partials' join.  One
// CU streams about 40 GB/s, all together kHbmGBs (paged and prompt rows at
// once); products of 32 WR rows take the rest (30 ns a key of 256 rows).
constexpr double kWgNs = 6500, kSweepNs = 3500, kJoinNs = 4500, kCuGBs = 40, kHbmGBs = 4400;

PrefixPlan plan_prefix(const hc_prefix_attn_args* x) {
  PrefixPlan p{};
  const int64_t es = dtype_size((int)x->dtype), G = x->Hq / x->Hk, rows = x->N * G, most = std::min(x->max_new, x->N);
  const int waves = x->D * es >= 512 ? 4 : 8;
  const double key_bytes = 2.0 * (double)(x->D * es);
  auto key_ns = [&](int n) { return std::max(key_bytes / kCuGBs, 0.117 * n * 8 / waves * (double)(x->D * es * es) / 512); };
  p.o_rows = tile_rows(most * G, waves);
  p.o_tiles = (int)cdiv(most * G, p.o_rows);
  // Own items: a request's keys are split only as far as it takes to give every
  // CU some.  Their lengths are on the device; half of what the table holds is
  // taken for the mean.
  const int64_t units = x->B * x->Hk * p.o_tiles, longest = x->table_width * x->page_size;
  p.o_splits = (int)std::max<int64_t>(1, std::min<int64_t>({cdiv((int64_t)kCus / 2, units), cdiv(longest, (int64_t)256), 64}));
  const double own_keys = 0.5 * (double)longest / p.o_splits;
  // (tiles that hold rows: a request's last one is half full)
  const double tiles = std::min((double)(x->B * p.o_tiles), (double)rows / p.o_rows + 0.5 * (double)x->B);
  const double own_n = tiles * (double)(x->Hk * p.o_splits), own_ns = kWgNs + own_keys * key_ns(p.o_rows);
  double two = own_n * own_ns / kCus;   // prompt and own items, and the join
  if (x->prefix_rows > 0) {
    p.p_rows = tile_rows(rows, waves);
    p.p_tiles = (int)cdiv(rows, p.p_rows);
    // (a tile's keys, as in the kernel)
    const int wk = waves * 32 / std::max(32, p.p_rows);
    const int64_t bn = wk * (wk <= waves / 4 ? 64 : 32), units_p = p.p_tiles * x->Hk;
    // Prompt items go first, and the own ones on the CUs they leave; what these
    // have not done by the prompt's end runs on all CUs.  Where both together
    // ask for more than the memory gives, a CU that asks for less than its even
    // part has all it asks for, and the others share the rest.
    const double rate_p = key_bytes / key_ns(p.p_rows), rate_o = key_bytes / key_ns(p.o_rows);
    double best = 0;
    for (int64_t s = 1; s <= 512; s += 1 + s / 12) {
      const int64_t chunk = cdiv(cdiv(x->prefix_rows, s), bn) * bn, splits = cdiv(x->prefix_rows, chunk);
      const double n = (double)(units_p * splits), busy = std::min(n, (double)kCus), left = kCus - busy;
      const double even = kHbmGBs / kCus, bytes_p = (double)chunk * key_bytes, bytes_o = own_keys * key_bytes;
      double gets_p = rate_p, gets_o = rate_o;
      if (busy * rate_p + left * rate_o > kHbmGBs) {
        gets_p = rate_o <= even ? (kHbmGBs - left * rate_o) / busy : std::min(rate_p, even);
        if (left > 0) gets_o = rate_p <= even ? (kHbmGBs - busy * rate_p) / left : std::min(rate_o, even);
      }
      const double beside = kWgNs + bytes_o / gets_o, all_o = left > 0 ? own_n * beside / left : 1e18;
      double t = kWgNs + bytes_p / gets_p;
      if (t > all_o) t = all_o + std::max(0.0, t - all_o) * gets_p / std::min(rate_p, kHbmGBs / busy);
      t *= std::ceil(n / kCus);
      const double rest = std::max(0.0, own_n - left * t / beside);
      if (rest > 0)   // (the last to end may be a request of twice the mean length)
        t += std::max(rest / kCus * own_ns, rest * bytes_o / kHbmGBs) + own_ns - kWgNs;
      t += (double)(splits * rows * x->Hk * x->D * 8) / kHbmGBs;   // partials, written and read
      if (p.p_splits == 0 || t < best) {
        best = t;
        p.p_splits = (int)splits;
        p.p_chunk = (int)chunk;
      }
      if (chunk == bn) break;
    }
    two = best;
  }
  two += kJoinNs + (double)(p.o_splits * rows * x->Hk * x->D * 8) / kHbmGBs;
  // Or each own item takes the prompt as well: no partials, but the prompt once
  // for every request's tile.  (Requests' own prompts of up to 512 tokens behind
  // 64 rows: 94 us -> 61.  Of 1024 behind 8192, where the estimates are close:
  // 802 us apart, 963 together.)  With no prompt and one item a row nothing is joined
  // (256 requests of up to 1024 rows: 145 -> 138 us; 8 prompts of up to
  // 512 tokens: 116 -> 88).
  const double both = std::ceil(tiles * (double)x->Hk / kCus) *
                      (kWgNs + (x->prefix_rows > 0 ? kSweepNs : 0) +
                       ((double)x->prefix_rows + 0.5 * (double)longest) * key_ns(p.o_rows));
  if ((p.both = both < 0.9 * two || (x->prefix_rows == 0 && p.o_splits == 1))) {
    p.p_tiles = p.p_splits = 0;
    p.o_splits = 1;
  }
  const int64_t vec = x->D / 4;   // threads of a row's group
  p.m_sub = x->B * cdiv(most * x->Hq * vec, (int64_t)256) < 2 * kCus && p.p_splits + p.o_splits >= 8 ? kMergeSub : 1;
  p.m_tiles = (int)cdiv(most * x->Hq * vec * p.m_sub, (int64_t)256);
  p.items = (int64_t)p.p_tiles * x->Hk * p.p_splits + units * p.o_splits;
  p.slots = p.both ? 0 : p.p_splits + p.o_splits;   // (rows written complete need no partials)
  return p;
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
  HC_REQUIRE(x->max_new >= 1 && x->max_new <= (1 << 20) && (x->cu_new || x->max_new == 1),
             "prefix_attention: max_new=%lld", (long long)x->max_new);
  HC_REQUIRE(x->N == 0 || (x->q && x->out && x->k_pages && x->v_pages && x->tables && x->lens &&
                 (x->prefix_rows == 0 || (x->k_prefix && x->v_prefix))),
             "prefix_attention: null pointer");
  const int64_t es = dtype_size((int)x->dtype);
  const void* ps[] = {x->q, x->k_prefix, x->v_prefix, x->k_pages, x->v_pages, x->out};
  for (const void* p : ps) HC_REQUIRE((uintptr_t)p % 16 == 0, "prefix_attention: rows must be 16-byte aligned");
  const int64_t st[] = {x->q_sn, x->q_sh, x->kp_sh, x->kp_ss, x->vp_sh, x->vp_ss, x->kg_sp, x->kg_sh, x->kg_ss,
                        x->vg_sp, x->vg_sh, x->vg_ss, x->o_sn, x->o_sh};
  for (const int64_t s : st)
    HC_REQUIRE(s >= 0 && (s * es) % 16 == 0, "prefix_attention: strides must be whole multiples of 16 bytes (got %lld elements)",
               (long long)s);
  // (a load addresses its rows by 32-bit offsets from the first)
  HC_REQUIRE(std::max({x->kp_ss, x->vp_ss, x->kg_ss, x->vg_ss}) * es <= (1 << 25),
             "prefix_attention: key and value rows more than 32 MiB apart");
  return HC_OK;
}

extern "C" int64_t hc_prefix_attn_workspace_size(const hc_prefix_attn_args* x) {
  if (const int rc = check_args(x)) return rc;
  if (x->N == 0) return 0;
  return (plan_prefix(x).slots * x->N * x->Hq * (x->D + 2) + 4) * 4;
}

extern "C" int hc_prefix_attn(const hc_prefix_attn_args* x, void* stream) {
  if (const int rc = check_args(x)) return rc;
  if (x->N == 0) return HC_OK;
  const int64_t need = hc_prefix_attn_workspace_size(x);
  if (!x->workspace || x->workspace_bytes < need)
    return set_error(HC_ERR_WORKSPACE, "prefix_attention: workspace of %lld bytes, %lld needed",
                     (long long)(x->workspace ? x->workspace_bytes : 0), (long long)need);
  HC_REQUIRE((uintptr_t)x->workspace % 16 == 0, "prefix_attention: the workspace must be 16-byte aligned");
  const PrefixPlan p = plan_prefix(x);
  // (a grid's threads are counted in 32 bits)
  HC_REQUIRE(p.items <= UINT32_MAX / 512 && x->B * p.m_tiles <= UINT32_MAX / 256, "prefix_attention: %lld workgroups",
             (long long)std::max(p.items, x->B * p.m_tiles));
  const int dtype = (int)x->dtype;
  const int64_t es = dtype_size(dtype);
  PrefixArgs a{};
  a.q = (const char*)x->q; a.q_sn = x->q_sn * es; a.q_sh = x->q_sh * es;
  a.kp = (const char*)x->k_prefix; a.kp_sh = x->kp_sh * es; a.kp_ss = x->kp_ss * es;
  a.vp = (const char*)x->v_prefix; a.vp_sh = x->vp_sh * es; a.vp_ss = x->vp_ss * es;
  a.kg = (const char*)x->k_pages; a.kg_sp = x->kg_sp * es; a.kg_sh = x->kg_sh * es; a.kg_ss = x->kg_ss * es;
  a.vg = (const char*)x->v_pages; a.vg_sp = x->vg_sp * es; a.vg_sh = x->vg_sh * es; a.vg_ss = x->vg_ss * es;
  a.prefix_lens = x->prefix_lens;
  a.tables = x->tables; a.t_sb = x->t_sb; a.lens = x->lens; a.cu = x->cu_new;
  a.out = (char*)x->out; a.o_sn = x->o_sn * es; a.o_sh = x->o_sh * es;
  a.lse = x->lse; a.l_sn = x->l_sn; a.l_sh = x->l_sh;
  a.part_ml = (float*)x->workspace;
  a.part_o = a.part_ml + (p.slots * x->N * x->Hq * 2 + 3) / 4 * 4;
  const float scale = (float)(std::fabs(x->scaling) * 1.4426950408889634);
  a.scale_log2 = scale == 0.f ? 1.f : scale;
  a.q_and = scale == 0.f ? 0u : ~0u;
  a.q_xor = scale == 0.f || !std::signbit(x->scaling) ? 0u : dtype == HC_DTYPE_F32 ? 0x80000000u : 0x80008000u;
  a.N = (int)x->N; a.B = (int)x->B; a.Hq = (int)x->Hq; a.Hk = (int)x->Hk; a.G = (int)(x->Hq / x->Hk);
  a.D = (int)x->D; a.S = (int)x->prefix_rows; a.T = (int)x->table_width; a.lp = page_shift(x->page_size);
  a.num_pages = (int)x->num_pages;
  a.max_new = (int)std::min<int64_t>(x->max_new, x->N);
  a.p_rows = p.p_rows; a.p_tiles = p.p_tiles; a.p_splits = p.p_splits; a.p_chunk = p.p_chunk;
  a.p_items = p.p_tiles * a.Hk * p.p_splits;
  a.o_rows = p.o_rows; a.o_tiles = p.o_tiles; a.o_splits = p.o_splits; a.both = p.both; a.m_tiles = p.m_tiles; a.m_sub = p.m_sub;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == HC_DTYPE_F16) launch_prefix<half_t>(a, p.items, s);
  else if (dtype == HC_DTYPE_BF16) launch_prefix<bf16_t>(a, p.items, s);
  else launch_prefix<float>(a, p.items, s);
  return check_launch("prefix_attention");
}
