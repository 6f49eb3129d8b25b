// The paged part of the hot tier: block tables and slot maps from request
// lengths, the pages' release, and the append of new rows into their slots.
// (No counterpart in the reference, whose caches are one dense tensor per
// layer with one length for the whole batch, cache.py:145-148.)
//
// A pool holds num_pages pages of P = 2^lp rows.  Request b's row r lives in
// page tables[b][r >> lp] at row r & (P - 1); its slot is page * P + row.
// free_pages[0 .. count) are the pages nobody holds, taken from the end.
#include <algorithm>

#include "hc_common.h"

namespace hc {

constexpr int kPageThreads = 256;
constexpr int kMaxRequests = 4096;   // three words of LDS each
constexpr int kMaxTokens = 1 << 20;  // a chunk's clamped token sum stays below 2^32

struct ExtendArgs {
  const int32_t* lens;
  const int32_t* new_lens;
  int32_t* tables;
  int64_t t_sb;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* lens_out;
  int32_t* count_out;
  int32_t* cu;
  int64_t* slots;
  int64_t* positions;
  int B, T, F, N, lp;
};

// Inclusive sum over the workgroup's threads, in thread order; total gets
// everyone's.  (The leading barrier protects sums from the previous call's
// readers.)
__device__ __forceinline__ uint32_t block_incl_scan(uint32_t x, uint32_t* sums, uint32_t* total) {
  const int wave = threadIdx.x >> 6;
  const uint32_t inc = wave_incl_scan(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sums[wave] = inc;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPageThreads / 64; ++w) {
    if (w < wave) before += sums[w];
    all += sums[w];
  }
  *total = all;
  return before + inc;
}

__device__ __forceinline__ int64_t pages_of(int64_t rows, int lp) { return (rows + ((int64_t)1 << lp) - 1) >> lp; }

// Block tables and slot maps.  Every workgroup scans the requests: token
// offsets cu (the packed batch's), and pages needed before each request.
// With the exclusive page sum x_b, request b's page have_b + k is
// free_pages[count - 1 - x_b - k].  Then each thread takes tokens: its
// request by a search of cu, its page from the old table entry or the free
// list; the token on a page's first row writes the table entry (each new page
// has exactly one such token, and old entries are never written, so the
// workgroups share nothing).
//   kFill: write tables, slots, positions and cu; kCommit: the first workgroup
//   writes lens_out and count_out.  Where several workgroups read the lengths
//   and the count that this replaces (lens_out is lens, or count_out
//   free_count), a second launch of one workgroup commits.
// Bound by latency: two dependent loads, two scans and a search (kernel 3.1 us
// for a step of 16 requests, 3.5 for 256 with 8192 tokens; the launch
// from the host takes 7).
template <bool kFill, bool kCommit>
__global__ __launch_bounds__(kPageThreads) void extend_pages_kernel(ExtendArgs a) {
  extern __shared__ uint32_t sm_words[];
  uint32_t* s_cu = sm_words;                                       // [B + 1]
  uint32_t* s_before = s_cu + a.B + 1;                             // [B]: pages before, or kNone
  int32_t* s_len = reinterpret_cast<int32_t*>(s_before + a.B);     // [B]
  __shared__ uint32_t s_sums[kPageThreads / 64];
  constexpr uint32_t kNone = 0xffffffffu;
  const int tid = threadIdx.x;
  const bool commit = kCommit && blockIdx.x == 0;
  const int count = min(max(*a.free_count, 0), a.F);
  const uint32_t N = (uint32_t)a.N;
  uint32_t tok0 = 0, page0 = 0, used = 0;
  if (tid == 0) s_cu[0] = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPageThreads) {
    const int b = b0 + tid;
    const bool in = b < a.B;
    const int64_t len = in ? a.lens[b] : 0, more = in ? a.new_lens[b] : 0;
    uint32_t total;
    // clamping a request to N + 1 tokens keeps "the sum passes N" as it is
    const uint32_t end = tok0 + block_incl_scan((uint32_t)min(max(more, (int64_t)0), (int64_t)N + 1), s_sums, &total);
    tok0 = min(tok0 + total, N + 1);
    const int64_t have = pages_of(len, a.lp), want = pages_of(len + more, a.lp);
    const bool bad = len < 0 || more < 0 || want > a.T || end > N;
    const uint32_t need = bad ? 0u : (uint32_t)(want - have);
    const uint32_t upto = page0 + block_incl_scan(need, s_sums, &total);
    const bool fits = upto <= (uint32_t)count;
    const bool ok = !bad && (need == 0 || fits);
    page0 += total;
    if (in) {
      s_cu[b + 1] = min(end, N);
      s_before[b] = ok ? upto - need : kNone;
      s_len[b] = (int32_t)len;
      if (kFill && blockIdx.x == 0) a.cu[b + 1] = (int32_t)min(end, N);
      if (commit) a.lens_out[b] = (int32_t)(ok ? len + more : len);
    }
    // the largest sum that fits: sums never fall, so it is what was taken
    if (commit) {
      uint32_t u = fits ? upto : 0u;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) u = max(u, (uint32_t)__shfl_xor((int)u, o, 64));
      used = max(used, u);
    }
  }
  if (commit) {
    __syncthreads();
    if ((tid & 63) == 0) s_sums[tid >> 6] = used;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kPageThreads / 64; ++w) used = max(used, s_sums[w]);
      *a.count_out = count - (int)used;
    }
  }
  if (!kFill) return;
  if (blockIdx.x == 0 && tid == 0) a.cu[0] = 0;
  __syncthreads();
  const int P = 1 << a.lp;
  for (uint32_t i = blockIdx.x * kPageThreads + tid; i < N; i += gridDim.x * kPageThreads) {
    int64_t slot = -1, pos = -1;
    if (i < s_cu[a.B]) {
      int lo = 0, hi = a.B - 1;   // the last request that starts at or before token i
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_cu[mid] <= i) lo = mid; else hi = mid - 1;
      }
      const uint32_t before = s_before[lo];
      if (before != kNone) {
        pos = (int64_t)s_len[lo] + (i - s_cu[lo]);
        const int64_t idx = pos >> a.lp, have = pages_of(s_len[lo], a.lp);
        const int32_t page = idx < have ? a.tables[lo * a.t_sb + idx]
                                        : a.free_pages[count - 1 - (int64_t)before - (idx - have)];
        const int row = (int)(pos & (P - 1));
        if (row == 0) a.tables[lo * a.t_sb + idx] = page;
        slot = page < 0 ? -1 : (((int64_t)page << a.lp) | row);
      }
    }
    a.slots[i] = slot;
    a.positions[i] = pos;
  }
}

struct ReleaseArgs {
  const int32_t* lens;
  const int32_t* keep;
  const int32_t* tables;
  int64_t t_sb;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* lens_out;
  int32_t* count_out;
  int B, T, F, lp;
};

// The pages behind each request's first `keep` rows go back to the free
// list, in request order and table order.  The scan is the extension's; the
// copies are a wave's per request.  Bound by latency like it (kernel 2.3 us for
// 16 requests, 3.2 for 256 that end).
template <bool kFill, bool kCommit>
__global__ __launch_bounds__(kPageThreads) void release_pages_kernel(ReleaseArgs a) {
  extern __shared__ uint32_t sm_words[];
  uint32_t* s_before = sm_words;                   // [B]
  uint32_t* s_first = s_before + a.B;              // [B]: first page given back
  uint32_t* s_n = s_first + a.B;                   // [B]: pages given back
  __shared__ uint32_t s_sums[kPageThreads / 64];
  const int tid = threadIdx.x;
  const bool commit = kCommit && blockIdx.x == 0;
  const int count = min(max(*a.free_count, 0), a.F);
  uint32_t page0 = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPageThreads) {
    const int b = b0 + tid;
    const bool in = b < a.B;
    const int64_t len = in ? a.lens[b] : 0, held = pages_of(len, a.lp);
    const bool bad = len < 0 || held > a.T;
    const int64_t kept = bad ? len : min(len, (int64_t)max(in ? a.keep[b] : 0, 0));
    const int64_t first = pages_of(kept, a.lp);
    const uint32_t n = bad ? 0u : (uint32_t)(held - first);
    uint32_t total;
    const uint32_t upto = page0 + block_incl_scan(n, s_sums, &total);
    page0 += total;
    if (in) {
      s_before[b] = upto - n;
      s_first[b] = (uint32_t)first;
      s_n[b] = n;
      if (commit) a.lens_out[b] = (int32_t)kept;
    }
  }
  if (commit && tid == 0) *a.count_out = (int)min((uint64_t)count + page0, (uint64_t)a.F);
  if (!kFill) return;
  __syncthreads();
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (int b = blockIdx.x * (kPageThreads / 64) + wave; b < a.B; b += gridDim.x * (kPageThreads / 64)) {
    const uint32_t n = s_n[b];
    const int32_t* from = a.tables + b * a.t_sb + s_first[b];
    const int64_t to = (int64_t)count + s_before[b];
    for (uint32_t k = lane; k < n; k += 64)
      if (to + k < a.F) a.free_pages[to + k] = from[k];
  }
}

struct AppendPagedArgs {
  const int64_t* slots;
  const char* k;
  int64_t k_sn, k_sh;  // byte strides
  const char* v;
  int64_t v_sn, v_sh;
  char* kp;
  int64_t kp_sp, kp_sh, kp_ss;
  char* vp;
  int64_t vp_sp, vp_sh, vp_ss;
  int64_t num_slots;
  int64_t pieces;  // 16-byte pieces of K: rows * heads * row pieces
  int heads, row_pieces, lp;
};

// Rows into their slots: a thread moves the same 16-byte piece of K and of V.
// Rows whose slot is outside the pool are skipped.  Bound by bytes: 8192 rows of
// 8 heads x 128 in 2 bytes, 67 MB read and written, in 11.3 us (5.9 TB/s: the
// sources stay in the last-level cache); a step of 16 rows by latency, 2.3.
__global__ __launch_bounds__(256) void append_paged_kernel(AppendPagedArgs a) {
  const int per_row = a.heads * a.row_pieces;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.pieces; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / per_row;
    const int x = (int)(i - n * per_row), h = x / a.row_pieces, c = x - h * a.row_pieces;
    const int64_t slot = a.slots[n];
    const u32x4 kk = ld16(a.k + n * a.k_sn + h * a.k_sh + 16 * c);
    const u32x4 vv = ld16(a.v + n * a.v_sn + h * a.v_sh + 16 * c);
    if (slot < 0 || slot >= a.num_slots) continue;
    const int64_t page = slot >> a.lp, row = slot & (((int64_t)1 << a.lp) - 1);
    st16(a.kp + page * a.kp_sp + h * a.kp_sh + row * a.kp_ss + 16 * c, kk);
    st16(a.vp + page * a.vp_sp + h * a.vp_sh + row * a.vp_ss + 16 * c, vv);
  }
}

// Whether [a, a + n) and [b, b + m) share a word.
static bool meet(const int32_t* a, int64_t n, const int32_t* b, int64_t m) { return a < b + m && b < a + n; }

// log2 of a page size, or -1
int page_shift(int64_t P) {
  if (P < 1 || P > 65536 || (P & (P - 1)) != 0) return -1;
  return __builtin_ctzll((unsigned long long)P);
}

}  // namespace hc

using namespace hc;

extern "C" int hc_extend_pages(int64_t B, const int32_t* lens, const int32_t* new_lens, int32_t* tables, int64_t t_sb,
                               int64_t table_width, const int32_t* free_pages, int64_t free_capacity,
                               const int32_t* free_count, int64_t page_size, int64_t N, int32_t* lens_out,
                               int32_t* count_out, int32_t* cu_new, int64_t* slots, int64_t* positions, void* stream) {
  HC_REQUIRE(B >= 1 && B <= kMaxRequests, "extend_pages: B=%lld outside [1, %d]", (long long)B, kMaxRequests);
  HC_REQUIRE(N >= 0 && N <= kMaxTokens, "extend_pages: num_tokens %lld outside [0, %d]", (long long)N, kMaxTokens);
  const int lp = page_shift(page_size);
  HC_REQUIRE(lp >= 0, "extend_pages: page size %lld must be a power of two up to 65536", (long long)page_size);
  HC_REQUIRE(table_width >= 1 && t_sb >= table_width && table_width <= INT32_MAX / B,
             "extend_pages: tables of %lld x %lld entries, row stride %lld", (long long)B, (long long)table_width,
             (long long)t_sb);
  HC_REQUIRE(table_width <= (INT32_MAX >> lp), "extend_pages: %lld pages of %lld rows pass 2^31 rows a request",
             (long long)table_width, (long long)page_size);
  HC_REQUIRE(free_capacity >= 1 && free_capacity <= INT32_MAX, "extend_pages: free list of %lld entries",
             (long long)free_capacity);
  HC_REQUIRE(lens && new_lens && tables && free_pages && free_count && lens_out && count_out && cu_new &&
                 (N == 0 || (slots && positions)),
             "extend_pages: null pointer");
  const ExtendArgs a{lens, new_lens, tables, t_sb, free_pages, free_count, lens_out, count_out, cu_new, slots, positions,
                     (int)B, (int)table_width, (int)free_capacity, (int)N, lp};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const size_t lds = (3 * (size_t)B + 1) * 4;
  const bool in_place = meet(lens_out, B, lens, B) || meet(lens_out, B, new_lens, B) || meet(lens_out, B, free_count, 1) ||
                        meet(count_out, 1, free_count, 1) || meet(count_out, 1, lens, B) || meet(count_out, 1, new_lens, B);
  // Kernel times for 16 requests: 256 tokens a workgroup 3.2 us at 256 to 4096
  // tokens; one workgroup for all 3.9, 5.0 and 7.8 at 512, 1024 and 2048; a second
  // launch to commit in place 1.8.
  const int64_t wanted = std::min<int64_t>(256, cdiv(std::max<int64_t>(N, 1), (int64_t)kPageThreads));
  const int64_t blocks = in_place && wanted <= 4 ? 1 : wanted;
  if (blocks == 1 || !in_place) {
    extend_pages_kernel<true, true><<<(unsigned)blocks, kPageThreads, lds, s>>>(a);
    return check_launch("extend_pages");
  }
  extend_pages_kernel<true, false><<<(unsigned)blocks, kPageThreads, lds, s>>>(a);
  if (const int rc = check_launch("extend_pages")) return rc;
  extend_pages_kernel<false, true><<<1, kPageThreads, lds, s>>>(a);
  return check_launch("extend_pages");
}

extern "C" int hc_release_pages(int64_t B, const int32_t* lens, const int32_t* keep_lens, const int32_t* tables,
                                int64_t t_sb, int64_t table_width, int32_t* free_pages, int64_t free_capacity,
                                const int32_t* free_count, int64_t page_size, int32_t* lens_out, int32_t* count_out,
                                void* stream) {
  HC_REQUIRE(B >= 1 && B <= kMaxRequests, "release_pages: B=%lld outside [1, %d]", (long long)B, kMaxRequests);
  const int lp = page_shift(page_size);
  HC_REQUIRE(lp >= 0, "release_pages: page size %lld must be a power of two up to 65536", (long long)page_size);
  HC_REQUIRE(table_width >= 1 && t_sb >= table_width && table_width <= INT32_MAX / B,
             "release_pages: tables of %lld x %lld entries, row stride %lld", (long long)B, (long long)table_width,
             (long long)t_sb);
  HC_REQUIRE(table_width <= (INT32_MAX >> lp), "release_pages: %lld pages of %lld rows pass 2^31 rows a request",
             (long long)table_width, (long long)page_size);
  HC_REQUIRE(free_capacity >= 1 && free_capacity <= INT32_MAX, "release_pages: free list of %lld entries",
             (long long)free_capacity);
  HC_REQUIRE(lens && keep_lens && tables && free_pages && free_count && lens_out && count_out,
             "release_pages: null pointer");
  const ReleaseArgs a{lens, keep_lens, tables, t_sb, free_pages, free_count, lens_out, count_out,
                      (int)B, (int)table_width, (int)free_capacity, lp};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const size_t lds = 3 * (size_t)B * 4;
  const bool in_place = meet(lens_out, B, lens, B) || meet(lens_out, B, keep_lens, B) || meet(lens_out, B, free_count, 1) ||
                        meet(count_out, 1, free_count, 1) || meet(count_out, 1, lens, B) || meet(count_out, 1, keep_lens, B);
  // Kernel times: four requests a workgroup 2.5 us up to 256; one workgroup for
  // all 2.6, 3.1 and 4.2 at 8, 16 and 32 that end; a second launch to commit in
  // place 1.7.
  const int64_t wanted = std::min<int64_t>(256, cdiv(B, (int64_t)(kPageThreads / 64)));
  const int64_t blocks = in_place && B <= 32 ? 1 : wanted;
  if (blocks == 1 || !in_place) {
    release_pages_kernel<true, true><<<(unsigned)blocks, kPageThreads, lds, s>>>(a);
    return check_launch("release_pages");
  }
  release_pages_kernel<true, false><<<(unsigned)blocks, kPageThreads, lds, s>>>(a);
  if (const int rc = check_launch("release_pages")) return rc;
  release_pages_kernel<false, true><<<1, kPageThreads, lds, s>>>(a);
  return check_launch("release_pages");
}

extern "C" int hc_append_paged(int dtype, int64_t N, int64_t Hk, int64_t D, const int64_t* slots,
                               const void* k_new, int64_t kn_sn, int64_t kn_sh,
                               const void* v_new, int64_t vn_sn, int64_t vn_sh,
                               void* k_pages, int64_t kp_sp, int64_t kp_sh, int64_t kp_ss,
                               void* v_pages, int64_t vp_sp, int64_t vp_sh, int64_t vp_ss,
                               int64_t num_pages, int64_t page_size, void* stream) {
  HC_REQUIRE(dtype == HC_DTYPE_F32 || dtype == HC_DTYPE_F16 || dtype == HC_DTYPE_BF16, "append_paged: bad dtype %d", dtype);
  HC_REQUIRE(N >= 0 && N <= INT32_MAX && Hk >= 1 && Hk <= 65535 && D >= 1 && D <= 65536,
             "append_paged: bad shape N=%lld Hk=%lld D=%lld", (long long)N, (long long)Hk, (long long)D);
  const int lp = page_shift(page_size);
  HC_REQUIRE(lp >= 0, "append_paged: page size %lld must be a power of two up to 65536", (long long)page_size);
  HC_REQUIRE(num_pages >= 1 && num_pages <= INT32_MAX, "append_paged: %lld pages", (long long)num_pages);
  const int64_t es = dtype_size(dtype);
  HC_REQUIRE((D * es) % 16 == 0, "append_paged: rows of %lld bytes must be a multiple of 16", (long long)(D * es));
  if (N == 0) return HC_OK;
  HC_REQUIRE(slots && k_new && v_new && k_pages && v_pages, "append_paged: null pointer");
  HC_REQUIRE((uintptr_t)k_new % 16 == 0 && (uintptr_t)v_new % 16 == 0 && (uintptr_t)k_pages % 16 == 0 &&
                 (uintptr_t)v_pages % 16 == 0,
             "append_paged: rows must be 16-byte aligned");
  const int64_t st[] = {kn_sn, kn_sh, vn_sn, vn_sh, kp_sp, kp_sh, kp_ss, vp_sp, vp_sh, vp_ss};
  for (const int64_t x : st)
    HC_REQUIRE((x * es) % 16 == 0, "append_paged: strides must be multiples of 16 bytes (got %lld elements)", (long long)x);
  AppendPagedArgs a{};
  a.slots = slots;
  a.k = (const char*)k_new; a.k_sn = kn_sn * es; a.k_sh = kn_sh * es;
  a.v = (const char*)v_new; a.v_sn = vn_sn * es; a.v_sh = vn_sh * es;
  a.kp = (char*)k_pages; a.kp_sp = kp_sp * es; a.kp_sh = kp_sh * es; a.kp_ss = kp_ss * es;
  a.vp = (char*)v_pages; a.vp_sp = vp_sp * es; a.vp_sh = vp_sh * es; a.vp_ss = vp_ss * es;
  a.num_slots = num_pages << lp;
  a.heads = (int)Hk; a.row_pieces = (int)(D * es / 16); a.lp = lp;
  a.pieces = N * Hk * a.row_pieces;
  const int64_t blocks = std::min<int64_t>(4096, cdiv(a.pieces, (int64_t)256));
  append_paged_kernel<<<(unsigned)blocks, 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(a);
  return check_launch("append_paged");
}
