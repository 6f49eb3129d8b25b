// Device side of the attention behind a shared prompt (hc_prefix.hip holds the
// host side and the C ABI; the kernels are instantiated once per element type
// in hc_prefix_{f16,bf16,f32}.hip, so the three compile in parallel).
//
// Query token i of request b (n tokens, len own rows) attends the prompt's
// rows [0, prefix_lens[b]) and its own rows [0, len - n + i].  With G query
// heads per KV head, the batch is N * G query rows per KV head.
//
// One launch has two kinds of items, each one workgroup:
//   * prompt items: (KV head, tile of query rows packed over all requests, key
//     range of the prompt): the prompt is read once per tile, for all requests;
//   * own items: (request, KV head, tile of its query rows, key range of its
//     pages).
// Each writes (max, sum, unnormalised output) of its rows for its keys, and a
// second launch joins them.  Where the prompt is short, or absent, the own items
// take it too and write their rows complete: one launch.
//
// A workgroup's NW waves are WR x WK: WR waves share the keys and take 32
// query rows each (16, where a tile has no more), WK waves take different keys.
// WR follows the rows there are (16 to 32 NW a tile): a single request's few
// rows put every wave on keys of its own.
//   * Scores are K.Q^T (v_mfma_f32_32x32x16, fp32 inputs 32x32x2; 16x16x32 and
//     16x16x4 for tiles of 16 rows): a lane holds one query row's scores of 16
//     keys, so the row's running max and sum live in its two (four) lanes, and
//     its probabilities are, as they stand, the B operand of V^T.P^T: the
//     product's order of keys is the score layout's (index, below), and V^T's
//     operand is read in that order, by LDS transpose reads (ds_read_b64_tr)
//     for 2-byte types.  The output is transposed, too: a lane owns its
//     query's column, and the rescale is a multiply by the lane's own factor.
//   * K and V tiles go to LDS by asynchronous loads (global_load_lds_dwordx4)
//     with a 16-byte piece p of row r stored at p ^ f(r): f spreads 16 rows'
//     same piece over all banks (K's operand reads) and 4 rows' piece pairs
//     over distinct ones (V's transpose reads).
//   * Softmax is online, in fp32 and the log2 domain, with a lazy reference
//     (kLazy): the accumulators are rescaled only where a row's max passes its
//     reference by 2^8.  Probabilities are rounded once to the inputs' 2-byte
//     type (fp32: not at all); their sum takes them unrounded.
//   * Tiles that every row of the wave sees whole take no masks.  Others
//     select per key; rows no request holds, or in pages outside the pool, are
//     zeroed in LDS first, so that nothing stale enters a product.  Where rows
//     of one tile see different keys and a value is not finite, the tile's
//     product is taken key by key (0 times infinity must not reach a row that
//     does not attend it).
#pragma once
#include "hc_common.h"

namespace hc {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

struct PrefixArgs {
  const char* q;   // strides in bytes
  int64_t q_sn, q_sh;
  const char* kp;
  int64_t kp_sh, kp_ss;
  const char* vp;
  int64_t vp_sh, vp_ss;
  const char* kg;
  int64_t kg_sp, kg_sh, kg_ss;
  const char* vg;
  int64_t vg_sp, vg_sh, vg_ss;
  const int32_t* prefix_lens;
  const int32_t* tables;
  int64_t t_sb;
  const int32_t* lens;
  const int32_t* cu;
  char* out;
  int64_t o_sn, o_sh;
  float* lse;
  int64_t l_sn, l_sh;
  float* part_o;   // [slots][N * Hq][D]
  float* part_ml;  // [slots][N * Hq][2]
  // |scaling| log2(e), its sign and zero moved to q: (q & q_and) ^ q_xor.  (A
  // scale of 0 would turn masked scores, -inf, into NaN.)
  float scale_log2;
  uint32_t q_and, q_xor;
  int N, B, Hq, Hk, G, D, S, T, lp, num_pages, max_new;
  // prompt items: query rows of a tile, tiles, key splits and keys a split; own
  // items: rows of a tile, tiles and splits of one request
  int p_rows, p_tiles, p_splits, p_chunk, p_items;
  int o_rows, o_tiles, o_splits;
  int both;   // own items take the prompt too: no prompt items, no partials
  // merge: tiles of rows of one request, groups of threads a row
  int m_tiles, m_sub;
};

constexpr float kLazy = 8.f;
constexpr int kMergeSub = 8;    // groups of threads a row, where few rows have many partials
constexpr int kPageIds = 2048;  // page numbers held in LDS at a time

// NW waves a workgroup, one workgroup a CU (256 registers a lane, most of LDS):
// 8, or 4 where rows are 512 bytes, as K and V of 32 keys a wave have to fit
// LDS.  (Workgroups of 4 waves, two a CU, took longer at every split: 16
// requests behind 32k prompt rows 51 us against 68, 64 behind 64k 139 / 180.)
template <typename T, int D>
struct PrefixShape {
  static constexpr int kRowB = D * (int)sizeof(T);
  static constexpr int NW = kRowB >= 512 ? 4 : 8;
  static constexpr int kPieces = kRowB / 16;
  static constexpr int kTileB = NW * 32 * 2 * kRowB;   // WR = 1: one buffer; more: two of BN keys
  static constexpr int kOutB = NW * 32 * (D + 4) * 4;  // the outputs of all waves
  static constexpr int kLds = kTileB > kOutB ? kTileB : kOutB;
};

// Rows of own keys per split of a request with len rows.
__host__ __device__ __forceinline__ int own_chunk(int len, int splits) {
  const int c = (len + splits - 1) / splits;
  return max((c + 255) / 256 * 256, 256);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// max / sum over a column's lanes (lane % RW)
template <int RW>
__device__ __forceinline__ float col_max(float x) {
  if constexpr (RW == 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
template <int RW>
__device__ __forceinline__ float col_sum(float x) {
  if constexpr (RW == 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// 16 bytes per lane from p (the lane's own) to LDS at byte offset lds (the
// wave's) + 16 * lane, asynchronously: complete after vm_wait.  The compiler
// does not see the write; every use is behind a vm_wait, which it does not
// move memory accesses across.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ void load_to_lds(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(uniform(lds)), "v"(p)
               : "memory");
}
// ... from the wave's address base plus the lane's offset.  (The base may come
// from a v_readfirstlane, which takes five wait states before a memory
// instruction may read it; the compiler's own count does not look into asm.)
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t off, uint32_t lds) {
  const uint64_t s = (uint64_t)uniform((uint32_t)((uint64_t)base >> 32)) << 32 | uniform((uint32_t)(uint64_t)base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(uniform(lds)), "v"(off), "s"(s)
               : "memory");
}
__device__ __forceinline__ void lds_wait() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <int N>
__device__ __forceinline__ void vm_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The lane's value again, as one the compiler does not know: what is computed
// from it in a rare path stays there, instead of in registers of the whole loop.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// One product of RW x RW outputs: A's RW rows are keys (or dimensions of V), B's
// RW columns query rows.  A lane holds column lane % RW; lanes / RW are its
// groups.  Register i of an output is row index(i, group) of its block.
template <typename T, int RW>
struct Mma;
template <>
struct Mma<half_t, 32> {
  typedef half8 frag;
  typedef floatx16 out;
  __device__ static out mma(frag a, frag b, out c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<half_t, 16> {
  typedef half8 frag;
  typedef floatx4 out;
  __device__ static out mma(frag a, frag b, out c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<bf16_t, 32> {
  typedef bf16x8 frag;
  typedef floatx16 out;
  __device__ static out mma(frag a, frag b, out c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<bf16_t, 16> {
  typedef bf16x8 frag;
  typedef floatx4 out;
  __device__ static out mma(frag a, frag b, out c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
// (fp32: a fragment's four elements are four products of one element each)
template <>
struct Mma<float, 32> {
  typedef floatx4 frag;
  typedef floatx16 out;
  __device__ static out one(float a, float b, out c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
  __device__ static out mma(frag a, frag b, out c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = one(a[j], b[j], c);
    return c;
  }
};
template <>
struct Mma<float, 16> {
  typedef floatx4 frag;
  typedef floatx4 out;
  __device__ static out one(float a, float b, out c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
  __device__ static out mma(frag a, frag b, out c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = one(a[j], b[j], c);
    return c;
  }
};

// What an item's workgroup works on: the prompt's keys, a request's own, or
// both, one after the other (then the rows are complete and go out as they are).
enum { kPromptItem, kOwnItem, kBothItem };
struct Item {
  int hk, tok0, row0, rows;   // query rows [row0, rows) of tokens tok0 + row / G
  int pbeg, pend;             // the prompt's keys
  int obeg, oend;             // own keys; row r sees those below lim0 + r / G (at least 0)
  int lim0;
  const int32_t* table;       // the request's pages
  int slot;                   // where the partial goes
};

// Four dimensions of a complete row, and its log-sum-exp.
template <typename T>
__device__ __forceinline__ void finish_row(const PrefixArgs& a, int t, int h, int dim, floatx4 x, float M, float L) {
  typedef T outx4 __attribute__((ext_vector_type(4)));
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<outx4*>(reinterpret_cast<T*>(a.out + t * a.o_sn + h * a.o_sh) + dim) =
      outx4{from_f32<T>(x[0] * inv), from_f32<T>(x[1] * inv), from_f32<T>(x[2] * inv), from_f32<T>(x[3] * inv)};
  if (a.lse && dim == 0)
    a.lse[t * a.l_sn + h * a.l_sh] = L == 0.f ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
}

// A workgroup's part: RW query rows a wave (16 where no more are there: half the
// work and registers of 32), WR waves sharing the keys.
template <typename T, int D, int RW, int WR, int kMode>
__device__ __forceinline__ void prefix_item(const PrefixArgs& a, const Item& it, char* smem, int32_t* s_pid, float* s_ml) {
  using Sh = PrefixShape<T, D>;
  typedef Mma<T, RW> M_;
  typedef typename M_::frag frag;
  typedef typename M_::out out_t;
  constexpr int NW = Sh::NW;
  constexpr int kRowB = Sh::kRowB, kPieces = Sh::kPieces, WK = NW / WR;
  constexpr int KT = WK <= NW / 4 ? 64 : 32;   // keys a wave takes of a tile
  constexpr int KB = KT / RW, BN = WK * KT;
  constexpr int kStages = WR == 1 ? 1 : 2;
  constexpr int kRows = KT / WR;               // rows of a tile a wave loads
  constexpr int kPerLoad = 64 / kPieces;       // rows of one load
  constexpr int kLoads = (kRows + kPerLoad - 1) / kPerLoad;
  constexpr bool kPartial = kRows < kPerLoad;  // a load's last lanes stay idle
  constexpr int kSt = BN * kRowB;              // bytes of a tile's K, or V
  static_assert(2 * kSt * kStages <= Sh::kLds, "tiles fit LDS");
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kGroups = 64 / RW, kAcc = RW * RW / 64;
  constexpr int NB = (D + RW - 1) / RW;        // blocks of RW output dimensions
  constexpr int NQ = (kPieces + kGroups - 1) / kGroups;   // a piece a group and product
  constexpr int kPk = 8 * kGroups;             // keys of an output product (2-byte types)

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wr = wave % WR, wk = wave / WR;
  const int col = lane % RW, grp = lane / RW;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  auto index = [](int i, int g) { return RW == 32 ? (i & 3) + 8 * (i >> 2) + 4 * g : i + 4 * g; };

  // ---- the wave's query rows (used, and so waited for, behind the first keys' loads)
  const int r = it.row0 + RW * wr + col;
  const bool live = r < it.rows;
  // a wave of no rows only loads (72 requests' 288 rows in two tiles of 256, behind
  // 32k: 99 -> 91 us)
  const bool works = it.row0 + RW * wr < it.rows;
  const int tok = it.tok0 + (live ? r / a.G : 0);
  const int head = it.hk * a.G + (live ? r % a.G : 0);
  u32x4 qw[NQ];
  {
    const char* qp = a.q + tok * a.q_sn + head * a.q_sh;
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      qw[t] = u32x4{0u, 0u, 0u, 0u};
      if (live && (kPieces % kGroups == 0 || kGroups * t + grp < kPieces)) qw[t] = ld16(qp + 16 * (kGroups * t + grp));
    }
  }
  out_t acc[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d)
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[d][i] = 0.f;
  float m = -INFINITY, l = 0.f;

  // f(r) of row r: pieces of 16 rows with the same number lie on distinct
  // 16-byte columns of the 256 bytes all banks hold, pairs of 4 rows too
  constexpr int kXor = kPieces < 16 ? kPieces : 16;
  constexpr int kXorBits = kXor == 16 ? 4 : kXor == 8 ? 3 : kXor == 4 ? 2 : 1;
  constexpr int kRows256 = 16 / kXor;
  auto swz = [](int row) {
    const int x = (row / kRows256) & (kXor - 1);
    return ((x << 1) | (x >> (kXorBits - 1))) & (kXor - 1);
  };

  // The keys [kbeg, kend) of the prompt or of the request's pages: the lane's
  // row sees those below lim, every row of the workgroup those below all.
  auto sweep = [&](auto own_keys, const int kbeg, const int kend, const int all, const int lim) {
    constexpr bool kOwn = decltype(own_keys)::value;
    // rows see different keys: a value that is not finite may have to reach some
    // of them only
    const bool ragged = all != kend;
    const char* kbase = kOwn ? a.kg + it.hk * a.kg_sh : a.kp + it.hk * a.kp_sh;
    const char* vbase = kOwn ? a.vg + it.hk * a.vg_sh : a.vp + it.hk * a.vp_sh;
    // (a segment's first page may be entered in its middle)
    const int seg_keys = kOwn ? ((kPageIds - 1) << min(a.lp, 12)) / BN * BN : 0x7fffffff;
    for (int seg = kbeg, send; seg < kend; seg = send) {
      send = kend - seg > seg_keys ? seg + seg_keys : kend;
      bool bad_pages = false;
      const int page0 = seg >> a.lp;
      if constexpr (kOwn) {
        if (seg != kbeg) __syncthreads();   // the last segment's pages are read
        int bad = 0;
        const int n = ((send - 1) >> a.lp) - page0 + 1;
        for (int i = threadIdx.x; i < n; i += NW * 64) {
          const int p = it.table[page0 + i];
          const bool ok = (uint32_t)p < (uint32_t)a.num_pages;
          s_pid[i] = ok ? p : -1;
          bad |= !ok;
        }
        int* s_bad = reinterpret_cast<int*>(s_ml);
        bad = __any(bad);
        if (lane == 0) s_bad[wave] = bad;
        __syncthreads();   // (also: the tiles of the keys before are read)
        int any = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) any |= s_bad[w];
        bad_pages = __builtin_amdgcn_readfirstlane(any) != 0;
      }

      // asynchronous loads of the wave's rows of the tile at key0: consecutive
      // keys, one address and the lanes' offsets where they are in one page
      auto issue = [&](int key0, int stage, bool v) {
        const int piece = lane % kPieces, sub = lane / kPieces;
        const uint32_t dst = lds0 + (uint32_t)((stage * 2 + (v ? 1 : 0)) * kSt + (wk * KT + wr * kRows) * kRowB);
        const int64_t ss = kOwn ? (v ? a.vg_ss : a.kg_ss) : (v ? a.vp_ss : a.kp_ss);
        const char* base = v ? vbase : kbase;
        const int first = key0 + wk * KT + wr * kRows;
        // (f of a sum of rows with distinct bits is the xor of theirs)
        const uint32_t at = 16 * (piece ^ swz(wr * kRows + sub));
        if (first + kRows <= send && (!kOwn || (1 << a.lp) >= kRows)) {
          if constexpr (kOwn) {
            const int pid = __builtin_amdgcn_readfirstlane(s_pid[(first >> a.lp) - page0]);
            base += (int64_t)max(pid, 0) * (v ? a.vg_sp : a.kg_sp) + (int64_t)(first & ((1 << a.lp) - 1)) * ss;
          } else {
            base += (int64_t)first * ss;
          }
          const uint32_t rows = (uint32_t)sub * (uint32_t)ss;
          if (!kPartial || lane < kRows * kPieces) {
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
              load_to_lds(base + j * kPerLoad * ss, (at ^ (16 * swz(j * kPerLoad))) + rows, dst + j * 1024);
          }
        } else {
#pragma unroll 1
          for (int j = 0; j < kLoads; ++j) {
            // keys past the end load the last one's row (zeroed below)
            const int key = min(first + j * kPerLoad + sub, send - 1);
            const char* p = base;
            if constexpr (kOwn) {
              const int pid = max(s_pid[(key >> a.lp) - page0], 0);
              p += (int64_t)pid * (v ? a.vg_sp : a.kg_sp) + (int64_t)(key & ((1 << a.lp) - 1)) * ss;
            } else {
              p += (int64_t)key * ss;
            }
            if (!kPartial || lane < kRows * kPieces) load_to_lds(p + (at ^ (16 * swz(j * kPerLoad))), dst + j * 1024);
          }
        }
      };
      auto hidden = [&](int key) {   // a key of the segment's tiles that nobody attends
        if (key >= send) return true;
        if constexpr (kOwn) return bad_pages && s_pid[(key >> a.lp) - page0] < 0;
        return false;
      };
      // zero the wave's loaded rows of keys nobody attends
      auto clear = [&](int key0, int stage, bool v) {
        const int ln = fresh(lane);
#pragma unroll 1
        for (int j = 0; j < kLoads; ++j) {
          const int row = wr * kRows + j * kPerLoad + ln / kPieces;
          if ((!kPartial || ln < kRows * kPieces) && hidden(key0 + wk * KT + row))
            st16(smem + (stage * 2 + (v ? 1 : 0)) * kSt + (wk * KT + row) * kRowB + (ln % kPieces) * 16,
                 u32x4{0u, 0u, 0u, 0u});
        }
      };
      // the order of a phase's LDS reads and products: operands a few products ahead
      auto order = [](auto products, auto reads, auto ahead, auto id) {
        constexpr int kN = decltype(products)::value, kR = decltype(reads)::value, kId = decltype(id)::value;
        constexpr int kA = kN < decltype(ahead)::value ? kN : decltype(ahead)::value;
        __builtin_amdgcn_sched_group_barrier(0x100, kR * kA, kId);
        static_for<kN - kA>([](auto) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, kId);
          __builtin_amdgcn_sched_group_barrier(0x100, kR, kId);
        });
        __builtin_amdgcn_sched_group_barrier(0x8, kA, kId);
      };
      using std::integral_constant;

      int tile = seg;
      const int whole = bad_pages ? seg : min(all, send);
      // one tile; kAll: every row sees all of its keys
      auto do_tile = [&](int n, auto all_see) {
        constexpr bool kAll = decltype(all_see)::value;
        const int stage = kStages == 1 ? 0 : (n & 1);
        const bool more = tile + BN < send;
        const bool edge = !kAll && (tile + BN > send || bad_pages);
        if constexpr (WR == 1) {
          // the wave's own rows: its V loads (kLoads of them) may be in flight
          vm_wait<kLoads>();
          if (edge) clear(tile, 0, false);
        } else {
          vm_wait<0>();
          if (edge) {
            clear(tile, stage, false);
            clear(tile, stage, true);
          }
          __syncthreads();
          if (more) {
            issue(tile + BN, stage ^ 1, false);
            issue(tile + BN, stage ^ 1, true);
          }
          if (!works) return;
        }
        const char* ks = smem + stage * 2 * kSt + wk * KT * kRowB;
        const char* vs = ks + kSt;
        const int key0 = tile + wk * KT;

        // ---- scores
        out_t s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < kAcc; ++i) s[kb][i] = 0.f;
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            const int row = RW * kb + col;
            u32x4 x = ld16(ks + row * kRowB + ((((kGroups * t + grp) % kPieces) ^ swz(row)) << 4));
            if constexpr (kPieces % kGroups != 0)
              if (kGroups * t + grp >= kPieces) x = u32x4{0u, 0u, 0u, 0u};
            s[kb] = M_::mma(__builtin_bit_cast(frag, x), __builtin_bit_cast(frag, qw[t]), s[kb]);
          }
        if constexpr (kAll && !kF32)
          order(integral_constant<int, NQ * KB>{}, integral_constant<int, 1>{}, integral_constant<int, 6>{},
                integral_constant<int, 0>{});
        if constexpr (WR == 1) {
          if (more) {
            lds_wait();   // the tile's reads are done
            issue(tile + BN, 0, false);
          }
        }
        __builtin_amdgcn_sched_barrier(0);

        // ---- softmax
        if constexpr (!kAll) {
          const int first = key0 + 4 * fresh(grp);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < kAcc; ++i) {
              const int key = first + RW * kb + index(i, 0);
              bool see = key < lim;
              if (bad_pages) see = see && !hidden(key);
              s[kb][i] = see ? s[kb][i] : -INFINITY;
            }
        }
        float t = s[0][0], u = s[0][1];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < kAcc; i += 4) {
            t = fmaxf(fmaxf(t, s[kb][i]), s[kb][i + 1]);
            u = fmaxf(fmaxf(u, s[kb][i + 2]), s[kb][i + 3]);
          }
        t = col_max<RW>(fmaxf(t, u)) * a.scale_log2;
        const bool bump = t > m + kLazy;
        if (__any(bump)) {
          const float mn = bump ? t : m;
          const float alpha = bump ? exp2_hw(m - mn) : 1.f;
          m = mn;
          l *= alpha;
#pragma unroll
          for (int d = 0; d < NB; ++d)
#pragma unroll
            for (int i = 0; i < kAcc; ++i) acc[d][i] *= alpha;
        }
        const float ref = m == -INFINITY ? 0.f : m;   // (a row that has seen nothing yet: its terms are 0)
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < kAcc; ++i) {
            s[kb][i] = exp2_hw(__builtin_fmaf(s[kb][i], a.scale_log2, -ref));
            sum[i & 3] += s[kb][i];
          }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if constexpr (WR == 1) {
          if (more) vm_wait<kLoads>(); else vm_wait<0>();
          if (edge) clear(tile, 0, true);
        }
        __builtin_amdgcn_sched_barrier(0);

        // ---- output
        bool slow = false;
        if (!kAll && ragged) {
          // a value that is not finite in this tile?
          uint32_t odd = 0;
          for (int i = fresh(lane); i < KT * kPieces; i += 64) {
            const u32x4 x = ld16(vs + 16 * i);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if constexpr (kF32) {
                odd |= (x[w] & 0x7f800000u) == 0x7f800000u;
              } else {
                constexpr uint32_t kExp = std::is_same<T, half_t>::value ? 0x7c00u : 0x7f80u;
                odd |= (x[w] & kExp) == kExp;
                odd |= ((x[w] >> 16) & kExp) == kExp;
              }
            }
          }
          slow = __any(odd);
        }
        // (with slow the product is taken of zeros, and the keys one at a time below)
        const uint32_t mask = !kAll && slow ? 0u : ~0u;
        if constexpr (kF32) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < kAcc; ++i) {
              const int row = RW * kb + index(i, grp);
#pragma unroll
              for (int d = 0; d < NB; ++d) {
                const int dim = min(RW * d + col, D - 1);   // (outputs past D are not used)
                uint32_t v =
                    *reinterpret_cast<const uint32_t*>(vs + row * kRowB + (((dim >> 2) ^ swz(row)) << 4) + (dim & 3) * 4);
                uint32_t p = __float_as_uint(s[kb][i]);
                if constexpr (!kAll) {
                  v &= mask;
                  p &= mask;
                }
                acc[d] = M_::one(__uint_as_float(v), __uint_as_float(p), acc[d]);
              }
            }
        } else {
          typedef __attribute__((address_space(3))) shortx4 lds4;
          constexpr int kFar = RW == 32 ? 8 : 16;   // the second four of a lane's keys
#pragma unroll
          for (int h = 0; h < KT / kPk; ++h) {
            // probabilities as they stand: element j is key kPk h + 4 grp + (j & 3) + kFar (j / 4)
            frag p;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              p[j] = from_f32<T>(RW == 32 ? s[h / 2][(8 * (h & 1) + j) % kAcc] : s[(2 * h + j / 4) % KB][j % 4]);
            if constexpr (!kAll) p = __builtin_bit_cast(frag, __builtin_bit_cast(u32x4, p) & mask);
            const int row = kPk * h + 4 * grp + ((lane & 15) >> 2);
#pragma unroll
            for (int d = 0; d < NB; ++d) {
              // dimensions past D (16) read the row's first ones; their output is not used
              const int dim = (D % RW == 0 ? RW * d + (RW == 32 ? 16 * ((lane >> 4) & 1) : 0) : 0) + 4 * (lane & 3);
              union {
                shortx4 h[2];
                u32x4 w;
              } v;
              v.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (lds4*)(vs + row * kRowB + (((dim >> 3) ^ swz(row)) << 4) + (dim & 4) * 2));
              v.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (lds4*)(vs + (row + kFar) * kRowB + (((dim >> 3) ^ swz(row + kFar)) << 4) + (dim & 4) * 2));
              if constexpr (!kAll) v.w &= mask;
              acc[d] = M_::mma(__builtin_bit_cast(frag, v.w), p, acc[d]);
            }
          }
          if constexpr (kAll)
            order(integral_constant<int, KT / kPk * NB>{}, integral_constant<int, 2>{}, integral_constant<int, 4>{},
                  integral_constant<int, 1>{});
        }
        if (!kAll && slow) {
          // one key at a time, into the rows that see it
#pragma unroll 1
          for (int only = 0; only < KT; ++only) {
            const int grp_ = fresh(grp);
            float p = 0.f;   // in the lane of the column that holds the key
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int i = 0; i < kAcc; ++i) p = RW * kb + index(i, 0) == only - 4 * grp_ ? s[kb][i] : p;
            p = to_f32(from_f32<T>(col_sum<RW>(p)));
            const bool take = key0 + only < lim && !hidden(key0 + only);
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
              for (int i = 0; i < kAcc; ++i) {
                const int at = min(RW * d + index(i, 0) + 4 * grp_, D - 1) * (int)sizeof(T);
                const T v = *reinterpret_cast<const T*>(vs + only * kRowB + (((at >> 4) ^ swz(only)) << 4) + (at & 15));
                acc[d][i] = take ? __builtin_fmaf(p, to_f32(v), acc[d][i]) : acc[d][i];
              }
          }
        }
        if constexpr (WR == 1) {
          if (more) {
            lds_wait();
            issue(tile + BN, 0, true);
          }
        }
      };
      int n = 0;
      issue(tile, 0, false);
      issue(tile, 0, true);
      // (the query rows are waited for here, once: in the loop the compiler's wait
      // would be for every load in flight)
#pragma unroll
      for (int t = 0; t < NQ; ++t) asm volatile("" : "+v"(qw[t]));
#pragma unroll 1
      for (; tile + BN <= whole; tile += BN, ++n) do_tile(n, std::true_type{});
#pragma unroll 1
      for (; tile < send; tile += BN, ++n) do_tile(n, std::false_type{});
    }
  };

  if ((a.q_xor | ~a.q_and) != 0) {   // a scaling below or of zero
#pragma unroll
    for (int t = 0; t < NQ; ++t) qw[t] = (qw[t] & a.q_and) ^ a.q_xor;
  }
  if constexpr (kMode == kPromptItem) {
    int lim = it.pend, all = it.pend, kend = it.pend;
    if (a.prefix_lens) {
      if (live) {
        int b = tok;
        if (a.cu) {   // the last request that starts at or before the token
          int lo = 0, hi = a.B - 1;
          while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.cu[mid] <= tok) lo = mid; else hi = mid - 1;
          }
          b = lo;
        }
        lim = min(lim, max(0, a.prefix_lens[b]));
      }
      // keys every row of the workgroup sees, and keys some row sees
      int lo = lim, hi = live ? lim : 0;
#pragma unroll
      for (int o = RW / 2; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o, 64));
        hi = max(hi, __shfl_xor(hi, o, 64));
      }
      int* s_lim = reinterpret_cast<int*>(s_ml);
      if (lane == 0) {
        s_lim[wave] = lo;
        s_lim[NW + wave] = hi;
      }
      __syncthreads();
      kend = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        all = min(all, s_lim[w]);
        kend = max(kend, s_lim[NW + w]);
      }
      all = __builtin_amdgcn_readfirstlane(all);
      kend = __builtin_amdgcn_readfirstlane(kend);
    }
    sweep(std::false_type{}, it.pbeg, kend, all, lim);
  }
  if constexpr (kMode == kBothItem) sweep(std::false_type{}, it.pbeg, it.pend, it.pend, it.pend);
  if constexpr (kMode != kPromptItem) {
    // (the first row sees least; oend is the last one's)
    const int all = min(it.oend, max(0, it.lim0 + it.row0 / a.G));
    sweep(std::true_type{}, it.obeg, it.oend, all, live ? min(it.oend, max(0, it.lim0 + r / a.G)) : it.oend);
  }

  // ---- the waves of the same rows join: through LDS, each row's sums weighted
  // by its waves' maxima
  l = col_sum<RW>(l);
  constexpr int kOs = D + 4;
  float* so = reinterpret_cast<float*>(smem);
  __syncthreads();   // no tile is read any more
  if (live) {
    if (grp == 0) {
      s_ml[(wave * RW + col) * 2] = m;
      s_ml[(wave * RW + col) * 2 + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
      for (int i = 0; i < kAcc; i += 4) {
        const int dim = RW * d + index(i, grp);
        if (D % RW == 0 || dim < D)
          *reinterpret_cast<floatx4*>(so + (wave * RW + col) * kOs + dim) =
              floatx4{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
      }
  }
  __syncthreads();
  const int64_t rows_all = (int64_t)a.N * a.Hq;
  constexpr int kVec = D / 4;                    // 16-byte pieces of a row
  const int first = it.row0 + RW * wr, join = min(RW, it.rows - first);   // the waves' live rows
  for (int i = wk * 64 + lane; i < join * kVec; i += 64 * WK) {
    const int c = i / kVec, dim = (i % kVec) * 4;
    float M = -INFINITY, L = 0.f;
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < WK; ++k) M = fmaxf(M, s_ml[((k * WR + wr) * RW + c) * 2]);
#pragma unroll
    for (int k = 0; k < WK; ++k) {
      const int w = (k * WR + wr) * RW + c;
      const float mk = s_ml[w * 2], scale = mk == -INFINITY ? 1.f : exp2_hw(mk - M);   // (no max: 0, or NaN)
      L += s_ml[w * 2 + 1] * scale;
      x += *reinterpret_cast<const floatx4*>(so + w * kOs + dim) * scale;
    }
    const int row = first + c, t = it.tok0 + row / a.G, h = it.hk * a.G + row % a.G;
    if constexpr (kMode == kBothItem) {
      finish_row<T>(a, t, h, dim, x, M, L);
    } else {
      const int64_t at = it.slot * rows_all + (int64_t)t * a.Hq + h;
      *reinterpret_cast<floatx4*>(a.part_o + at * D + dim) = x;
      if (dim == 0) {
        a.part_ml[at * 2] = M;
        a.part_ml[at * 2 + 1] = L;
      }
    }
  }
}

// The items of one kind, by the rows of their tiles.
template <typename T, int D, int kMode>
__device__ __forceinline__ void prefix_items(int rows, const PrefixArgs& a, const Item& it, char* smem, int32_t* s_pid,
                                             float* s_ml) {
  switch (rows) {
    case 16: prefix_item<T, D, 16, 1, kMode>(a, it, smem, s_pid, s_ml); break;
    case 32: prefix_item<T, D, 32, 1, kMode>(a, it, smem, s_pid, s_ml); break;
    case 64: prefix_item<T, D, 32, 2, kMode>(a, it, smem, s_pid, s_ml); break;
    case 128: prefix_item<T, D, 32, 4, kMode>(a, it, smem, s_pid, s_ml); break;
    default:
      if constexpr (PrefixShape<T, D>::NW >= 8) prefix_item<T, D, 32, 8, kMode>(a, it, smem, s_pid, s_ml);
      break;
  }
}

template <typename T, int D>
__global__ __launch_bounds__((PrefixShape<T, D>::NW * 64)) __attribute__((amdgpu_waves_per_eu(1, 2))) void
prefix_attn_kernel(PrefixArgs a) {
  using Sh = PrefixShape<T, D>;
  constexpr int NW = Sh::NW;
  __shared__ __attribute__((aligned(16))) char smem[Sh::kLds];
  __shared__ int32_t s_pid[kPageIds];
  __shared__ float s_ml[NW * 64];
  Item it{};
  const int tokens = a.cu ? min(max(a.cu[a.B], 0), a.N) : a.N;
  int x = blockIdx.x;
  if (x < a.p_items) {
    const int per = a.Hk * a.p_splits, pair = x % per;
    it.hk = pair % a.Hk;
    const int split = pair / a.Hk;
    it.row0 = x / per * a.p_rows;
    it.rows = tokens * a.G;
    it.pbeg = split * a.p_chunk;
    it.pend = min(a.S, it.pbeg + a.p_chunk);
    it.slot = a.o_splits + split;
    if (it.row0 >= it.rows) return;
    prefix_items<T, D, kPromptItem>(a.p_rows, a, it, smem, s_pid, s_ml);
  } else {
    x -= a.p_items;
    it.hk = x % a.Hk;
    x /= a.Hk;
    const int split = x % a.o_splits;
    x /= a.o_splits;
    // (late rows see most: they go first)
    const int tile = a.o_tiles - 1 - x % a.o_tiles, b = x / a.o_tiles;
    int c0 = b, c1 = b + 1;
    if (a.cu) {
      c0 = min(max(a.cu[b], 0), tokens);
      c1 = min(max(a.cu[b + 1], c0), tokens);
    }
    const int n = c1 - c0, len = min(max(a.lens[b], 0), a.T << a.lp);
    it.tok0 = c0;
    it.row0 = tile * a.o_rows;
    it.rows = min(n, a.max_new) * a.G;
    if (it.row0 >= it.rows) return;
    const int chunk = own_chunk(len, a.o_splits);
    it.lim0 = len - n + 1;
    it.obeg = min((int64_t)split * chunk, (int64_t)len);
    const int last = min(it.row0 + a.o_rows, it.rows) - 1;   // the tile's row that sees most
    it.oend = min(min(it.obeg + chunk, len), max(0, it.lim0 + last / a.G));
    it.table = a.tables + b * a.t_sb;
    it.slot = split;
    if (a.both) {
      it.oend = min(len, max(0, it.lim0 + last / a.G));
      it.pend = a.prefix_lens ? min(max(a.prefix_lens[b], 0), a.S) : a.S;
      prefix_items<T, D, kBothItem>(a.o_rows, a, it, smem, s_pid, s_ml);
      return;
    }
    if (it.obeg >= it.oend) return;
    prefix_items<T, D, kOwnItem>(a.o_rows, a, it, smem, s_pid, s_ml);
  }
}

// Joins the partials of every query row: grid m_tiles tiles of rows of each
// request; kSub groups of D / 4 threads a row take every kSub-th partial.  A
// partial exists where the row sees keys of its range, and where it does not the
// row has nothing there.  The threads of a group take a partial's (max, sum)
// each, so that all of them are one load deep; then the outputs' loads, four
// dimensions a thread, go out eight at a time.  Several groups a row pay where
// few rows have many partials (128 query rows of 128 dimensions with 17 of them:
// the call 15.5 -> 13.0 us; 444 of 64 dimensions with 21: 38.0 -> 36.4).
template <typename T, int D, int kSub>
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixArgs a) {
  constexpr int kVec = D / 4, kRows = 256 / kVec / kSub;
  static_assert(kRows >= 1, "a row's groups fit a workgroup");
  __shared__ floatx4 s_x[kSub > 1 ? 256 : 1];
  const int b = blockIdx.x / a.m_tiles, tile = blockIdx.x % a.m_tiles;
  int c0 = b, c1 = b + 1;
  if (a.cu) {
    const int tokens = min(max(a.cu[a.B], 0), a.N);
    c0 = min(max(a.cu[b], 0), tokens);
    c1 = min(max(a.cu[b + 1], c0), tokens);
  }
  const int n = c1 - c0, len = min(max(a.lens[b], 0), a.T << a.lp);
  const int j = threadIdx.x % kVec, dim = 4 * j, sub = threadIdx.x / kVec % kSub;
  const int i = tile * kRows + threadIdx.x / kVec / kSub;
  const int t = i / a.Hq, h = i - t * a.Hq;
  const bool live = t < min(n, a.max_new);   // (a row's threads together)
  const int S = a.prefix_lens ? min(max(a.prefix_lens[b], 0), a.S) : a.S;
  const int own = max(0, len - n + 1 + t), chunk = own_chunk(len, a.o_splits);
  const int n_own = (own + chunk - 1) / chunk, n_pre = a.p_splits ? (S + a.p_chunk - 1) / a.p_chunk : 0;
  const int64_t rows_all = (int64_t)a.N * a.Hq, ridx = (int64_t)(c0 + t) * a.Hq + h;
  const int count = live ? n_own + n_pre : 0;
  // partial s of the row: the own ones first, then the prompt's
  auto at = [&](int s) { return (s < n_own ? s : a.o_splits + s - n_own) * rows_all + ridx; };
  typedef float floatx2 __attribute__((ext_vector_type(2)));
  float M = -INFINITY;
  for (int s = j; s < count; s += kVec) M = fmaxf(M, a.part_ml[at(s) * 2]);
#pragma unroll
  for (int o = kVec / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  float L = 0.f;
  floatx4 x = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < count; s0 += kVec) {
    const int mine = min(s0 + j, count - 1);
    const floatx2 ml = *reinterpret_cast<const floatx2*>(a.part_ml + at(mine) * 2);
    const float w = ml[0] == -INFINITY ? 1.f : exp2_hw(ml[0] - M);   // (sums without a max are 0, or NaN)
    if (s0 + j < count) L += ml[1] * w;
    const int todo = min(kVec, count - s0);
    for (int k0 = sub; k0 < todo; k0 += 8 * kSub) {
      floatx4 o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        o[k] = *reinterpret_cast<const floatx4*>(a.part_o + at(s0 + min(k0 + k * kSub, todo - 1)) * D + dim);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float wk = __shfl(w, (k0 + k * kSub) % kVec, kVec);
        if (k0 + k * kSub < todo) x += o[k] * wk;
      }
    }
  }
#pragma unroll
  for (int o = kVec / 2; o > 0; o >>= 1) L += __shfl_xor(L, o, 64);
  if constexpr (kSub > 1) {
    s_x[threadIdx.x] = x;
    __syncthreads();
    if (sub != 0) return;
#pragma unroll
    for (int k = 1; k < kSub; ++k) x += s_x[threadIdx.x + k * kVec];
  }
  if (live) finish_row<T>(a, c0 + t, h, dim, x, M, L);
}

template <typename T, int D>
void launch_prefix_d(const PrefixArgs& a, int64_t items, hipStream_t s) {
  prefix_attn_kernel<T, D><<<(unsigned)items, PrefixShape<T, D>::NW * 64, 0, s>>>(a);
  if (a.both) return;
  if (a.m_sub > 1) prefix_merge_kernel<T, D, kMergeSub><<<(unsigned)(a.B * a.m_tiles), 256, 0, s>>>(a);
  else prefix_merge_kernel<T, D, 1><<<(unsigned)(a.B * a.m_tiles), 256, 0, s>>>(a);
}

template <typename T>
void launch_prefix(const PrefixArgs& a, int64_t items, hipStream_t s) {
  switch (a.D) {
    case 16: launch_prefix_d<T, 16>(a, items, s); break;
    case 32: launch_prefix_d<T, 32>(a, items, s); break;
    case 64: launch_prefix_d<T, 64>(a, items, s); break;
    default: launch_prefix_d<T, 128>(a, items, s); break;
  }
}

}  // namespace hc
