// sy_attend.cu -- attention over a shared prefix and over each sequence's own
// pages, on tcgen05 tensor cores.
//
// Mathematics: out = sum_j p_j v_j / sum_j p_j, p_j = 2^(c (s_j - m)), c =
// scale log2(e), over any split of the keys: partial results (o, m, l) with
// their own m are joined by o = sum_i 2^(c (m_i - m)) o_i, l likewise. So a
// row's keys are cut into tiles of 128, runs of tiles go to different CTAs, and
// a second small kernel joins what was cut.
//
// Work. A unit is a set of rows that read the same keys for one key head: with
// a shared prefix, up to 256 of the batch's rows (sequences x queries x heads of
// the group) over the prefix; and per sequence, up to 256 of its rows over its
// own keys (with the prefix in front when it is not shared: one sequence, or
// more than 128 rows per sequence and key head, where stacking sequences would
// save nothing). The units' tiles form one line that is cut into equal parts,
// one per CTA; every CTA finds its part by a scan over the lengths, so the host
// needs none of them. All of this is decided by sizes; the result depends only
// on sizes, lengths and the number of SMs.
//
// CTA. 12 warps: one loads K and V tiles by TMA through a ring of buffers (the
// pages' rows land in tile order, so a page may end inside a tile), one issues
// the MMAs, two gather query rows, and two streams of four warps each own 128
// softmax rows (one row a thread, so no shuffles). S = Q K^T goes to TMEM, a
// stream reads its row, moves the maximum only when it grew by more than 2^8
// (then rescales its part of O in TMEM), writes P over S as 16-bit, and P V
// accumulates in TMEM with P as the TMEM operand. Units of more than 128 rows
// give each stream 128 of the rows ("wide": one K/V tile serves 256 rows);
// smaller ones give both streams the same rows and every second tile, each with
// its own O and (m, l), so the MMAs of one overlap the softmax of the other.
#include <cmath>

#include "sy_common.cuh"
#include "sy_launch.cuh"
#include "sy_serving.cuh"
#include "sy_tc.cuh"

namespace sy {
namespace {

constexpr int kTile = 128;     // keys of a tile, rows of a stream
constexpr int kThreads = 384;  // load, MMA, 2 query warps, 2 x 4 softmax warps
// Registers a thread: at launch (what the bound of 384 threads leaves), then per role. The shares
// may not sum above the launch's total, or the increase would wait for ever.
constexpr int kRegsLaunch = 168, kRegsOther = 104, kRegsSoftmax = 200;
static_assert(128 * kRegsOther + 256 * kRegsSoftmax <= kThreads * kRegsLaunch, "register shares");
constexpr int kBarBytes = 3072;  // barriers and scratch behind the tiles
constexpr float kGrow = 8.f;   // log2 of the growth of a maximum that is let pass

struct Plan {
  sy_attend_args a;
  int group;             // query heads per key head
  int rows;              // rows per sequence and key head
  int share;             // the prefix has units of its own
  int pre_wide, own_wide;
  int pre_row_tiles, own_row_tiles;
  int pre_tiles;         // tiles of a prefix unit
  int lead_tiles;        // prefix tiles in front of a sequence's own
  int entries;           // sequences x own_row_tiles
  int box;               // rows of a TMA box
  int grid;              // CTAs of the main kernel
  float c;               // scale * log2(e)
  int pre_slot_rows, own_slot_rows;
  long long pre_total;   // tiles of all prefix units
  // workspace
  long long* starts;     // [entries + 1] tiles before an entry's units
  float *pre_ml, *pre_o, *own_ml, *own_o;
};

// ---------------------------------------------------------------------------
// the line of tiles
// ---------------------------------------------------------------------------
__device__ __forceinline__ int own_len(const Plan& p, int b) {
  const long long room = p.a.table_width * p.a.page_size;
  const long long len = p.a.kv_lens[b];
  return (int)(len < 0 ? 0 : len > room ? room : len);
}
// own keys that the last row of a row tile sees
__device__ __forceinline__ int entry_limit(const Plan& p, int row_tile, int len) {
  const int last = p.own_wide ? min(p.rows, (row_tile + 1) * 2 * kTile) - 1 : p.rows - 1;
  const long long lim = (long long)len - p.a.q_len + last / p.group + 1;
  return (int)(lim < 0 ? 0 : lim);
}
__device__ __forceinline__ int entry_tiles(const Plan& p, int lim) {
  return p.lead_tiles + (lim + kTile - 1) / kTile;
}

// The line's cut: CTA c has the tiles [first(c), first(c + 1)).
struct Cut {
  long long total;
  int grid;
  long long q;  // total = q grid + rem
  int rem;
  __device__ __forceinline__ Cut(long long t, int g) : total(t), grid(g), q(t / g), rem((int)(t % g)) {}
  __device__ __forceinline__ long long first(int c) const { return q * c + rem * c / grid; }
  __device__ __forceinline__ int cta_of(long long tile) const {
    int c = min(grid - 1, (int)((float)tile * (float)grid / (float)total));
    while (first(c) > tile) --c;
    while (first(c + 1) <= tile) ++c;
    return c;
  }
};

// A place on the line: tile `off` of unit (e, h); j counts the tiles of this CTA
// in this phase (prefix units, own units), [j0, j1) is its run in the unit.
template <bool Pre>
struct Cursor {
  int e, h, n, lim, len, off, first, j, j0, j1, end;
  __device__ __forceinline__ void enter(const Plan& p) {
    if (Pre) {
      n = p.pre_tiles;
    } else {
      len = own_len(p, e / p.own_row_tiles);
      lim = entry_limit(p, e % p.own_row_tiles, len);
      n = entry_tiles(p, lim);
    }
  }
  __device__ __forceinline__ void run() {
    first = off;
    j0 = j;
    j1 = min(end, j + n - off);
  }
  __device__ __forceinline__ void start(const Plan& p, int entry, int head, int tile, int count) {
    e = entry, h = head, off = tile, j = 0, end = count;
    if (count > 0) {
      enter(p);
      run();
    }
  }
  __device__ __forceinline__ bool live() const { return j < end; }
  __device__ __forceinline__ void next(const Plan& p) {
    ++j;
    ++off;
    if (j < end && off == n) {
      off = 0;
      // prefix units are ordered (head, row tile), own units (entry, head)
      if (Pre) {
        if (++e == p.pre_row_tiles) e = 0, ++h;
      } else {
        do {
          if (++h == (int)p.a.kv_heads) {
            h = 0;
            ++e;
            enter(p);
          }
        } while (n == 0);
      }
      run();
    }
  }
  // to the first tile of the next run
  __device__ __forceinline__ void skip_run(const Plan& p) {
    off += j1 - j - 1;
    j = j1 - 1;
    next(p);
  }
  __device__ __forceinline__ bool whole() const { return first == 0 && j1 - j0 == n; }
  // the tile's part of the keys: in the prefix or not, first key, keys that are there
  __device__ __forceinline__ bool in_prefix(const Plan& p) const { return Pre || off < p.lead_tiles; }
  __device__ __forceinline__ int key0(const Plan& p) const {
    return (Pre || off < p.lead_tiles ? off : off - p.lead_tiles) * kTile;
  }
  __device__ __forceinline__ int keys(const Plan& p) const {
    const int upto = in_prefix(p) ? (int)p.a.prefix_len : lim;
    return min(kTile, upto - key0(p));
  }
};

// The row of a unit: output row (sequence, query, head), query address, and how many own keys it sees.
template <bool Pre>
__device__ __forceinline__ int unit_rows(const Plan& p, int e) {
  if (Pre) {
    const long long all = p.a.batch * p.rows, at = (long long)e * 2 * kTile;
    return (int)(p.pre_wide ? min((long long)2 * kTile, all - at) : all);
  }
  return p.own_wide ? min(2 * kTile, p.rows - e % p.own_row_tiles * 2 * kTile) : p.rows;
}
struct RowAt {
  int b, t, head;
};
template <bool Pre>
__device__ __forceinline__ RowAt row_at(const Plan& p, int e, int h, int r) {
  RowAt x;
  if (Pre) {
    const int row = e * 2 * kTile + r;
    x.b = row / p.rows;
    r = row % p.rows;
  } else {
    x.b = e / p.own_row_tiles;
    r += e % p.own_row_tiles * 2 * kTile;
  }
  x.t = r / p.group;
  x.head = h * p.group + r % p.group;
  return x;
}

// Slot of a partial result. Own units that are wide keep only the runs that a
// CTA shares with another: its first and its last.
template <bool Pre>
__device__ __forceinline__ long long slot_of(const Plan& p, int e, int h, int cta, bool began_before) {
  if (Pre) return (long long)h * p.pre_row_tiles + e + cta;
  if (p.own_wide) return 2ll * cta + (began_before ? 0 : 1);
  return (long long)e * p.a.kv_heads + h + cta;
}

// ---------------------------------------------------------------------------
// the main kernel
// ---------------------------------------------------------------------------
template <int DP>
struct Smem {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kStages = DP == 128 ? 5 : 10;
  static constexpr int kQ = 0;  // two query tiles
  static constexpr int kRing = 2 * kTileBytes;
  static constexpr int kBars = kRing + kStages * kTileBytes;
  static constexpr int kBytes = kBars + kBarBytes;
};

struct Bars {
  uint64_t full[10], empty[10];
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2];
  uint32_t tmem;
  int own_e, own_h, own_off;
  long long scan[kThreads / 32];
  long long q_at[2 * kTile];  // byte offset of a run's query rows
};
static_assert(sizeof(Bars) <= kBarBytes, "barriers and scratch");

struct Part {  // this CTA's part of the line
  long long start, pre_first;
  int pre_count, own_count;
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(kFull, mbar_wait(bar, parity));
}
#define SY_WAIT(bar, parity) \
  if (!warp_wait(bar, parity)) return false

// ---- loads ----
template <int DP, bool Pre>
__device__ __forceinline__ bool load_tiles(const Plan& p, const CUtensorMap* kmap,
                                           const CUtensorMap* vmap, char* smem, Bars* bars,
                                           Cursor<Pre> cur, int& pos) {
  using S = Smem<DP>;
  const int lane = threadIdx.x & 31;
  const int pieces = kTile / p.box;  // boxes of a tile, per 64 columns
  // own keys of narrow units are read once; everything else by several row tiles
  const uint64_t policy = Pre || p.own_wide ? policy_evict_normal() : policy_evict_first();
  for (; cur.live(); cur.next(p)) {
    const bool pre = cur.in_prefix(p);
    const int key0 = cur.key0(p), keys = cur.keys(p);
    const int used = (keys + p.box - 1) / p.box;
    const int b = Pre ? 0 : cur.e / p.own_row_tiles;
    const int* table = pre ? p.a.prefix_pages : p.a.page_table + b * p.a.table_row;
    const int piece = lane % pieces;
    int page = 0, row = 0;
    if (piece < used) {
      const int key = key0 + piece * p.box, ps = (int)p.a.page_size;
      page = __ldg(table + key / ps);
      row = key % ps;
      if (page < 0 || page >= p.a.pages) {
        record_device_error(kDevErrBadIndex);
        page = (int)p.a.pages;  // past the tensor: the copy fills zeros
      }
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv, ++pos) {
      const int stage = pos % S::kStages;
      if (pos >= S::kStages) SY_WAIT(&bars->empty[stage], (pos / S::kStages - 1) & 1);
      if (lane == 0)
        mbar_arrive_expect_tx(&bars->full[stage], (uint32_t)used * p.box * 128u * (DP / 64));
      __syncwarp();
      char* dst = smem + S::kRing + stage * S::kTileBytes;
      for (int i = lane; i < pieces * (DP / 64); i += 32)
        if (piece < used)
          tma_load_4d(dst + (i / pieces) * (kTile * 128) + piece * p.box * 128, kv ? vmap : kmap,
                      &bars->full[stage], (i / pieces) * 64, row, cur.h, page, policy);
    }
  }
  return true;
}

// ---- query rows: gathered into the MMA's swizzled layout ----
// 16 lanes copy a row's 16-byte chunks (fewer than 16 below head_dim 128), four
// rows a step; where the rows start is worked out once per run.
template <int DP, bool Pre>
__device__ __forceinline__ bool load_queries(const Plan& p, char* smem, Bars* bars, Cursor<Pre> cur,
                                             bool wide, int& slot) {
  using S = Smem<DP>;
  const int tid = threadIdx.x - 64;  // 64 threads
  const int c = tid & 15, r0 = tid >> 4;
  const bool on = c < (int)p.a.head_dim / 8;
  const char* q = static_cast<const char*>(p.a.q) + c * 16;
  const uint32_t to = smem_u32(smem) + S::kQ + (c >> 3) * (kTile * 128);
  while (cur.live()) {
    const int rows = unit_rows<Pre>(p, cur.e);
    named_sync(1, 64);  // the table's readers are done
    for (int r = tid; r < rows; r += 64) {
      const RowAt at = row_at<Pre>(p, cur.e, cur.h, r);
      bars->q_at[r] = 2 * (at.b * p.a.q_b + at.t * p.a.q_t + at.head * p.a.q_h);
    }
    named_sync(1, 64);
    for (int s = 0; s < (wide ? 2 : 1); ++s, ++slot) {
      const int buf = slot & 1;
      if (slot >= 2) SY_WAIT(&bars->q_empty[buf], (slot / 2 - 1) & 1);
      const int count = min(kTile, rows - s * kTile);
      if (on)
        for (int r = r0; r < count; r += 4)
          cp_async16(to + buf * S::kTileBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                     q + bars->q_at[s * kTile + r]);
      cp_async_wait_all();
      fence_proxy_async();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&bars->q_full[buf]);
    }
    cur.skip_run(p);
  }
  return true;
}

// ---- MMAs ----
struct MmaState {
  int pos = 0;         // ring position of the phase's first tile
  int slot = 0;        // query slots used by S so far
  uint32_t p_phase = 0;  // bit s: parity of stream s's next P
};

template <int DP, bool BF16, bool Pre>
__device__ __forceinline__ bool issue_mmas(const Plan& p, char* smem, Bars* bars, uint32_t tmem,
                                           Cursor<Pre> cur, bool wide, MmaState& st) {
  using S = Smem<DP>;
  constexpr uint32_t kIdS = f16_idesc(BF16, kTile, kTile, false);
  constexpr uint32_t kIdO = f16_idesc(BF16, kTile, DP, true);
  const int lane = threadIdx.x & 31;
  const uint32_t base = smem_u32(smem);
  Cursor<Pre> ahead = cur;

  // S of stream s for the tile `ahead` stands at
  auto scores = [&](int s) -> bool {
    const int kpos = st.pos + 2 * ahead.j, stage = kpos % S::kStages;
    const int slots = wide ? 2 : 1;
    const int slot = st.slot + (wide ? s : 0), buf = slot & 1;
    if (!wide || s == 0) SY_WAIT(&bars->full[stage], (kpos / S::kStages) & 1);
    if (ahead.j == ahead.j0) SY_WAIT(&bars->q_full[buf], (slot / 2) & 1);
    tc_fence_after();
    if (lane == 0) {
      const uint64_t a = sw128_desc(base + S::kQ + buf * S::kTileBytes, 16, 1024);
      const uint64_t b = sw128_desc(base + S::kRing + stage * S::kTileBytes, 16, 1024);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint64_t step = (uint64_t)((k >> 2) * (kTile * 128) + (k & 3) * 32) >> 4;
        mma_ss(tmem + s * kTile, a + step, b + step, kIdS, k > 0);
      }
      tc_commit(&bars->s_full[s]);
      if (!wide || s == 1) tc_commit(&bars->empty[stage]);
      if (ahead.j + 1 == ahead.j1) tc_commit(&bars->q_empty[buf]);
    }
    __syncwarp();
    if (!wide || s == 1) {
      if (ahead.j + 1 == ahead.j1) st.slot += slots;
      ahead.next(p);
    }
    return true;
  };

  for (int i = 0; i < (wide ? 1 : 2); ++i)
    if (ahead.live())
      for (int s = wide ? 0 : i; s <= (wide ? 1 : i); ++s)
        if (!scores(s)) return false;

  for (; cur.live(); cur.next(p)) {
    const int vpos = st.pos + 2 * cur.j + 1, stage = vpos % S::kStages;
    SY_WAIT(&bars->full[stage], (vpos / S::kStages) & 1);
    const int keys = cur.keys(p);
    if (keys < kTile) {
      // what lies behind the last key in its page may be anything, and 0 * NaN is NaN
      char* v = smem + S::kRing + stage * S::kTileBytes;
      const int n = (kTile - keys) * 8;
      for (int half = 0; half < DP / 64; ++half)
        for (int i = lane; i < n; i += 32)
          *reinterpret_cast<uint4*>(v + half * (kTile * 128) + keys * 128 + i * 16) =
              make_uint4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
    }
    const uint64_t b = sw128_desc(base + S::kRing + stage * S::kTileBytes, kTile * 128, 1024);
    for (int s = wide ? 0 : cur.j & 1; s <= (wide ? 1 : cur.j & 1); ++s) {
      SY_WAIT(&bars->p_full[s], (st.p_phase >> s) & 1);
      st.p_phase ^= 1u << s;
      tc_fence_after();
      const int step = wide ? 1 : 2;  // tiles between two of this stream
      if (lane == 0) {
        const bool fresh = cur.j - cur.j0 < step;
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
          mma_ts(tmem + 2 * kTile + s * kTile, tmem + s * kTile + k * 8, b + (uint64_t)(k * (2048 >> 4)),
                 kIdO, k > 0 || !fresh);
        if (!wide || s == 1) tc_commit(&bars->empty[stage]);
        if (cur.j1 - cur.j <= step) tc_commit(&bars->o_full[s]);
      }
      __syncwarp();
      if (ahead.live() && !scores(s)) return false;
    }
  }
  st.pos += 2 * cur.end;
  return true;
}

// ---- softmax ----
struct SoftState {
  int s_count = 0, o_count = 0;
};

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// fp16 weights are kept 2^6 higher: they may reach 2^(6 + 8) and lose bits only
// below 2^-20 of the highest.
template <typename T>
__device__ __forceinline__ constexpr float weight_shift() {
  return sizeof(T) == 2 && std::is_same<T, __half>::value ? 6.f : 0.f;
}

__device__ __forceinline__ void mask_columns(uint32_t* x, int upto) {
#pragma unroll
  for (int k = 0; k < 32; ++k)
    if (k >= upto) x[k] = 0xff800000u;  // -inf
}
__device__ __forceinline__ float row_max(const uint32_t* x) {
  float a = __uint_as_float(x[0]), b = __uint_as_float(x[1]);
#pragma unroll
  for (int k = 2; k < 32; k += 2) {
    a = fmaxf(a, __uint_as_float(x[k]));
    b = fmaxf(b, __uint_as_float(x[k + 1]));
  }
  return fmaxf(a, b);
}

template <typename T, int DP, bool Pre>
__device__ __forceinline__ bool softmax_tiles(const Plan& p, Bars* bars, uint32_t tmem, int s,
                                              Cursor<Pre> cur, bool wide, const Part& part,
                                              SoftState& st) {
  const int row = threadIdx.x & 127, warp = row >> 5;
  const uint32_t lanes = (uint32_t)warp << 21;  // TMEM lane in bits 16..31
  const uint32_t s_at = tmem + lanes + s * kTile, o_at = tmem + lanes + (2 + s) * kTile;
  const float c = p.c;
  float m = -INFINITY, l = 0.f;
  int rows = 0, see = 0;
  for (; cur.live(); cur.next(p)) {
    if (!wide && (cur.j & 1) != s) continue;
    const int step = wide ? 1 : 2;
    const bool fresh = cur.j - cur.j0 < step;
    if (fresh) {
      m = -INFINITY;
      l = 0.f;
      rows = unit_rows<Pre>(p, cur.e) - (wide ? s * kTile : 0);
      if (!Pre) {  // own keys that this row sees
        const RowAt at = row_at<Pre>(p, cur.e, cur.h, (wide ? s * kTile : 0) + min(row, rows - 1));
        see = cur.len - (int)p.a.q_len + at.t + 1;
      }
    }
    SY_WAIT(&bars->s_full[s], st.s_count & 1);
    ++st.s_count;
    tc_fence_after();
    if (warp * 32 < rows) {
      uint32_t x[4][32];
      tmem_ld32(s_at, x[0]);
      tmem_ld32(s_at + 32, x[1]);
      const int keys = cur.keys(p);
      const int upto = cur.in_prefix(p) ? keys : min(keys, see - cur.key0(p));
      const bool masked = __any_sync(kFull, upto < kTile);
      tmem_wait_ld(x[0]);
      tmem_landed(x[1]);
      tmem_ld32(s_at + 64, x[2]);
      tmem_ld32(s_at + 96, x[3]);
      if (masked) mask_columns(x[0], upto), mask_columns(x[1], upto - 32);
      float top = fmaxf(row_max(x[0]), row_max(x[1]));
      tmem_wait_ld(x[2]);
      tmem_landed(x[3]);
      if (masked) mask_columns(x[2], upto - 64), mask_columns(x[3], upto - 96);
      top = fmaxf(top, fmaxf(row_max(x[2]), row_max(x[3])));
      // The first maximum is taken as it is; later ones only past 2^kGrow.
      const bool moves = m == -INFINITY ? top > -INFINITY : (top - m) * c > kGrow;
      if (__any_sync(kFull, moves)) {
        const float keep = !moves ? 1.f : m == -INFINITY ? 0.f : ex2((m - top) * c);
        if (moves) m = top;
        l *= keep;
        if (!fresh) {
          // S of this tile follows the last P V in the MMA order, so O stands still
#pragma unroll
          for (int i = 0; i < DP / 32; ++i) {
            uint32_t o[32];
            tmem_ld32(o_at + 32 * i, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
            tmem_st32(o_at + 32 * i, o);
          }
        }
      }
      const float off = (m == -INFINITY ? 0.f : -m * c) + weight_shift<T>();
      const float2 c2 = make_float2(c, c), off2 = make_float2(off, off);
      float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          float2 u = make_float2(__uint_as_float(x[i][k]), __uint_as_float(x[i][k + 1]));
          float2 w = make_float2(__uint_as_float(x[i][k + 2]), __uint_as_float(x[i][k + 3]));
          u = __ffma2_rn(u, c2, off2);
          w = __ffma2_rn(w, c2, off2);
          u = make_float2(ex2(u.x), ex2(u.y));
          w = make_float2(ex2(w.x), ex2(w.y));
          sum0 = __fadd2_rn(sum0, u);
          sum1 = __fadd2_rn(sum1, w);
          x[i][k / 2] = pack16<T>(u.x, u.y);
          x[i][k / 2 + 1] = pack16<T>(w.x, w.y);
        }
        tmem_st16(s_at + 16 * i, x[i]);  // P takes half of S's columns
      }
      l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
      tmem_wait_st();
    }
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&bars->p_full[s]);

    if (cur.j1 - cur.j <= step) {  // this stream's last tile of the run
      SY_WAIT(&bars->o_full[s], st.o_count & 1);
      ++st.o_count;
      tc_fence_after();
      if (warp * 32 < rows) {
        const RowAt at = row_at<Pre>(p, cur.e, cur.h, (wide ? s * kTile : 0) + min(row, rows - 1));
        const long long out_row = (at.b * p.a.q_len + at.t) * p.a.q_heads + at.head;
        const bool final = !Pre && !p.share && cur.whole() && (wide || cur.n == 1);
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const bool mine = row < rows;
        float* po = nullptr;
        if (!final) {
          const bool before = cur.first > 0;
          const long long slot = 2 * slot_of<Pre>(p, cur.e, cur.h, blockIdx.x, before) + s;
          const long long at_row = slot * (Pre ? p.pre_slot_rows : p.own_slot_rows) + min(row, rows - 1);
          po = (Pre ? p.pre_o : p.own_o) + at_row * DP;
          if (mine)
            reinterpret_cast<float2*>(Pre ? p.pre_ml : p.own_ml)[at_row] = make_float2(m * c, l);
        } else if (mine && p.a.lse) {
          p.a.lse[out_row] =
              l > 0.f ? m * (c * 0.69314718055994531f) + logf(l) - weight_shift<T>() * 0.69314718055994531f
                      : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          uint32_t o[32];
          tmem_ld32(o_at + 32 * i, o);
          tmem_wait_ld(o);
          if (!final) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              if (mine)
                *reinterpret_cast<uint4*>(po + 32 * i + k) =
                    make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          } else {
            T* out = static_cast<T*>(p.a.out) + out_row * p.a.head_dim + 32 * i;
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              uint4 w;
              float f[8];
#pragma unroll
              for (int u = 0; u < 8; ++u) f[u] = l > 0.f ? __uint_as_float(o[k + u]) * inv : 0.f;
              w = make_uint4(pack16<T>(f[0], f[1]), pack16<T>(f[2], f[3]), pack16<T>(f[4], f[5]),
                             pack16<T>(f[6], f[7]));
              if (mine && 32 * i + k < (int)p.a.head_dim) *reinterpret_cast<uint4*>(out + k) = w;
            }
          }
        }
        tc_fence_before();  // the next run's P V overwrites O after the next p_full
      }
    }
  }
  return true;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const Plan p, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  using S = Smem<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) char smem[];
  Bars* bars = reinterpret_cast<Bars*>(smem + S::kBars);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  if (smem_u32(smem) & 1023u) {  // the swizzle and the descriptors count on it
    if (tid == 0) record_device_error(kDevErrBadPlan);
    return;
  }

  // where this CTA's part of the line starts
  const int per = (p.entries + kThreads - 1) / kThreads;
  const int e_first = min(p.entries, tid * per), e_last = min(p.entries, e_first + per);
  long long mine = 0;
  for (int e = e_first; e < e_last; ++e) {
    const int b = e / p.own_row_tiles;
    const int len = own_len(p, b);
    if (blockIdx.x == 0 && len != p.a.kv_lens[b]) record_device_error(kDevErrBadIndex);
    mine += entry_tiles(p, entry_limit(p, e % p.own_row_tiles, len));
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(kFull, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) bars->scan[warp] = upto;
  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->q_full[i], 2);
      mbar_init(&bars->q_empty[i], 1);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], 4);
      mbar_init(&bars->o_full[i], 1);
    }
    mbar_fence_init();
    tma_prefetch_map(&kmap);
    tma_prefetch_map(&vmap);
  }
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) upto += bars->scan[w];
    total += bars->scan[w];
  }
  const int heads = (int)p.a.kv_heads;
  total = total * heads + p.pre_total;
  Part part;
  const Cut cut(total, p.grid);
  part.start = cut.first(blockIdx.x);
  const long long stop = cut.first(blockIdx.x + 1);
  const long long pre_stop = min(stop, p.pre_total);
  part.pre_first = part.start;
  part.pre_count = (int)max(0ll, pre_stop - part.start);
  const long long own_first = max(part.start, p.pre_total) - p.pre_total;
  part.own_count = (int)max(0ll, stop - p.pre_total - own_first);
  long long before = (upto - mine) * heads;
  for (int e = e_first; e < e_last; ++e) {
    const int n = entry_tiles(p, entry_limit(p, e % p.own_row_tiles, own_len(p, e / p.own_row_tiles)));
    if (own_first >= before && own_first < before + (long long)n * heads) {
      bars->own_e = e;
      bars->own_h = (int)((own_first - before) / n);
      bars->own_off = (int)((own_first - before) % n);
    }
    if (blockIdx.x == 0) p.starts[e] = before;
    before += (long long)n * heads;
  }
  if (blockIdx.x == 0 && tid == kThreads - 1) p.starts[p.entries] = total - p.pre_total;
  if (part.pre_count + part.own_count == 0) return;

  if (warp == 2) tmem_alloc(&bars->tmem, 512);
  if ((int)p.a.head_dim < DP)  // columns past head_dim stay zero: K's are filled with zeros
    for (int i = tid; i < 2 * S::kTileBytes / 16; i += kThreads)
      reinterpret_cast<uint4*>(smem + S::kQ)[i] = make_uint4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;

  Cursor<true> pre;
  Cursor<false> own;
  {
    const long long unit = p.pre_tiles > 0 ? part.pre_first / p.pre_tiles : 0;
    pre.start(p, part.pre_count ? (int)(unit % p.pre_row_tiles) : 0,
              part.pre_count ? (int)(unit / p.pre_row_tiles) : 0,
              part.pre_count ? (int)(part.pre_first % p.pre_tiles) : 0, part.pre_count);
    own.start(p, part.own_count ? bars->own_e : 0, part.own_count ? bars->own_h : 0,
              part.own_count ? bars->own_off : 0, part.own_count);
  }
  const bool pre_wide = p.pre_wide, own_wide = p.own_wide;
  // A softmax thread holds a row of 128 scores: the other warps hand registers over.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 0) {
      int pos = 0;
      load_tiles<DP, true>(p, &kmap, &vmap, smem, bars, pre, pos) &&
          load_tiles<DP, false>(p, &kmap, &vmap, smem, bars, own, pos);
      // every copy has landed before the CTA may end
      for (int i = max(0, pos - S::kStages); i < pos; ++i)
        mbar_wait(&bars->full[i % S::kStages], (i / S::kStages) & 1);
    } else if (warp == 1) {
      MmaState st;
      issue_mmas<DP, kBf16, true>(p, smem, bars, tmem, pre, pre_wide, st) &&
          issue_mmas<DP, kBf16, false>(p, smem, bars, tmem, own, own_wide, st);
    } else {
      int slot = 0;
      load_queries<DP, true>(p, smem, bars, pre, pre_wide, slot) &&
          load_queries<DP, false>(p, smem, bars, own, own_wide, slot);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    SoftState st;
    const int s = warp >= 8;
    softmax_tiles<T, DP, true>(p, bars, tmem, s, pre, pre_wide, part, st) &&
        softmax_tiles<T, DP, false>(p, bars, tmem, s, own, own_wide, part, st);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// joining the parts of a row
// ---------------------------------------------------------------------------
struct Runs {
  long long start, stop, phase;  // tiles of the unit, first tile of its phase
};

constexpr int kJoinWarps = 8, kJoinRows = 16, kJoinBlocks = 5;  // blocks an SM

template <typename T, int DP>
__global__ void __launch_bounds__(32 * kJoinWarps, kJoinBlocks) join_kernel(const Plan p) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int unit_max = p.own_wide ? min(p.rows, 2 * kTile) : p.rows;
  const int groups = (unit_max + kJoinRows - 1) / kJoinRows;
  const int heads = (int)p.a.kv_heads;
  const long long block = blockIdx.x;
  const int e = (int)(block / groups / heads), h = (int)(block / groups % heads);
  const int r0 = (int)(block % groups) * kJoinRows;
  const long long own_total = p.starts[p.entries], total = own_total + p.pre_total;
  const long long n = (p.starts[e + 1] - p.starts[e]) / heads;
  Runs own;
  own.start = p.pre_total + p.starts[e] + h * n, own.stop = own.start + n;
  own.phase = p.pre_total;
  const Cut cut(total, p.grid);
  const int c0 = n ? cut.cta_of(own.start) : 0, c1 = n ? cut.cta_of(own.stop - 1) : -1;
  if (!p.share && n && c0 == c1 && (p.own_wide || n == 1)) return;  // already written
  const int rows = unit_rows<false>(p, e);
  const float ln2 = 0.69314718055994531f;
  for (int r = r0 + warp; r < min(rows, r0 + kJoinRows); r += kJoinWarps) {
    const RowAt at = row_at<false>(p, e, h, r);
    const long long out_row = (at.b * p.a.q_len + at.t) * p.a.q_heads + at.head;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    // candidates: (CTA, stream) of the prefix unit, then of the own unit
    int pu_e = 0, pu_r = 0, pc0 = 0, pc1 = -1;
    Runs pre = own;
    if (p.share) {
      const int row = at.b * p.rows + r;
      pu_e = row / (2 * kTile), pu_r = row % (2 * kTile);
      pre.start = ((long long)h * p.pre_row_tiles + pu_e) * p.pre_tiles;
      pre.stop = pre.start + p.pre_tiles, pre.phase = 0;
      pc0 = cut.cta_of(pre.start), pc1 = cut.cta_of(pre.stop - 1);
    }
    const int n_pre = 2 * (pc1 - pc0 + 1), n_all = n_pre + 2 * (c1 - c0 + 1);
    for (int base = 0; base < n_all; base += 32) {
      const int i = base + lane;
      float cm = -INFINITY, cl = 0.f;
      long long at_row = 0;
      const bool is_pre = i < n_pre;
      if (i < n_all) {
        const int k = is_pre ? i : i - n_pre;
        const int cta = (is_pre ? pc0 : c0) + (k >> 1), s = k & 1;
        const Runs& u = is_pre ? pre : own;
        const bool wide = is_pre ? p.pre_wide : p.own_wide;
        const long long c_start = cut.first(cta), c_stop = cut.first(cta + 1);
        const long long from = max(u.start, c_start), to = min(u.stop, c_stop);
        const int ur = is_pre ? pu_r : r;
        bool there = to > from;
        if (wide)
          there = there && (ur >> 7) == s;
        else  // tile j of a CTA's phase went to stream j & 1
          there = there && (to - from >= 2 || ((from - max(c_start, u.phase)) & 1) == s);
        if (there) {
          const long long slot =
              2 * (is_pre ? slot_of<true>(p, pu_e, h, cta, false)
                          : slot_of<false>(p, e, h, cta, u.start < c_start)) + s;
          at_row = slot * (is_pre ? p.pre_slot_rows : p.own_slot_rows) + (wide ? ur & 127 : ur);
          const float2 ml = reinterpret_cast<const float2*>(is_pre ? p.pre_ml : p.own_ml)[at_row];
          if (ml.y > 0.f) cm = ml.x, cl = ml.y;
        }
      }
      const float top = fmaxf(m, warp_max(cm));
      if (top == -INFINITY) continue;
      const float keep = m == -INFINITY ? 0.f : ex2(m - top);
      const float w = cm == -INFINITY ? 0.f : ex2(cm - top);
      m = top;
      l = l * keep + warp_sum(w * cl);
      o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
      const float* src = (is_pre ? p.pre_o : p.own_o) + at_row * DP;
      unsigned live = __ballot_sync(kFull, w > 0.f);
      while (live) {
        constexpr int kAtOnce = 4;
        float4 x[kAtOnce];
        float f[kAtOnce];
        unsigned rest = live;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int from = rest ? __ffs(rest) - 1 : 0;
          f[k] = __shfl_sync(kFull, w, from);
          const float* ptr = reinterpret_cast<const float*>(
              __shfl_sync(kFull, reinterpret_cast<unsigned long long>(src), from));
          if (!rest) f[k] = 0.f;
          x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (rest && lane * 4 < DP) x[k] = __ldcs(reinterpret_cast<const float4*>(ptr) + lane);
          rest &= rest - 1;
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          o.x += f[k] * x[k].x, o.y += f[k] * x[k].y;
          o.z += f[k] * x[k].z, o.w += f[k] * x[k].w;
        }
        live = rest;
      }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    if (lane * 4 < (int)p.a.head_dim) {
      T* out = static_cast<T*>(p.a.out) + out_row * p.a.head_dim + lane * 4;
      *reinterpret_cast<uint2*>(out) =
          make_uint2(pack16<T>(o.x * inv, o.y * inv), pack16<T>(o.z * inv, o.w * inv));
    }
    if (lane == 0 && p.a.lse)
      p.a.lse[out_row] = l > 0.f ? m * ln2 + logf(l) - weight_shift<T>() * ln2 : -INFINITY;
  }
}

// No page anywhere: every row is empty.
template <typename T>
__global__ void __launch_bounds__(256) no_keys_kernel(const sy_attend_args a) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  const long long rows = a.batch * a.q_len * a.q_heads;
  if (i < rows * (a.head_dim / 8)) static_cast<uint4*>(a.out)[i] = make_uint4(0, 0, 0, 0);
  if (i < rows && a.lse) a.lse[i] = -INFINITY;
  if (i < a.batch && (a.kv_lens[i] != 0 || a.prefix_len > 0)) record_device_error(kDevErrBadIndex);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int64_t align16(int64_t x) { return (x + 15) / 16 * 16; }

// Fills everything but the pointers into the workspace; returns its bytes.
int64_t make_plan(const sy_attend_args& a, int sms, Plan* p, char* ws) {
  p->a = a;
  const int dp = a.head_dim > 64 ? 128 : 64;
  p->group = (int)(a.q_heads / a.kv_heads);
  p->rows = (int)(a.q_len * p->group);
  const int64_t pre_rows = a.batch * p->rows;
  p->share = a.prefix_len > 0 && a.batch > 1 && p->rows <= kTile;
  const int ptiles = (int)((a.prefix_len + kTile - 1) / kTile);
  p->pre_tiles = p->share ? ptiles : 0;
  p->lead_tiles = p->share ? 0 : ptiles;
  p->pre_wide = pre_rows > kTile;
  p->own_wide = p->rows > kTile;
  p->pre_row_tiles = p->pre_wide ? (int)((pre_rows + 2 * kTile - 1) / (2 * kTile)) : 1;
  p->own_row_tiles = p->own_wide ? (p->rows + 2 * kTile - 1) / (2 * kTile) : 1;
  p->entries = (int)(a.batch * p->own_row_tiles);
  p->pre_total = (int64_t)p->pre_tiles * p->pre_row_tiles * a.kv_heads;
  p->box = (int)(a.page_size & -a.page_size);
  if (p->box > kTile) p->box = kTile;
  p->grid = sms;
  p->c = a.scale * 1.44269504088896341f;
  p->pre_slot_rows = (int)(pre_rows < kTile ? pre_rows : kTile);
  p->own_slot_rows = p->rows < kTile ? p->rows : kTile;
  const int64_t pre_slots =
      p->share ? 2 * (a.kv_heads * p->pre_row_tiles + p->grid) * p->pre_slot_rows : 0;
  const int64_t own_slots =
      (p->own_wide ? 4 * (int64_t)p->grid : 2 * (p->entries * a.kv_heads + p->grid)) * p->own_slot_rows;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* q = ws + at;
    at += align16(bytes);
    return q;
  };
  p->starts = reinterpret_cast<long long*>(take((p->entries + 1) * 8));
  p->pre_ml = reinterpret_cast<float*>(take(pre_slots * 8));
  p->own_ml = reinterpret_cast<float*>(take(own_slots * 8));
  p->pre_o = reinterpret_cast<float*>(take(pre_slots * dp * 4));
  p->own_o = reinterpret_cast<float*>(take(own_slots * dp * 4));
  return at;
}

// cuTensorMapEncodeTiled through the runtime, so nothing links the driver library
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault,
                                         &r) != cudaSuccess)
      return (EncodeTiled) nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

bool cache_map(CUtensorMap* map, const void* base, const sy_attend_args& a, int64_t page,
               int64_t head, int64_t row, int box) {
  EncodeTiled enc = encode_tiled();
  if (!enc) return false;
  // an axis of one element may carry any stride; the map wants a positive one
  const cuuint64_t dims[4] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.page_size,
                              (cuuint64_t)a.kv_heads, (cuuint64_t)a.pages};
  const cuuint64_t strides[3] = {(cuuint64_t)row * 2, (cuuint64_t)(a.kv_heads > 1 ? head : 8) * 2,
                                 (cuuint64_t)(a.pages > 1 ? page : 8) * 2};
  const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1};
  const cuuint32_t steps[4] = {1, 1, 1, 1};
  return enc(map,
             a.dtype == SY_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
             4, const_cast<void*>(base), dims, strides, boxes, steps,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
cudaError_t launch_type(const Plan& p, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st) {
  static const cudaError_t fits = [] {  // the register shares count on the launch's total
    cudaFuncAttributes f;
    const cudaError_t e = cudaFuncGetAttributes(&f, attend_kernel<T, DP>);
    return e != cudaSuccess ? e : f.numRegs == kRegsLaunch ? cudaSuccess : cudaErrorInvalidConfiguration;
  }();
  if (fits != cudaSuccess) return fits;
  cudaError_t e = launch_smem(attend_kernel<T, DP>, dim3(p.grid), kThreads, Smem<DP>::kBytes, st, p,
                              k, v);
  if (e != cudaSuccess) return e;
  const int unit_max = p.own_wide ? (p.rows < 2 * kTile ? p.rows : 2 * kTile) : p.rows;
  const int64_t groups = (unit_max + kJoinRows - 1) / kJoinRows;
  return launch_smem_pdl(join_kernel<T, DP>, dim3((unsigned)(p.entries * p.a.kv_heads * groups)),
                         32 * kJoinWarps, 0, st, p);
}

}  // namespace

cudaError_t take_attend_error(unsigned int* word) {
  const cudaError_t e = cudaMemcpyFromSymbol(word, g_device_error, sizeof(*word));
  if (e != cudaSuccess) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
}

int64_t attend_workspace(const sy_attend_args& a, const ServingDev& dev) {
  Plan p;
  return make_plan(a, dev.sms, &p, nullptr);
}

cudaError_t launch_attend(const sy_attend_args& a, const ServingDev& dev, cudaStream_t st) {
  if (a.pages == 0 || (a.table_width == 0 && a.prefix_len == 0)) {
    const int64_t n = a.batch * a.q_len * a.q_heads * (a.head_dim / 8);
    return launch_smem(no_keys_kernel<__half>, dim3((unsigned)((n + 255) / 256)), 256, 0, st, a);
  }
  Plan p;
  make_plan(a, dev.sms, &p, static_cast<char*>(a.workspace));
  CUtensorMap k, v;
  if (!cache_map(&k, a.k_cache, a, a.kc_page, a.kc_head, a.kc_row, p.box) ||
      !cache_map(&v, a.v_cache, a, a.vc_page, a.vc_head, a.vc_row, p.box))
    return cudaErrorInvalidValue;
  const bool big = a.head_dim > 64;
  if (a.dtype == SY_BF16)
    return big ? launch_type<__nv_bfloat16, 128>(p, k, v, st) : launch_type<__nv_bfloat16, 64>(p, k, v, st);
  return big ? launch_type<__half, 128>(p, k, v, st) : launch_type<__half, 64>(p, k, v, st);
}

}  // namespace sy
