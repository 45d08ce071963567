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
// Every unit also stands on the line with a few places of its own for what a
// run costs beside its tiles (query rows in, O out, the pipeline's filling).
//
// CTA. 12 warps: one loads K and V tiles by TMA through a ring of buffers (the
// pages' rows land in tile order, so a page may end inside a tile), one gathers
// query rows, two issue MMAs, and two streams of four warps each own 128
// softmax rows (one row a thread, so no shuffles). S = Q K^T goes to TMEM, a
// stream reads its row, moves the maximum only when it grew much (then rescales
// its part of O in TMEM), writes P over S as 16-bit, and P V
// accumulates in TMEM with P as the TMEM operand. Units of more than 128 rows
// give each stream 128 of the rows ("wide": one K/V tile serves 256 rows);
// smaller ones give both streams the same rows and half of every tile's keys, each
// with its own O and (m, l).
//
// What bounds it (B200, bf16, head_dim 128). Few rows a sequence: DRAM; four
// sequences of up to 65536 keys take 93 us, 0.88 of the measured copy rate, with
// the 8 us of the join 0.81. Many rows: a step's scores wait for P V two steps
// back, as two score buffers a stream are what 512 TMEM columns hold beside two
// outputs; a prompt of 4096 tokens takes 107 us and 16 us of joining, 565 TFLOP/s
// over both, with the tensor pipe 37 % and the exponentials 38 % busy.
#include <cmath>

#include "sy_common.cuh"
#include "sy_launch.cuh"
#include "sy_serving.cuh"
#include "sy_tc.cuh"

namespace sy {
namespace {

constexpr int kTile = 128;     // keys of a tile, rows of a stream
constexpr int kThreads = 384;  // load, query, 2 MMA warps, 2 streams x 4 softmax warps
constexpr int kHalf = 64;      // keys of a step of the softmax
constexpr int kBarBytes = 3072;  // barriers and scratch behind the tiles

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
  int pre_extra, own_extra;  // places of a unit on the line beside its tiles'
  int pre_cost;          // places of a prefix tile; an own tile has one
  int pre_total;         // places of all prefix units
  // workspace
  int* starts;           // [entries + 1] places before an entry's units
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
// places of a unit of n tiles; its tiles are the last n of them
__device__ __forceinline__ int own_places(const Plan& p, int n) { return n > 0 ? n + p.own_extra : 0; }

// The line's cut: CTA c has the places [first(c), first(c + 1)). (The host
// checked that the line is shorter than 2^31.)
struct Cut {
  int q, rem;  // the first rem CTAs have q + 1 places, the others q
  __device__ __forceinline__ Cut(int total, int grid) : q(total / grid), rem(total - q * grid) {}
  __device__ __forceinline__ int first(int c) const { return q * c + min(c, rem); }
  __device__ __forceinline__ int cta_of(int place) const {
    const int big = rem * (q + 1);
    return place < big ? place / (q + 1) : rem + (place - big) / q;
  }
};

// A CTA's part of the line in tiles: the first of the prefix units' tiles, the
// entry, head and tile it begins at in the own units, and how many of each.
struct Part {
  int pre_first, pre_count, own_e, own_h, own_off, own_count;
};

// A place on the line: tile `off` of unit (e, h) of a phase (prefix units, own
// units); j counts the tiles of this CTA in the phase, [j0, j1) is its run in
// the unit.
struct Cursor {
  bool pre;
  int e, h, n, lim, len, off, first, j, j0, j1, end;
  __device__ __forceinline__ void enter(const Plan& p) {
    if (pre) {
      n = p.pre_tiles;
      lim = len = 0;
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
  __device__ __forceinline__ void start(const Plan& p, const Part& part, bool prefix) {
    pre = prefix;
    j = 0;
    if (pre) {
      end = part.pre_count;
      if (end == 0) return;
      const int unit = part.pre_first / p.pre_tiles;
      off = part.pre_first % p.pre_tiles;
      e = unit % p.pre_row_tiles, h = unit / p.pre_row_tiles;
    } else {
      end = part.own_count;
      if (end == 0) return;
      e = part.own_e, h = part.own_h, off = part.own_off;
    }
    enter(p);
    run();
  }
  __device__ __forceinline__ bool live() const { return j < end; }
  // to the first tile of the next run
  __device__ __forceinline__ void next_run(const Plan& p) {
    j = j1;
    if (j >= end) return;
    off = 0;
    // prefix units are ordered (head, row tile), own units (entry, head)
    if (pre) {
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
  __device__ __forceinline__ bool whole() const { return first == 0 && j1 - j0 == n; }
  // tile `t` of the unit: in the prefix or not, its first key, the keys that are there
  __device__ __forceinline__ bool in_prefix(const Plan& p, int t) const { return pre || t < p.lead_tiles; }
  __device__ __forceinline__ int key0(const Plan& p, int t) const {
    return (in_prefix(p, t) ? t : t - p.lead_tiles) * kTile;
  }
  __device__ __forceinline__ int keys(const Plan& p, int t) const {
    return min(kTile, (in_prefix(p, t) ? (int)p.a.prefix_len : lim) - key0(p, t));
  }
};

// The rows of a unit, and one of them: sequence, query, head.
__device__ __forceinline__ int unit_rows(const Plan& p, bool pre, int e) {
  if (pre) {
    const long long all = p.a.batch * p.rows, at = (long long)e * 2 * kTile;
    return (int)(p.pre_wide ? min((long long)2 * kTile, all - at) : all);
  }
  return p.own_wide ? min(2 * kTile, p.rows - e % p.own_row_tiles * 2 * kTile) : p.rows;
}
struct RowAt {
  int b, t, head;
};
__device__ __forceinline__ RowAt row_at(const Plan& p, bool pre, int e, int h, int r) {
  RowAt x;
  if (pre) {
    r += e * 2 * kTile;
    x.b = r / p.rows;
    r -= x.b * p.rows;
  } else {
    x.b = e / p.own_row_tiles;
    r += (e - x.b * p.own_row_tiles) * 2 * kTile;
  }
  x.t = r / p.group;
  x.head = h * p.group + r - x.t * p.group;
  return x;
}

// Slot of a partial result. Own units that are wide keep only the runs that a
// CTA shares with another: its first and its last.
__device__ __forceinline__ long long slot_of(const Plan& p, bool pre, int e, int h, int cta,
                                             bool began_before) {
  if (pre) return (long long)h * p.pre_row_tiles + e + cta;
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
  // [stream][buffer of S]; o_done: P V of the step that had this buffer
  uint64_t q_full[2], q_empty[2], s_full[2][2], p_full[2][2], o_done[2][2];
  uint32_t tmem;
  int run_tiles[2];  // tiles of the run that a query tile belongs to
  int own_e, own_h, own_off, own_start, own_stop;
  long long scan[kThreads / 32];
  uint32_t q_at[kTile];  // where a query tile's rows start, in 16 bytes
};
static_assert(sizeof(Bars) <= kBarBytes, "barriers and scratch");

// Waits are bounded; the slow way is kept out of line, as the kernel's speed
// hangs on its code staying small (see attend_kernel).
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 255u) == 0 && globaltimer_ns() - t0 > kWaitLimitNs) {
      record_device_error(kDevErrWaitTimeout);
      return false;
    }
  }
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
  const uint32_t b = smem_u32(bar);
  return mbar_try_wait(b, parity) || mbar_try_wait(b, parity) || wait_long(b, parity);
}
// all lanes go on, or none: what follows is executed by whole warps
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(kFull, wait(bar, parity));
}

// ---- loads ----
template <int DP>
__device__ __forceinline__ void load_tiles(const Plan& p, const CUtensorMap* kmap,
                                           const CUtensorMap* vmap, char* smem, Bars* bars,
                                           const Part& part) {
  using S = Smem<DP>;
  const int lane = threadIdx.x & 31;
  const int pieces = kTile / p.box;  // boxes of a tile, per 64 columns; 16 at most
  const int piece = lane % pieces, half = lane / pieces;
  const int ps = (int)p.a.page_size;
  // own keys of narrow units are read once; everything else by several row tiles
  const uint64_t once = policy_evict_first(), more = policy_evict_normal();
  int stage = 0, filled = 0;
  uint32_t phase = 1;  // of the buffer's release: the first round waits for nothing
  bool ok = true;
#pragma unroll 1
  for (int ph = 0; ph < 2; ++ph) {
    Cursor cur;
    cur.start(p, part, ph == 0);
    const uint64_t policy = ph == 0 || p.own_wide ? more : once;
#pragma unroll 1
    for (; ok && cur.live(); cur.next_run(p)) {
      const int* own_table = p.a.page_table + (cur.pre ? 0 : cur.e / p.own_row_tiles) * p.a.table_row;
#pragma unroll 1
      for (int t = cur.first; ok && t < cur.first + cur.j1 - cur.j0; ++t) {
        const int used = (cur.keys(p, t) + p.box - 1) / p.box;
        const bool mine = piece < used && half < DP / 64;
        int page = 0, row = 0;
        if (mine) {
          const int key = cur.key0(p, t) + piece * p.box, at = key / ps;
          page = __ldg((cur.in_prefix(p, t) ? p.a.prefix_pages : own_table) + at);
          row = key - at * ps;
          if (page < 0 || page >= p.a.pages) {
            record_device_error(kDevErrBadIndex);
            page = (int)p.a.pages;  // past the tensor: the copy fills zeros, which count as keys
          }
        }
#pragma unroll 1
        for (int kv = 0; ok && kv < 2; ++kv) {
          ok = warp_wait(&bars->empty[stage], phase);
          if (ok) {
            if (lane == 0)
              mbar_arrive_expect_tx(&bars->full[stage], (uint32_t)used * p.box * 128u * (DP / 64));
            __syncwarp();
            if (mine)
              tma_load_4d(smem + S::kRing + stage * S::kTileBytes + half * (kTile * 128) + piece * p.box * 128,
                          kv ? vmap : kmap, &bars->full[stage], half * 64, row, cur.h, page, policy);
            if (filled < S::kStages) ++filled;
            if (++stage == S::kStages) stage = 0, phase ^= 1;
          }
        }
      }
    }
  }
  // every copy has landed before the CTA may end: the last round of fills
#pragma unroll 1
  for (int i = 0; i < filled; ++i) {
    if (--stage < 0) stage = S::kStages - 1, phase ^= 1;
    wait(&bars->full[stage], phase ^ 1);
  }
}

// ---- query rows: gathered into the MMA's swizzled layout ----
// 16 lanes copy a row's 16-byte chunks (fewer than 16 below head_dim 128), two
// rows a step; where the rows start is worked out once per run.
template <int DP>
__device__ __forceinline__ void load_queries(const Plan& p, char* smem, Bars* bars, const Part& part) {
  using S = Smem<DP>;
  const int lane = threadIdx.x & 31;
  const int c = lane & 15, r0 = lane >> 4;
  const bool on = c < (int)p.a.head_dim / 8;
  const char* q = static_cast<const char*>(p.a.q) + c * 16;
  const uint32_t to = smem_u32(smem) + S::kQ + (c >> 3) * (kTile * 128);
  int slot = 0;
#pragma unroll 1
  for (int ph = 0; ph < 2; ++ph) {
    Cursor cur;
    cur.start(p, part, ph == 0);
    const bool wide = ph == 0 ? p.pre_wide : p.own_wide;
#pragma unroll 1
    for (; cur.live(); cur.next_run(p)) {
      const int rows = unit_rows(p, cur.pre, cur.e);
#pragma unroll 1
      for (int s = 0; s < (wide ? 2 : 1); ++s, ++slot) {
        const int buf = slot & 1, count = min(kTile, rows - s * kTile);
        if (!warp_wait(&bars->q_empty[buf], ((slot >> 1) & 1) ^ 1)) return;
#pragma unroll 1
        for (int r = lane; r < count; r += 32) {
          const RowAt at = row_at(p, cur.pre, cur.e, cur.h, s * kTile + r);
          bars->q_at[r] = (uint32_t)((at.b * p.a.q_b + at.t * p.a.q_t + at.head * p.a.q_h) / 8);
        }
        __syncwarp();
        if (on)
#pragma unroll 4
          for (int r = r0; r < count; r += 2)
            cp_async16(to + buf * S::kTileBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                       q + 16ll * bars->q_at[r]);
        cp_async_wait_all();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          bars->run_tiles[buf] = cur.j1 - cur.j0;
          mbar_arrive(&bars->q_full[buf]);
        }
      }
    }
  }
}

// ---- MMAs ----
// A warp per stream; one elected lane issues. (The loop is the whole warp's, so
// that the compiler sees uniform values: with one lane in it every descriptor
// went through vector registers and an MMA took 80 cycles to issue instead of
// 35. One warp for both streams spent most of its time on waits and commits, one
// after the other: 4.8k cycles a wide tile against 2.6k of tensor work.)
// A stream's work is a line of steps of 64 keys: both halves of every tile in a
// wide unit, half s of every tile in a narrow one. Step n's S goes to buffer
// n & 1 of the stream, its P to the first columns of that buffer; P V of step n
// comes before S of step n + 2 in the tensor pipe, which executes in order, so
// nothing else guards the buffer. The next S is always under way while the
// softmax is busy with the one before.
// The warp does not know the units: the query warp publishes every run's length
// with its query tile.
struct MmaState {
  int k_stage = 0, v_stage = 1;  // ring buffers of the next K and V tile
  uint32_t k_phase = 0, v_phase = 0;
  int slot = 0;          // query tiles used up, by both streams
  uint32_t p_phase = 0;  // bit b: parity of the next P in buffer b
};

template <int DP, bool BF16>
__device__ __forceinline__ bool issue_mmas(uint32_t base, Bars* bars, uint32_t tmem, int s, int count,
                                           bool wide, MmaState& st) {
  using S = Smem<DP>;
  constexpr uint32_t kIdS = f16_idesc(BF16, kTile, kHalf, false);
  constexpr uint32_t kIdO = f16_idesc(BF16, kTile, DP, true);
  const uint64_t q_desc = sw128_desc(base + S::kQ, 16, 1024);
  const uint64_t k_desc = sw128_desc(base + S::kRing, 16, 1024);
  const uint64_t v_desc = sw128_desc(base + S::kRing, kTile * 128, 1024);
  const int steps = wide ? 2 * count : count;
  const uint32_t o_at = tmem + (2 + s) * kTile;
  int at = 0, run = 0;  // place in the run, its length, in steps, of the next S
  uint32_t fresh = 0;   // bit i: the i-th step between S and P V opens a run
#pragma unroll 1
  for (int n = 0; n < steps + 2; ++n) {
    // a wide unit's tile is done with its second half
    const bool tile_first = !wide || (n & 1) == 0, tile_last = !wide || (n & 1) == 1;
    const int half = wide ? n & 1 : s, buf = n & 1;
    const uint32_t s_at = tmem + s * kTile + buf * kHalf;
    if (n >= 2) {
      if (tile_first && !warp_wait(&bars->full[st.v_stage], st.v_phase)) return false;
      if (!warp_wait(&bars->p_full[s][buf], (st.p_phase >> buf) & 1)) return false;
      st.p_phase ^= 1u << buf;
      tc_fence_after();
      const uint64_t v = v_desc + (uint32_t)((st.v_stage * S::kTileBytes + half * kHalf * 128) >> 4);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kHalf / 16; ++k)
          mma_ts(o_at, s_at + k * 8, v + (uint32_t)(k * (2048 >> 4)), kIdO, k > 0 || !(fresh & 1u));
        tc_commit(&bars->o_done[s][buf]);
        if (tile_last) tc_commit(&bars->empty[st.v_stage]);
      }
      __syncwarp();
      fresh >>= 1;
      if (tile_last) {
        st.v_stage += 2;
        if (st.v_stage >= S::kStages) st.v_stage -= S::kStages, st.v_phase ^= 1;
      }
    }
    if (n < steps) {
      if (tile_first && !warp_wait(&bars->full[st.k_stage], st.k_phase)) return false;
      const int slot = st.slot + (wide ? s : 0), q = slot & 1;
      if (at == 0) {
        if (!warp_wait(&bars->q_full[q], (slot >> 1) & 1)) return false;
        run = __shfl_sync(kFull, bars->run_tiles[q], 0) * (wide ? 2 : 1);
        fresh |= 1u << (n < 2 ? n : 1);
      }
      const uint64_t a = q_desc + (uint32_t)(q * (S::kTileBytes >> 4));
      const uint64_t b = k_desc + (uint32_t)((st.k_stage * S::kTileBytes + half * kHalf * 128) >> 4);
      const bool run_last = at + 1 == run;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t off = ((k >> 2) * (kTile * 128) + (k & 3) * 32) >> 4;
          mma_ss(s_at, a + off, b + off, kIdS, k > 0);
        }
        tc_commit(&bars->s_full[s][buf]);
        if (tile_last) tc_commit(&bars->empty[st.k_stage]);
        if (run_last) {
          // a query tile is released by two: both streams, or one of them twice
          tc_commit(&bars->q_empty[q]);
          if (wide) tc_commit(&bars->q_empty[q]);
        }
      }
      __syncwarp();
      if (tile_last) {
        st.k_stage += 2;
        if (st.k_stage >= S::kStages) st.k_stage -= S::kStages, st.k_phase ^= 1;
      }
      if (++at == run) at = 0, st.slot += wide ? 2 : 1;
    }
  }
  return true;
}

// ---- softmax ----
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

// A row's maximum only moves when a tile exceeds it by more than 2^grow: every
// move costs a pass over O. Weights are then at most 2^grow, which bf16 and the
// fp32 sums hold with the same relative precision; fp16 weights are kept 2^6
// higher, may reach 2^(6 + 8) and lose bits only below 2^-20 of the highest.
template <typename T>
__device__ __forceinline__ constexpr float grow() {
  return std::is_same<T, __half>::value ? 8.f : 32.f;
}
template <typename T>
__device__ __forceinline__ constexpr float weight_shift() {
  return std::is_same<T, __half>::value ? 6.f : 0.f;
}

__device__ __forceinline__ void mask_columns(uint32_t* x, int upto) {
#pragma unroll
  for (int k = 0; k < 32; ++k)
    if (k >= upto) x[k] = 0xff800000u;  // -inf
}
__device__ __forceinline__ float row_max(const uint32_t* x) {
  float a[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = __uint_as_float(x[k]);
#pragma unroll
  for (int k = 4; k < 28; k += 8)
#pragma unroll
    for (int u = 0; u < 4; ++u)
      a[u] = fmaxf(fmaxf(a[u], __uint_as_float(x[k + u])), __uint_as_float(x[k + 4 + u]));
#pragma unroll
  for (int u = 0; u < 4; ++u) a[u] = fmaxf(a[u], __uint_as_float(x[28 + u]));
  return fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
}

// 32 weights 2^(c x + off) from x[0..31]: summed, then rounded to 16 bits into x[0..15].
// The rounding is the tensor cores' price: an MMA takes P and V in one type, and
// 32-bit weights would be two 16-bit parts and twice the MMAs of P V. It adds about
// as much as the output's own rounding: against 64 bits bf16 outputs are off by
// 1.9e-3 to 2.3e-3 of their size where 32-bit weights give 1.6e-3 to 1.7e-3, fp16
// by 2.8e-4 against 2.1e-4. The sums are of the unrounded weights, so lse keeps
// 32 bits.
template <typename T>
__device__ __forceinline__ void weights(uint32_t* x, float c, float off, float2& sum0, float2& sum1) {
  const float2 c2 = make_float2(c, c), off2 = make_float2(off, off);
#pragma unroll
  for (int k = 0; k < 32; k += 4) {
    float2 u = make_float2(__uint_as_float(x[k]), __uint_as_float(x[k + 1]));
    float2 w = make_float2(__uint_as_float(x[k + 2]), __uint_as_float(x[k + 3]));
    u = __ffma2_rn(u, c2, off2);
    w = __ffma2_rn(w, c2, off2);
    u = make_float2(ex2(u.x), ex2(u.y));
    w = make_float2(ex2(w.x), ex2(w.y));
    sum0 = __fadd2_rn(sum0, u);
    sum1 = __fadd2_rn(sum1, w);
    x[k / 2] = pack16<T>(u.x, u.y);
    x[k / 2 + 1] = pack16<T>(w.x, w.y);
  }
}

// Where a stream's partial result of a row stands.
__device__ __forceinline__ long long part_at(const Plan& p, const Cursor& cur, int s, int row) {
  const long long slot = 2 * slot_of(p, cur.pre, cur.e, cur.h, blockIdx.x, cur.first > 0) + s;
  return slot * (cur.pre ? p.pre_slot_rows : p.own_slot_rows) + row;
}
__device__ __forceinline__ float2& part_ml(const Plan& p, const Cursor& cur, int s, int row) {
  return reinterpret_cast<float2*>(cur.pre ? p.pre_ml : p.own_ml)[part_at(p, cur, s, row)];
}

// The end of a stream's run: O goes out, finished if no other run or stream has
// keys of these rows, else in fp32 with its maximum and sum.
template <typename T, int DP>
__device__ __forceinline__ void put_rows(const Plan& p, const Cursor& cur, int s, bool wide, int rows,
                                         uint32_t o_at, float m, float l) {
  const int row = min((int)threadIdx.x & 127, rows - 1);
  const bool mine = ((int)threadIdx.x & 127) < rows;
  const bool final = !cur.pre && !p.share && wide && cur.whole();
  const float inv = l > 0.f ? 1.f / l : 0.f;
  char* dst;
  if (final) {
    const RowAt at = row_at(p, false, cur.e, cur.h, (wide ? s * kTile : 0) + row);
    const long long out_row = (at.b * p.a.q_len + at.t) * p.a.q_heads + at.head;
    dst = static_cast<char*>(p.a.out) + out_row * p.a.head_dim * 2;
    if (mine && p.a.lse)
      p.a.lse[out_row] = l > 0.f ? (m * p.c - weight_shift<T>()) * 0.69314718055994531f + logf(l)
                                 : -INFINITY;
  } else {
    dst = reinterpret_cast<char*>((cur.pre ? p.pre_o : p.own_o) + part_at(p, cur, s, row) * DP);
    if (mine) part_ml(p, cur, s, row) = make_float2(m * p.c, l);
  }
#pragma unroll 1
  for (int col = 0; col < DP; col += 32) {
    uint32_t o[32];
    __syncwarp();  // the lanes part where they store; the TMEM load takes the whole warp
    tmem_ld32(o_at + col, o);
    tmem_wait_ld(o);
    if (mine && !final) {
#pragma unroll
      for (int k = 0; k < 32; k += 4)
        *reinterpret_cast<uint4*>(dst + (col + k) * 4) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
    } else if (mine) {
#pragma unroll
      for (int k = 0; k < 32; k += 8) {
        uint32_t w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float lo = __uint_as_float(o[k + 2 * u]) * inv, hi = __uint_as_float(o[k + 2 * u + 1]) * inv;
          w[u] = l > 0.f ? pack16<T>(lo, hi) : 0u;
        }
        if (col + k < (int)p.a.head_dim)
          *reinterpret_cast<uint4*>(dst + (col + k) * 2) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

template <typename T, int DP>
__device__ __forceinline__ void softmax_rows(const Plan& p, char* smem, Bars* bars, uint32_t tmem,
                                             int s, const Part& part) {
  using S = Smem<DP>;
  const int row = threadIdx.x & 127, warp = row >> 5;
  const uint32_t lanes = (uint32_t)warp << 21;  // TMEM lane in bits 16..31
  const uint32_t o_at = tmem + lanes + (2 + s) * kTile;
  const float c = p.c;
  int base_pos = 1;  // ring position of the phase's first V tile
  // bit b: parity of the next S in buffer b; P V of the step before this one has
  // the parity that its S had. (P V of the step before that is done: this step's
  // S came after it.)
  uint32_t phases = 0;
#pragma unroll 1
  for (int ph = 0; ph < 2; ++ph) {
    Cursor cur;
    cur.start(p, part, ph == 0);
    const bool wide = ph == 0 ? p.pre_wide : p.own_wide;
    uint32_t buf = 0;  // a phase begins with buffer 0
#pragma unroll 1
    for (; cur.live(); cur.next_run(p)) {
      const int rows = unit_rows(p, cur.pre, cur.e) - (wide ? s * kTile : 0);
      const bool active = warp * 32 < rows;
      int see = 0;  // own keys that this row sees
      if (!cur.pre)
        see = cur.len - (int)p.a.q_len + 1 +
              row_at(p, false, cur.e, cur.h, (wide ? s * kTile : 0) + max(0, min(row, rows - 1))).t;
      float m = -INFINITY, l = 0.f;
      const int steps = (cur.j1 - cur.j0) * (wide ? 2 : 1);
#pragma unroll 1
      for (int i = 0; i < steps; ++i, buf ^= 1) {
        const int half = wide ? i & 1 : s, j = cur.j0 + (wide ? i >> 1 : i);
        const int t = cur.first + j - cur.j0;
        const int keys = cur.keys(p, t);
        if (!warp_wait(&bars->s_full[s][buf], (phases >> buf) & 1)) return;
        phases ^= 1u << buf;
        tc_fence_after();
        if (keys < kTile && (!wide || half == 0)) {
          // What lies behind the last key in its page may be anything, and 0 * NaN
          // is NaN: clear V there, every warp before it gives its weights away.
          const int vpos = base_pos + 2 * j, stage = vpos % S::kStages;
          if (!warp_wait(&bars->full[stage], (vpos / S::kStages) & 1)) return;
          char* v = smem + S::kRing + stage * S::kTileBytes + keys * 128;
#pragma unroll 1
          for (int z = row; z < (kTile - keys) * 8; z += 128)
#pragma unroll
            for (int d = 0; d < DP / 64; ++d)
              *reinterpret_cast<uint4*>(v + d * (kTile * 128) + z * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
          __syncwarp();  // lanes cleared different numbers of chunks
        }
        if (active) {
          const uint32_t s_at = tmem + lanes + s * kTile + buf * kHalf;
          const int upto = (cur.in_prefix(p, t) ? keys : min(keys, see - cur.key0(p, t))) - kHalf * half;
          uint32_t x[kHalf];
          tmem_ld32(s_at, x);
          tmem_ld32(s_at + 32, x + 32);
          tmem_wait_ld(x);
          tmem_landed(x + 32);
          if (__any_sync(kFull, upto < kHalf)) mask_columns(x, upto), mask_columns(x + 32, upto - 32);
          const float top = fmaxf(row_max(x), row_max(x + 32));
          // The first maximum is taken as it is; later ones only past 2^grow.
          const bool moves = m == -INFINITY ? top > -INFINITY : top > m + grow<T>() / c;
          if (__any_sync(kFull, moves)) {
            const float keep = !moves ? 1.f : m == -INFINITY ? 0.f : ex2((m - top) * c);
            m = moves ? top : m;
            l *= keep;
            if (i > 0) {
              // O stands still once the last P V is done: the next needs this step's weights
              if (!warp_wait(&bars->o_done[s][buf ^ 1], (~phases >> (buf ^ 1)) & 1)) return;
              tc_fence_after();
#pragma unroll 1
              for (int col = 0; col < DP; col += 32) {
                uint32_t o[32];
                tmem_ld32(o_at + col, o);
                tmem_wait_ld(o);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                tmem_st32(o_at + col, o);
              }
            }
          }
          const float off = (m == -INFINITY ? 0.f : -m * c) + weight_shift<T>();
          float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
          weights<T>(x, c, off, sum0, sum1);
          tmem_st16(s_at, x);  // P takes the first half of its S
          weights<T>(x + 32, c, off, sum0, sum1);
          tmem_st16(s_at + 16, x + 32);
          l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&bars->p_full[s][buf]);
      }
      if (!warp_wait(&bars->o_done[s][buf ^ 1], (~phases >> (buf ^ 1)) & 1)) return;
      tc_fence_after();
      if (active) put_rows<T, DP>(p, cur, s, wide, rows, o_at, m, l);
      tc_fence_before();  // the next run's P V overwrites O after the next weights
    }
    base_pos += 2 * cur.end;
  }
}

// The kernel is latency all the way (a tile's S, softmax and P V follow one
// another, twelve warps run different code), and instructions that come from L2
// cost ten times those in the SM's cache: with both phases and every chunk
// unrolled the code was 190 KB and a tile took 3 to 7 times as long. So the
// phases share their code and the loops over chunks are real loops.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ Plan p, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  using S = Smem<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) char smem[];
  Bars* bars = reinterpret_cast<Bars*>(smem + S::kBars);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(kFull, tid >> 5, 0);
  pdl_trigger();
  if (smem_u32(smem) & 1023u) {  // the swizzle and the descriptors count on it
    if (tid == 0) record_device_error(kDevErrBadPlan);
    return;
  }

  // where this CTA's part of the line starts: a scan over the entries
  const int per = (p.entries + kThreads - 1) / kThreads;
  const int e_first = min(p.entries, tid * per), e_last = min(p.entries, e_first + per);
  long long mine = 0;  // places in the low half, tiles in the high half, both per head
#pragma unroll 1
  for (int e = e_first; e < e_last; ++e) {
    const int b = e / p.own_row_tiles;
    const int len = own_len(p, b);
    if (blockIdx.x == 0 && len != p.a.kv_lens[b]) record_device_error(kDevErrBadIndex);
    const int n = entry_tiles(p, entry_limit(p, e - b * p.own_row_tiles, len));
    mine += own_places(p, n) + ((long long)n << 32);
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(kFull, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) bars->scan[warp] = upto;
  if (tid == 0) {
#pragma unroll 1
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 2);
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->q_full[i], 1);
      mbar_init(&bars->q_empty[i], 2);
#pragma unroll 1
      for (int k = 0; k < 2; ++k) {
        mbar_init(&bars->s_full[i][k], 1);
        mbar_init(&bars->o_done[i][k], 1);
        mbar_init(&bars->p_full[i][k], 4);
      }
    }
    mbar_fence_init();
    tma_prefetch_map(&kmap);
    tma_prefetch_map(&vmap);
  }
  __syncthreads();
  long long sums = 0;
#pragma unroll 1
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) upto += bars->scan[w];
    sums += bars->scan[w];
  }
  const int heads = (int)p.a.kv_heads;
  const int total = (int)(sums & 0xffffffffll) * heads + p.pre_total;
  const Cut cut(total, p.grid);
  const int from = cut.first(blockIdx.x), to = cut.first(blockIdx.x + 1);
  auto pre_tiles_before = [&](int place) -> int {
    if (place <= 0 || p.pre_total == 0) return 0;
    const int len = p.pre_tiles * p.pre_cost + p.pre_extra;
    const int at = min(place, p.pre_total), unit = at / len;
    return unit * p.pre_tiles + max(0, at - unit * len - p.pre_extra + p.pre_cost - 1) / p.pre_cost;
  };
  Part part;
  part.pre_first = pre_tiles_before(from);
  part.pre_count = pre_tiles_before(to) - part.pre_first;
  // The own part's ends: the thread whose entries they fall into works them out.
  const int own_from = max(from, p.pre_total) - p.pre_total, own_to = to - p.pre_total;
  int before = (int)((upto - mine) & 0xffffffffll) * heads, tiles = (int)((upto - mine) >> 32) * heads;
#pragma unroll 1
  for (int e = e_first; e < e_last; ++e) {
    const int b = e / p.own_row_tiles;
    const int n = entry_tiles(p, entry_limit(p, e - b * p.own_row_tiles, own_len(p, b)));
    const int len = own_places(p, n);
    if (blockIdx.x == 0) p.starts[e] = before;
#pragma unroll 1
    for (int end = 0; end < 2; ++end) {
      const int rel = (end ? own_to : own_from) - before;
      if (rel < end || rel >= len * heads + end) continue;
      const int h = (rel - end) / len, off = max(0, rel - h * len - p.own_extra);
      if (end) {
        bars->own_stop = tiles + h * n + off;
      } else {
        bars->own_e = e, bars->own_h = h, bars->own_off = off;
        bars->own_start = tiles + h * n + off;
      }
    }
    before += len * heads;
    tiles += n * heads;
  }
  if (blockIdx.x == 0 && tid == kThreads - 1) p.starts[p.entries] = total - p.pre_total;
  __syncthreads();
  part.own_e = bars->own_e, part.own_h = bars->own_h, part.own_off = bars->own_off;
  part.own_count = __shfl_sync(kFull, own_to > own_from ? bars->own_stop - bars->own_start : 0, 0);
  part.pre_count = __shfl_sync(kFull, part.pre_count, 0);
  if (part.pre_count + part.own_count == 0) return;

  if (warp == 2) tmem_alloc(&bars->tmem, 512);
  if ((int)p.a.head_dim < DP)  // columns past head_dim stay zero: K's are filled with zeros
    for (int i = tid; i < 2 * S::kTileBytes / 16; i += kThreads)
      reinterpret_cast<uint4*>(smem + S::kQ)[i] = make_uint4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(kFull, bars->tmem, 0);

  if (warp == 0) {
    load_tiles<DP>(p, &kmap, &vmap, smem, bars, part);
  } else if (warp == 1) {
    load_queries<DP>(p, smem, bars, part);
  } else if (warp < 4) {
    MmaState st;
    bool ok = true;
#pragma unroll 1
    for (int ph = 0; ok && ph < 2; ++ph)
      ok = issue_mmas<DP, kBf16>(smem_u32(smem), bars, tmem, warp - 2,
                                 ph ? part.own_count : part.pre_count, ph ? p.own_wide : p.pre_wide, st);
  } else {
    softmax_rows<T, DP>(p, smem, bars, tmem, warp >= 8, part);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// joining the parts of a row
// ---------------------------------------------------------------------------
// The places of a unit's tiles.
struct Places {
  int start, stop;
};

constexpr int kJoinWarps = 8;

// A warp joins R rows. 32 / R lanes a row look at the runs that may hold a part
// of it (an online softmax over them); the whole warp then adds the parts up, a
// lane having four columns of each row, with 8 loads in flight. Units of many
// rows have few runs (R = 4), units of few rows many (R = 1).
template <typename T, int DP, int R>
__global__ void __launch_bounds__(32 * kJoinWarps, 4) join_kernel(const __grid_constant__ Plan p) {
  constexpr int kLanes = 32 / R, kAtOnce = 8 / R;
  const int lane = threadIdx.x & 31, sub = lane % kLanes;
  const int unit_max = p.own_wide ? min(p.rows, 2 * kTile) : p.rows;
  const int groups = (unit_max + R - 1) / R;
  const int heads = (int)p.a.kv_heads;
  const int group = blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
  const int unit = group / groups;
  const int e = unit / heads, h = unit - e * heads;
  if (e >= p.entries) return;
  const int rows = unit_rows(p, false, e), r = (group - unit * groups) * R + lane / kLanes;
  pdl_wait();
  const int own_at = p.starts[e], places = (p.starts[e + 1] - own_at) / heads;
  const Cut cut(p.starts[p.entries] + p.pre_total, p.grid);
  Places own, pre;
  own.stop = p.pre_total + own_at + (h + 1) * places;
  own.start = own.stop - places + (places ? p.own_extra : 0);
  const bool any = own.stop > own.start;
  const int c0 = any ? cut.cta_of(own.start) : 0, c1 = any ? cut.cta_of(own.stop - 1) : -1;
  if (!p.share && any && c0 == c1 && p.own_wide) return;  // already written
  const bool mine = r < rows;
  const RowAt at = row_at(p, false, e, h, mine ? r : 0);
  const long long out_row = (at.b * p.a.q_len + at.t) * p.a.q_heads + at.head;
  // candidates: (CTA, stream) of the prefix unit, then of the own unit
  int pu_e = 0, pu_r = 0, pc0 = 0, pc1 = -1;
  pre = own;
  if (p.share) {
    const int row = at.b * p.rows + (mine ? r : 0);
    pu_e = row / (2 * kTile), pu_r = row - pu_e * 2 * kTile;
    pre.stop = (h * p.pre_row_tiles + pu_e + 1) * (p.pre_tiles * p.pre_cost + p.pre_extra);
    pre.start = pre.stop - p.pre_tiles * p.pre_cost;
    // a tile is its first place's
    pc0 = cut.cta_of(pre.start), pc1 = cut.cta_of(pre.stop - p.pre_cost);
  }
  const int n_pre = 2 * (pc1 - pc0 + 1), n_all = mine ? n_pre + 2 * (c1 - c0 + 1) : 0;
  float m = -INFINITY, l = 0.f;
  float4 o[R];
#pragma unroll
  for (int k = 0; k < R; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int i = sub; __any_sync(kFull, i - sub < n_all); i += kLanes) {
    float cm = -INFINITY, cl = 0.f;
    const float* src = p.own_o;
    if (i < n_all) {
      const bool is_pre = i < n_pre;
      const int k = is_pre ? i : i - n_pre;
      const int cta = (is_pre ? pc0 : c0) + (k >> 1), s = k & 1;
      const int start = is_pre ? pre.start : own.start, stop = is_pre ? pre.stop : own.stop;
      const int from = max(start, cut.first(cta)) - start, to = min(stop, cut.first(cta + 1)) - start;
      // tiles whose first place lies in [from, to); a prefix tile has pre_cost (1 or 2) places
      const int up = is_pre ? p.pre_cost - 1 : 0;
      const bool wide = is_pre ? p.pre_wide : p.own_wide;
      const int ur = is_pre ? pu_r : r;
      if (((to + up) >> up) > ((from + up) >> up) && (!wide || (ur >> 7) == s)) {
        const long long slot = 2 * slot_of(p, is_pre, is_pre ? pu_e : e, h, cta, from > 0) + s;
        const long long at_row = slot * (is_pre ? p.pre_slot_rows : p.own_slot_rows) + (wide ? ur & 127 : ur);
        const float2 ml = reinterpret_cast<const float2*>(is_pre ? p.pre_ml : p.own_ml)[at_row];
        src = (is_pre ? p.pre_o : p.own_o) + at_row * DP;
        if (ml.y > 0.f) cm = ml.x, cl = ml.y;
      }
    }
    float top = fmaxf(m, cm);
#pragma unroll
    for (int x = 1; x < kLanes; x <<= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, x));
    const float keep = m == -INFINITY ? 0.f : ex2(m - top);
    const float w = cm == -INFINITY ? 0.f : ex2(cm - top);
    m = top;
    float add = w * cl;
#pragma unroll
    for (int x = 1; x < kLanes; x <<= 1) add += __shfl_xor_sync(kFull, add, x);
    l = l * keep + add;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const float f = __shfl_sync(kFull, keep, kLanes * k);
      o[k].x *= f, o[k].y *= f, o[k].z *= f, o[k].w *= f;
    }
    unsigned live = __ballot_sync(kFull, w > 0.f);
#pragma unroll
    for (int x = kLanes; x < 32; x <<= 1) live |= live >> x;  // candidates live in any row
    if (kLanes < 32) live &= (1u << (kLanes & 31)) - 1u;
#pragma unroll 1
    while (live) {
      float4 x[kAtOnce][R];
      float f[kAtOnce][R];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int j = live ? __ffs(live) - 1 : 0;
#pragma unroll
        for (int k = 0; k < R; ++k) {
          f[u][k] = __shfl_sync(kFull, w, kLanes * k + j);
          const float* ptr = reinterpret_cast<const float*>(
              __shfl_sync(kFull, reinterpret_cast<unsigned long long>(src), kLanes * k + j));
          if (!live) f[u][k] = 0.f;
          x[u][k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (f[u][k] > 0.f && lane * 4 < DP) x[u][k] = __ldcs(reinterpret_cast<const float4*>(ptr) + lane);
        }
        live &= live - 1;
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
        for (int k = 0; k < R; ++k) {
          o[k].x += f[u][k] * x[u][k].x, o[k].y += f[u][k] * x[u][k].y;
          o[k].z += f[u][k] * x[u][k].z, o[k].w += f[u][k] * x[u][k].w;
        }
    }
  }
  const float ln2 = 0.69314718055994531f;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (mine && sub == 0 && p.a.lse)
    p.a.lse[out_row] = l > 0.f ? (m - weight_shift<T>()) * ln2 + logf(l) : -INFINITY;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const float f = __shfl_sync(kFull, inv, kLanes * k);
    const long long row = __shfl_sync(kFull, out_row, kLanes * k);
    const bool put = __shfl_sync(kFull, (int)mine, kLanes * k);
    if (put && lane * 4 < (int)p.a.head_dim)
      *reinterpret_cast<uint2*>(static_cast<T*>(p.a.out) + row * p.a.head_dim + lane * 4) =
          make_uint2(pack16<T>(o[k].x * f, o[k].y * f), pack16<T>(o[k].z * f, o[k].w * f));
  }
}

// No page anywhere: every row is empty.
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
constexpr int64_t kMaxLine = int64_t(1) << 31;

int64_t align16(int64_t x) { return (x + 15) / 16 * 16; }

// Fills the plan, its pointers from `ws` on; returns the workspace's bytes, or -status.
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
  // measured: a wide tile takes about twice a narrow one's time, a run of a wide
  // unit costs about two of its tiles, one of a narrow unit about one
  p->pre_cost = p->pre_wide ? 2 : 1;
  p->pre_extra = p->pre_wide ? 4 : 1;
  p->own_extra = p->own_wide ? 2 : 1;
  const int64_t pre_line =
      p->share ? ((int64_t)p->pre_tiles * p->pre_cost + p->pre_extra) * p->pre_row_tiles * a.kv_heads : 0;
  const int64_t own_line =
      (p->lead_tiles + (a.table_width * a.page_size + kTile - 1) / kTile + p->own_extra) * a.kv_heads;
  // the kernels count places in 32 bits
  if (pre_line >= kMaxLine || own_line >= kMaxLine || own_line * p->entries >= kMaxLine - pre_line)
    return -SY_ERR_UNSUPPORTED;
  p->pre_total = (int)pre_line;
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
  p->starts = reinterpret_cast<int*>(take((p->entries + 1) * 4));
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
  cudaError_t e = launch_smem(attend_kernel<T, DP>, dim3(p.grid), kThreads, Smem<DP>::kBytes, st, p,
                              k, v);
  if (e != cudaSuccess) return e;
  const int unit_max = p.own_wide ? (p.rows < 2 * kTile ? p.rows : 2 * kTile) : p.rows;
  const int each = unit_max >= kTile ? 4 : 1;
  const int64_t warps = (int64_t)p.entries * p.a.kv_heads * ((unit_max + each - 1) / each);
  const dim3 grid((unsigned)((warps + kJoinWarps - 1) / kJoinWarps));
  return each == 4 ? launch_smem_pdl(join_kernel<T, DP, 4>, grid, 32 * kJoinWarps, 0, st, p)
                   : launch_smem_pdl(join_kernel<T, DP, 1>, grid, 32 * kJoinWarps, 0, st, p);
}

}  // namespace

int64_t attend_workspace(const sy_attend_args& a, const ServingDev& dev) {
  Plan p;
  return make_plan(a, dev.sms, &p, nullptr);
}

cudaError_t launch_attend(const sy_attend_args& a, const ServingDev& dev, cudaStream_t st) {
  if (a.pages == 0 || (a.table_width == 0 && a.prefix_len == 0)) {
    const int64_t n = a.batch * a.q_len * a.q_heads * (a.head_dim / 8);
    return launch_smem(no_keys_kernel, dim3((unsigned)((n + 255) / 256)), 256, 0, st, a);
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
