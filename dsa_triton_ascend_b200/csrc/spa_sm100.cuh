// Attention over the paged latent cache behind a shared prefix, on tcgen05: MLA-absorb, D = 512 (+64 rope), one KV head, any
// number of heads, any page size.
//
// Rows.  A row is a (token, head) pair; rows are flat in memory (token * n1 + head), so that 128 consecutive ones are one
// M = 128 tile whatever the number of heads.  A job is a row tile against a range of key positions:
//   - where it pays, a sequence of few rows (up to 64) that sees the whole prefix is PACKED: its rows meet the prefix together
//     with those of its neighbours, in tiles cut from the flat rows of the whole batch (prefix jobs), and its own keys in a
//     job of its own;
//   - every other sequence is cut into row tiles of its own, each over all the tile's visible keys.  Its tiles are full (or
//     nearly), so that packing would save nothing; that the prefix is the same pages for everybody then shows as L2 hits.
// A plan (a kernel, or with few jobs every CTA for itself) lists the jobs (the lengths live on the device) and cuts their key
// tiles, 128 keys each, into shares, one per CTA pair, along a line on which every job also takes what it costs besides its
// tiles: all pairs work for about the same time whatever the lengths are.  A job that lies in one pair's share and has no other part writes its result; the others leave
// normalised fp32 partials (maximum, sum, O), which spa_join_kernel adds up in a fixed order:
//   out = sum_i w_i O_i / sum_i w_i,   w_i = l_i exp(m_i - max m).
//
// Products.  A CTA pair works on a tile with tcgen05.mma.cta_group::2, M = 128 = 2 x 64 rows: S = Q K^T (N = 128 keys, B split
// along the keys: CTA c loads keys 64 c .. 64 c + 63 with all 576 features) and O += P V (two N = 256 products per 16 keys, B
// split along the value columns: CTA c loads all 128 keys x columns {c 128 .., 256 + c 128 ..}).  Q (72 KB a CTA), a tile of K
// and three quarters of one of V fill the shared memory; M = 256 would need 144 KB of Q, and O of 128 rows all of tensor memory.
// Tensor memory: lanes 0..63 hold a CTA's rows with the first half of N, lanes 64..127 the same rows with the second: O 256
// columns, S 2 buffers x 2 partial sums x 64.  (The tensor cores cut the running sum off: of normally distributed queries and
// keys a row's maximum is too small by 5e-7 of itself after 36 steps and its sum of exponentials too large by 2e-6; as two sums
// of 20 and 16 steps by half.)
//
// Data movement.  Pages are whole in the cache, so that keys come with tiled TMA, as many per box (64, 32, 16, 8) as divide the
// page size, else with gather4, four rows each.  Absent pages are read at a row past the tensor, which gives zeros without
// touching memory, and so are the values behind a sequence's end (gathered where they share a group of 8 with others):
// 0 x NaN would be NaN.  Keys behind the end only make scores that are masked.  Bytes are counted on the even CTA's barriers,
// where the products are issued.  Rings: K five units of 64 keys x 128 features (the fifth, the rope, 64), one tile, V three units
// of 32 keys x 256 columns, refilled unit by unit; P has two buffers.
//
// Softmax.  Eight warps take every tile together: the four threads of a row (two halves of N x two groups of 32 keys) exchange
// their maxima through shared memory.  P is relative to a running reference that follows the maximum only when that has risen
// by more than 2^8: then O is rescaled in tensor memory (P <= 2^8 in bf16, 2^15 in fp16; the sums are fp32).  P is rounded to
// the io dtype, the operand type of the second product; its sum is that of the unrounded values.
// Rows of one tile may see different numbers of keys (causal tokens of one sequence).  A hidden key has P = 0, and 0 x infinity
// would be NaN: a hidden key whose score is not finite (every non-finite latent makes it so, for every row) marks the
// token, and sfa_redo_kernel computes it again from its visible keys alone.  Normally no token.
//
// What bounds it: 2710 - 2780 cycles per tile of 128 keys, where the products at their full rate take 2176 (tensor pipe 83 %
// active, issue slots 44 %): 64 x 128 heads behind 16384 + 64 .. 2048 keys 229 us a call in short runs (1360 TFLOP/s, 0.80 of the
// measured burst rate), 271 under the power cap.  What brought it there, us for that call: one issuer and four loads per block
// 551; two issuers, wide loads, look-ups a tile ahead 274; two P buffers 246; one thread per loader 238; elected
// threads (elect.sync; a thread chosen by its number takes twice as long per product) 229.
//
// Warps (512 threads): 0 and 14 K loads, 1 and 15 V loads, 2 Q loads and tensor memory, 3 and 13 QK issuers, 4..11 softmax,
// 12 PV issuer.  All waits are bounded; one that gives up sets the status word.
#pragma once

#include <algorithm>
#include <atomic>
#include <mutex>

#include "ptx_sm100.cuh"
#include "sfa_fwd_mma.cuh"
#include "sfa_fwd_sm100.cuh"

namespace dsa {

constexpr int kSpaRows = 128;        // rows per tile (64 per CTA)
constexpr int kSpaKeys = 128;        // keys per tile
constexpr int kSpaThreads = 512;
constexpr int kSpaQkWarp0 = 3, kSpaSoftWarp0 = 4, kSpaPvWarp = 12, kSpaQkWarp1 = 13, kSpaKWarp1 = 14, kSpaVWarp1 = 15;
constexpr int kSpaPackRows = 64;     // a sequence with more rows has row tiles of its own (32 x 96 behind 8192 keys: 92 us packed, 83 not)
constexpr int kSpaPackKeys = 128;    // prefix that can save a tile
// Packing pays when the key tiles that it saves outweigh the partials and jobs that it makes.  us a call packed / not, with the
// tiles saved: 16 x 8 heads behind 512 keys 24.4 / 22.4 (60), 2048 25.5 / 26.3 (240); 64 x 8 behind 256 33.4 / 30.1 (120),
// 512 33.0 / 33.2 (240), 2048 34.6 / 50.8 (960); 64 x 16 behind 512 35.1 / 33.3 (224), 1024 34.6 / 39.2 (448); 64 x 32 behind 512
// 35.5 / 33.4 (192), 1024 36.5 / 39.4 (384); 64 x 64 behind 1024 42.4 / 40.4 (256), 2048 48.0 / 53.1 (512).
__host__ __device__ constexpr int64_t spa_pack_least(int64_t rows) { return 200 + rows / 32; }
constexpr int kSpaPlanThreads = 1024;   // 256 where there are no more places: its barriers are cheaper
// Places up to which every CTA of the main kernel plans for itself, which saves a launch: 8 x 8 heads 28.1 us of the host against 25.6,
// the GPU's side 20.4 / 20.7; one sequence of 60000 keys 39 / 36 on the GPU, 16 x 16 heads over 16000 keys 74.4 / 75.8, 64 x 16
// heads behind 16384 (72 places) 63.6 / 65.6.
constexpr int kSpaPlanEach = 64;
constexpr int kSpaClusters = 74;     // shares of the work (the workspace size must not depend on the device)
// What a job costs its pair besides its tiles (Q, the fill of the pipeline, the epilogue), in tiles.  64 x 64 heads behind 8192
// keys, us with 0 .. 6: 114, 102, 90, 83, 80, 81, 83; calls of one job per pair do not mind.
constexpr int kSpaJobTiles = 4;

constexpr uint32_t kSpaQBlk = 64 * 128;                     // 64 rows x 64 features
constexpr uint32_t kSpaQBytes = 9 * kSpaQBlk;
constexpr uint32_t kSpaBlk = 64 * 128;                      // 64 keys x 64 features
// Keys lie in groups of 8 (1024 bytes per 64 features, one swizzle atom), all of a group's blocks together, so that a box of any
// multiple of 8 keys is in one piece: K [8 groups][2 blocks][8 keys][128 bytes], V [4 groups][4 blocks of columns][8 keys]
// [128 bytes].  (Block after block, pages of 16 take a load per block and 16 keys: 105 -> 86 us for 33 x 2 x 64 heads;
// pages of 64 take the same time either way.)
constexpr uint32_t kSpaKUnit = 2 * kSpaBlk;                 // 64 keys x 128 features; the fifth unit, the rope, has 64
constexpr uint32_t kSpaVUnit = 4 * 32 * 128;                // 32 keys x 256 columns
constexpr uint32_t kSpaPBlk = 64 * 128;                     // 64 rows x 64 keys
constexpr uint32_t kSpaPBuf = 2 * kSpaPBlk;
constexpr uint32_t kSpaVUnits = 3;                          // units in the ring (a tile has four)
constexpr uint32_t kSpaOffQ = 0;
constexpr uint32_t kSpaOffK = kSpaOffQ + kSpaQBytes;
constexpr uint32_t kSpaOffV = kSpaOffK + 9 * kSpaBlk;
constexpr uint32_t kSpaOffP = kSpaOffV + kSpaVUnits * kSpaVUnit;
constexpr uint32_t kSpaOffX = kSpaOffP + 2 * kSpaPBuf;      // float [2][4][64]
constexpr uint32_t kSpaOffBar = kSpaOffX + 2048;
constexpr uint32_t kSpaSmemBytes = kSpaOffBar + 512;
static_assert(kSpaSmemBytes <= 232448, "shared memory");
constexpr uint32_t kSpaTmO = 0, kSpaTmS = 256;
constexpr float kSpaGuard = 8.f;     // log2 units that the maximum may rise by before the reference follows
// log2 units that the reference lies below the maximum that it was taken from, in fp16: P reaches from 2^15 at most down to the
// type's smallest numbers, 21 nats below the maximum (without it 17, and half a step's accuracy ends 10 nats below: 4000 keys
// 14 nats below a first one weighed 3 % too much or too little, and nothing 18 nats below).
constexpr float kSpaLiftFp16 = 7.f;

// One row tile against positions lo .. hi - 1, in tiles of 128 keys that start at key0.
struct SpaJob {
  int32_t row0, nrows;      // flat rows
  int32_t table_row;        // whose row of the block table the positions are looked up in
  int32_t key0, lo, hi;
  int32_t tile0, tiles;     // place of its first tile in the line of all jobs' work, and its tiles
  int32_t vis0;             // positions that the first row's token sees (mode 3: one more per token)
  int32_t head0;            // head of the first row
  int32_t packed;           // 1: rows of packed sequences against the prefix (those of other sequences are not read)
  int32_t slot;             // partial that the whole job leaves; -1: it writes its result
};
static_assert(sizeof(SpaJob) == 48, "three 16-byte loads");

struct SpaPlan {
  int32_t share;                // work per CTA pair, in tiles
  int32_t prefix;               // positions shared
};
// A CTA pair's share: the tiles at places at .. end - 1 of the line, from job `index` on.
struct SpaStart {
  int32_t at, end, index, unused;
  SpaJob j;
};
static_assert(sizeof(SpaStart) == 64, "four 16-byte loads");

struct SpaDev {
  SeqDesc seq;              // seq_k: keys with the prefix; paged
  const int32_t* prefix_device;
  int32_t prefix;
  int32_t rows, n1;         // tokens, heads
  int32_t prefix_tiles, own_tiles, own_tiles_per_seq;   // places in the list of row tiles (own_tiles_per_seq: BSND)
  int32_t pack_rows;        // kSpaPackRows, or 0 when nothing may be packed
  int32_t clusters;
  int32_t places_each;      // > 0: every CTA of the main kernel plans for itself, with room for so many jobs; 0: a plan kernel
  // workspace
  SpaPlan* plan;
  SpaJob* job;              // [prefix_tiles + own_tiles]
  int2* place;              // [prefix_tiles + own_tiles] job of a row tile (-1: none), and its sequence
  SpaStart* start;          // [clusters]
  int32_t* redo;            // [rows]
  int32_t* redo_list;       // [rows]
  int32_t* redo_count;
  int32_t* status;
  int32_t* fail;            // [2 clusters] CTAs that plan for themselves: what they have to say in place of the status
  float* part_o;            // [slots, 64 groups of 8 columns, 128, 8]: a warp's store of 8 columns is in one piece
  float* part_m;            // [slots, 128] maximum of the scaled scores, log2 units
  float* part_l;            // [slots, 128] sum relative to it; 0: the row sees nothing here
  // outputs
  void* out;
  float* softmax_max;
  float* softmax_sum;
  int32_t return_lse;
};

// What the plan and the kernels that follow it agree on about a sequence (b = batch: the rows behind the last one).
struct SpaSeq {
  int32_t start, act_q, act_k;   // first token, query tokens (within the tensor), keys (within the table)
  int32_t vis0;                  // positions that its first token sees (may be negative)
  bool packed;
};
// Few enough rows, and some (s.packed: and the whole prefix seen by all of them)
__device__ __forceinline__ bool spa_may_pack(const SpaDev& p, const SpaSeq& s) {
  return s.act_q > 0 && (int64_t)s.act_q * p.n1 <= p.pack_rows;
}
__device__ __forceinline__ SpaSeq spa_seq(const SpaDev& p, int32_t b, int32_t prefix) {
  SpaSeq s;
  int32_t act_q;
  if (b >= p.seq.batch) {            // the rows behind the last sequence (TND)
    s.start = min(max(p.seq.seq_q[p.seq.batch - 1], 0), p.rows);
    s.act_q = s.act_k = s.vis0 = 0;
    s.packed = false;
    return s;
  }
  if (p.seq.layout_q == DSA_LAYOUT_TND) {
    s.start = b > 0 ? p.seq.seq_q[b - 1] : 0;
    act_q = p.seq.seq_q[b] - s.start;
    s.start = min(max(s.start, 0), p.rows);
    s.act_q = max(0, min(act_q, p.rows - s.start));
  } else {
    s.start = b * p.seq.s1;
    act_q = p.seq.seq_q ? p.seq.seq_q[b] : p.seq.s1;
    s.act_q = max(0, min(act_q, p.seq.s1));
  }
  const int32_t act_k = p.seq.seq_k[b];
  s.act_k = max(0, min(act_k, p.seq.s2));
  // (the mask counts with the lengths as they were given)
  s.vis0 = p.seq.sparse_mode == 3 ? (int32_t)max((int64_t)-0x40000000, (int64_t)act_k - act_q + 1) : s.act_k;
  s.packed = prefix >= kSpaPackKeys && spa_may_pack(p, s) && s.act_k >= prefix && s.vis0 >= prefix;
  return s;
}
// First place of a sequence's row tiles in the list (behind the prefix tiles).
__device__ __forceinline__ int32_t spa_own_place(const SpaDev& p, int32_t b, int32_t start) {
  if (p.seq.layout_q != DSA_LAYOUT_TND) return b * p.own_tiles_per_seq;
  return (int32_t)((int64_t)start * p.n1 / kSpaRows) + b;
}

// ---- plan: one block -----------------------------------------------------------------------------------
struct SpaPlanSmem {
  unsigned long long best_s[32];
  int32_t sum_s[3][33];
  int32_t total_s[3];
  int32_t tiles_s[kSpaClusters], place_s[kSpaClusters];   // of the first jobs: tiles, and their place
};
// cluster < 0: a kernel of its own, which leaves every pair's start.  Otherwise for the pair `cluster` by each of its CTAs: its start
// in `start`, the jobs of its share in `own_jobs`; `publish`: one CTA leaves what the join reads.
__device__ __noinline__ void spa_plan(const SpaDev& p, SpaPlanSmem& sm, int32_t cluster, SpaStart* start, SpaJob* own_jobs,
                                      bool publish) {
  auto& best_s = sm.best_s;
  auto& sum_s = sm.sum_s;
  auto& total_s = sm.total_s;
  auto& tiles_s = sm.tiles_s;
  auto& place_s = sm.place_s;
  const int nt = blockDim.x, warps = nt >> 5;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Of the sequences that may be packed, the one whose first token sees most (the first of them) lends its pages for the prefix.
  // Others may have lengths and pages of before (a batch's idle slots, without query tokens), or see less than their length.
  int32_t prefix = 0, ref = 0;
  if (p.pack_rows > 0) {
    unsigned long long best = 0;
    for (int32_t b = tid; b < p.seq.batch; b += nt) {
      const SpaSeq s = spa_seq(p, b, 0);
      if (!spa_may_pack(p, s)) continue;
      const int32_t k = max(0, min(s.act_k, s.vis0));
      best = max(best, ((unsigned long long)(uint32_t)k << 32) | (uint32_t)(0x7FFFFFFF - b));
    }
    const int32_t asked = p.prefix_device ? *p.prefix_device : p.prefix;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) best_s[warp] = best;
    __syncthreads();
    best = lane < warps ? best_s[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    ref = 0x7FFFFFFF - (int32_t)(uint32_t)best;
    prefix = max(0, min(asked, (int32_t)(best >> 32)));
    // worth it?  (prefix = 0: nothing is packed)
    int32_t n = 0, r = 0;
    for (int32_t b = tid; b < p.seq.batch; b += nt) {
      const SpaSeq s = spa_seq(p, b, prefix);
      if (s.packed) { ++n; r += s.act_q * p.n1; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      n += __shfl_xor_sync(0xffffffffu, n, o);
      r += __shfl_xor_sync(0xffffffffu, r, o);
    }
    if (lane == 0) { sum_s[0][warp] = n; sum_s[1][warp] = r; }
    __syncthreads();
    n = lane < warps ? sum_s[0][lane] : 0;
    r = lane < warps ? sum_s[1][lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      n += __shfl_xor_sync(0xffffffffu, n, o);
      r += __shfl_xor_sync(0xffffffffu, r, o);
    }
    const int64_t saved = (int64_t)n * (prefix / kSpaKeys) -
                          (int64_t)((r + kSpaRows - 1) / kSpaRows) * ((prefix + kSpaKeys - 1) / kSpaKeys);
    if (saved < spa_pack_least(r)) prefix = 0;
    __syncthreads();                          // (sum_s is written again)
  }

  const int32_t places = p.prefix_tiles + p.own_tiles, rows = p.rows * p.n1;
  int32_t jobs = 0, tiles = 0, packed = 0;   // listed so far
  SpaJob j;
  int32_t mine = -1;                         // this thread's job of the last turn
  for (int32_t f0 = 0; f0 < places; f0 += nt) {
    const int32_t f = f0 + tid;
    mine = -1;
    j.tiles = 0;
    j.slot = -1;
    int32_t of_seq = 0;
    if (f < p.prefix_tiles) {
      j.row0 = f * kSpaRows;
      j.nrows = min(kSpaRows, rows - j.row0);
      // does any of its rows belong to a packed sequence?
      const int32_t t0 = j.row0 / p.n1, t1 = (j.row0 + j.nrows - 1) / p.n1;
      int32_t b = 0;
      bool any = false;
      if (prefix >= kSpaPackKeys) {
        const RowInfo ri = row_info(p.seq, t0);
        for (b = ri.b; b < p.seq.batch && !any; ++b) {
          const SpaSeq s = spa_seq(p, b, prefix);
          if (s.start > t1) break;
          any = s.packed && s.start + s.act_q > t0;
        }
      }
      j.table_row = ref;
      j.key0 = 0; j.lo = 0; j.hi = prefix;
      j.vis0 = prefix;
      j.head0 = j.row0 % p.n1;
      j.packed = 1;
      if (any) j.tiles = (prefix + kSpaKeys - 1) / kSpaKeys;
      j.slot = 0;
    } else if (f < places) {
      const int32_t g = f - p.prefix_tiles;
      int32_t b;
      if (p.seq.layout_q != DSA_LAYOUT_TND) b = g / p.own_tiles_per_seq;
      else {
        int32_t lo = 0, hi = p.seq.batch;      // the last sequence (or the rows behind them) whose first place is g or before
        while (lo < hi) {
          const int32_t mid = (lo + hi + 1) >> 1;
          if (spa_own_place(p, mid, min(max(p.seq.seq_q[mid - 1], 0), p.rows)) <= g) lo = mid; else hi = mid - 1;
        }
        b = lo;
      }
      of_seq = b;
      const SpaSeq s = spa_seq(p, b, prefix);
      const int32_t i = g - spa_own_place(p, b, s.start), n = s.act_q * p.n1;
      j.row0 = s.start * p.n1 + i * kSpaRows;
      j.nrows = min(kSpaRows, n - i * kSpaRows);
      if (i >= 0 && j.nrows > 0) {
        const int32_t first = i * kSpaRows / p.n1, last = (i * kSpaRows + j.nrows - 1) / p.n1;   // its tokens
        j.table_row = b;
        j.lo = s.packed ? prefix : 0;
        j.hi = p.seq.sparse_mode == 3 ? min(s.vis0 + last, s.act_k) : s.act_k;
        j.key0 = j.lo & ~(kSpaKeys - 1);
        j.vis0 = p.seq.sparse_mode == 3 ? s.vis0 + first : s.act_k;
        j.head0 = i * kSpaRows % p.n1;
        j.packed = 0;
        if (j.hi > j.lo) j.tiles = (j.hi - j.key0 + kSpaKeys - 1) / kSpaKeys;
        j.slot = s.packed ? 0 : -1;
      }
    }
    // running sums over the block: jobs, tiles, jobs that leave a partial
    const int32_t v[3] = {j.tiles > 0, j.tiles, j.tiles > 0 && j.slot == 0};
    int32_t x[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      x[k] = v[k];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t y = __shfl_up_sync(0xffffffffu, x[k], o);
        if (lane >= o) x[k] += y;
      }
      if (lane == 31) sum_s[k][warp] = x[k];
    }
    __syncthreads();
    if (warp < 3) {
      const int32_t in = lane < warps ? sum_s[warp][lane] : 0;
      int32_t z = in;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t y = __shfl_up_sync(0xffffffffu, z, o);
        if (lane >= o) z += y;
      }
      sum_s[warp][lane] = z - in;
      if (lane == 31) total_s[warp] = z;
    }
    __syncthreads();
    if (f < places) {
      const int32_t at = jobs + sum_s[0][warp] + x[0] - v[0];
      if (publish) p.place[f] = make_int2(v[0] ? at : -1, of_seq);
      if (v[0]) {
        j.tile0 = tiles + sum_s[1][warp] + x[1] - v[1] + kSpaJobTiles * (at + 1);
        if (v[2]) j.slot = 2 * p.clusters + packed + sum_s[2][warp] + x[2] - v[2];
        if (publish) p.job[at] = j;
        mine = at;
        if (at < kSpaClusters) tiles_s[at] = j.tiles;
      }
    }
    jobs += total_s[0]; tiles += total_s[1]; packed += total_s[2];
    __syncthreads();
  }
  // the line: a job's tiles lie behind kSpaJobTiles places for what it costs besides
  int32_t line = tiles + kSpaJobTiles * jobs;
  int32_t share = max(1, (line + p.clusters - 1) / p.clusters);
  // Few jobs: shares that end with their jobs save a pair its second job for tiles that its neighbours do not have.  Warp w tries
  // shares of w tiles more than the least; the first that needs no more than one share per pair, and is no longer than the
  // others would be, is taken: the places of the jobs' tiles are then rounded up to whole shares.
  bool single = false;
  if (jobs > 0 && jobs <= kSpaClusters) {
    const int32_t least = max(1, (tiles + p.clusters - 1) / p.clusters);
    const int32_t try_share = least + warp;
    int32_t parts = 0;
    for (int32_t i = lane; i < jobs; i += 32) parts += (tiles_s[i] + try_share - 1) / try_share;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) parts += __shfl_xor_sync(0xffffffffu, parts, o);
    if (lane == 0) sum_s[0][warp] = parts;
    __syncthreads();
    int32_t extra = 0;
    while (least + extra <= share && extra < warps && sum_s[0][extra] > p.clusters) ++extra;
    if (least + extra <= share && extra < warps) {
      single = true;
      share = least + extra;
      if (warp == 0) {
        int32_t before = 0;
        for (int32_t i0 = 0; i0 < jobs; i0 += 32) {
          const int32_t i = i0 + lane, mine_parts = i < jobs ? (tiles_s[i] + share - 1) / share : 0;
          int32_t z = mine_parts;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int32_t y = __shfl_up_sync(0xffffffffu, z, o);
            if (lane >= o) z += y;
          }
          if (i < jobs) place_s[i] = (before + z - mine_parts) * share;
          before += __shfl_sync(0xffffffffu, z, 31);
        }
        if (lane == 0) total_s[1] = before * share;
      }
      __syncthreads();
      line = total_s[1];
    }
  }
  if (tid == 0 && publish) {
    p.plan->share = share;
    p.plan->prefix = prefix;
  }
  if (cluster < 0) {
    for (int32_t c = tid; c < p.clusters; c += nt)
      if ((int64_t)c * share >= line) p.start[c].at = p.start[c].end = 0;
  } else if (tid == 0 && (int64_t)cluster * share >= line) {
    start->at = start->end = 0;
  }
  auto deal = [&](int32_t i) {               // job i = j: its place, and the pairs that begin in it
    if (single) {
      j.tile0 = place_s[i];
      if (publish) p.job[i].tile0 = j.tile0;
    }
    SpaStart w;
    w.j = j;
    w.index = i;
    w.unused = 0;
    const int32_t t0 = single ? j.tile0 : j.tile0 - kSpaJobTiles, t1 = j.tile0 + j.tiles;
    auto begin = [&](int32_t c, SpaStart& to) {
      w.at = max(c * share, j.tile0);
      w.end = min((c + 1) * share, single ? t1 : line);
      to = w;
    };
    if (cluster < 0) {
      for (int32_t c = (t0 + share - 1) / share; c < p.clusters && c * share < t1; ++c) begin(c, p.start[c]);
    } else {
      const int32_t at = cluster * share;
      if (at >= t0 && at < t1) begin(cluster, *start);
      if (t0 < at + share && t1 > at) own_jobs[i] = j;
    }
  };
  if (places <= nt) {                        // (the jobs are still at hand)
    if (mine >= 0) deal(mine);
  } else {
    for (int32_t i = tid; i < jobs; i += nt) {   // (a kernel of its own)
      j = p.job[i];
      deal(i);
    }
  }
}
__global__ void __launch_bounds__(kSpaPlanThreads) spa_plan_kernel(const __grid_constant__ SpaDev p) {
  __shared__ SpaPlanSmem sm;
  const int tid = threadIdx.x;
  grid_dep_launch();
  grid_dep_wait();
  if (tid < 64) p.status[tid] = 0;
  if (p.redo != nullptr) {
    if (tid == 0) *p.redo_count = 0;
    for (int32_t i = tid; i < p.rows; i += blockDim.x) p.redo[i] = 0;
  }
  spa_plan(p, sm, -1, nullptr, nullptr, true);
}

// Where the tiles a .. b - 1 of a job leave their result: -1 in the output, else a partial.  A pair's share has at most one
// job that began before it and one more that goes on after it.
__device__ __forceinline__ int32_t spa_slot(const SpaJob& j, int32_t a, int32_t b, int32_t cluster) {
  if (a == 0 && b == j.tiles) return j.slot;
  return 2 * cluster + (a > 0 ? 0 : 1);
}

__device__ __forceinline__ SpaJob spa_load_job(const SpaJob* p) {
  SpaJob j;
#pragma unroll
  for (int i = 0; i < 3; ++i) reinterpret_cast<int4*>(&j)[i] = reinterpret_cast<const int4*>(p)[i];
  return j;
}

// Walks over the tiles of a pair's share.
struct SpaWalk {
  const SpaJob* jobs;
  int32_t at, end, index;
  SpaJob j;
  __device__ __forceinline__ void start(const SpaJob* list, const SpaStart* from) {
    jobs = list;
    SpaStart w;
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<int4*>(&w)[i] = reinterpret_cast<const int4*>(from)[i];
    at = w.at; end = w.end; index = w.index;
    j = w.j;
  }
  __device__ __forceinline__ bool more() const { return at < end; }
  __device__ __forceinline__ int32_t tile() const { return at - j.tile0; }                       // of the job
  __device__ __forceinline__ int32_t stop() const { return min(j.tiles, end - j.tile0); }        // tile of the job to stop at
  __device__ __forceinline__ void next_tile() {
    if (++at < end && at >= j.tile0 + j.tiles) {
      j = spa_load_job(jobs + ++index);
      at = j.tile0;                      // (may lie past the end)
    }
  }
  __device__ __forceinline__ void next_job() {
    at = j.tile0 + stop();
    if (at < end) {
      j = spa_load_job(jobs + ++index);
      at = j.tile0;
    }
  }
};

struct SpaArgs {
  SpaDev p;
  uint32_t idesc_qk, idesc_pv;
  float scale_log2;
  int32_t is_bf16, key_rows, blocks;
  int32_t box_keys;                // 64, 32, 16 or 8 keys per box; 0: pages that are no multiple of 8 are gathered
  uint32_t page_mul, page_shift;   // position / page size = position * page_mul >> page_shift (positions below 2^31)
};

// Where a position of a job lies in the cache: the look-up first, so that it is in flight over the waits of the tile before, the
// row when it is needed.  A position that is not wanted, or whose block is absent, gets key_rows, a row past the tensor,
// which is loaded as zeros.
struct SpaSpot {
  int32_t blk, off;
  __device__ __forceinline__ void look_up(const SpaArgs& a, const SpaJob& j, int32_t pos, bool wanted) {
    const int32_t page = (int32_t)(((uint64_t)(uint32_t)pos * a.page_mul) >> a.page_shift);
    off = pos - page * a.p.seq.block_size;
    blk = wanted ? a.p.seq.block_table[(int64_t)j.table_row * a.p.seq.max_blocks + page] : -1;
  }
  __device__ __forceinline__ int32_t row(const SpaArgs& a) const {
    return blk >= 0 && blk < a.blocks ? blk * a.p.seq.block_size + off : a.key_rows;
  }
};
// A warp's loads: who it loads for, and where to.
struct SpaLoads {
  const CUtensorMap *box, *box8, *rope, *gather, *rope_gather;
  uint64_t *full, *empty;
  uint32_t full_lead;          // full[0] of the even CTA
  uint32_t dst;
  const SpaJob* jobs;
  const SpaStart* start;
  int32_t rank;
  int32_t u0;                  // first unit
  volatile int* abort_flag;
};

// K, pages that are multiples of 8: kBoxes boxes of 64 / kBoxes keys per unit, whole even where only some of their keys are wanted
// (what the others score is masked).  One thread: a load takes uniform operands, and a tile is a handful of them.
template <int kBoxes>
__device__ __forceinline__ void spa_k_boxes(const SpaArgs& a, const SpaLoads& o) {
  constexpr int kKeys = 64 / kBoxes;
  SpaWalk w;
  w.start(o.jobs, o.start);
  SpaSpot spot[kBoxes];
  auto look_up = [&]() {
    if (!w.more()) return;
    const int32_t pos = w.j.key0 + w.tile() * kSpaKeys + o.rank * 64;
#pragma unroll
    for (int b = 0; b < kBoxes; ++b) {
      const int32_t x = pos + b * kKeys;
      spot[b].look_up(a, w.j, x, x + kKeys > w.j.lo && x < w.j.hi);
    }
  };
  look_up();
  for (uint32_t n = 0; w.more(); ++n) {
    int32_t y[kBoxes];
#pragma unroll
    for (int b = 0; b < kBoxes; ++b) y[b] = spot[b].row(a);
    w.next_tile();
    look_up();
    auto unit = [&](int u) -> bool {
      if (!ptx::mbar_spin(&o.empty[u], (n & 1) ^ 1, o.abort_flag)) return false;
      if (o.rank == 0) ptx::mbar_arrive_expect_tx(&o.full[u], 2 * kSpaKUnit);
#pragma unroll
      for (int b = 0; b < kBoxes; ++b)
        ptx::tma_load_4d_pair(o.dst + u * kSpaKUnit + b * (kKeys / 8) * 2048, o.box, o.full_lead + u * 8, u * 128, 0, 0, (y[b] + 7) >> 3);
      return true;
    };
    if (!unit(o.u0) || !unit(o.u0 + 1)) return;
    if (o.u0 != 0) continue;
    if (!ptx::mbar_spin(&o.empty[4], (n & 1) ^ 1, o.abort_flag)) return;
    if (o.rank == 0) ptx::mbar_arrive_expect_tx(&o.full[4], kSpaKUnit);
#pragma unroll
    for (int b = 0; b < kBoxes; ++b)
      ptx::tma_load_2d_pair(o.dst + 4 * kSpaKUnit + b * (kKeys / 8) * 1024, o.rope, o.full_lead + 32, 0, y[b]);
  }
}

// V, pages that are multiples of 8: kBoxes boxes of 32 / kBoxes keys per unit.  What is not wanted has to be zero here: where a
// box would hold some of it, the unit is loaded in groups of 8, and a group that is cut itself is gathered.
template <int kBoxes>
__device__ __forceinline__ void spa_v_boxes(const SpaArgs& a, const SpaLoads& o) {
  constexpr int kKeys = 32 / kBoxes;
  SpaWalk w;
  w.start(o.jobs, o.start);
  SpaSpot spot[2][kBoxes];
  int32_t first = 0, lo = 0, hi = 0;          // position of the tile, and what is wanted
  auto look_up = [&]() {
    if (!w.more()) return;
    const int32_t pos = w.j.key0 + w.tile() * kSpaKeys;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int b = 0; b < kBoxes; ++b) {
        const int32_t x = pos + (o.u0 + 2 * i) * 32 + b * kKeys;
        spot[i][b].look_up(a, w.j, x, x + kKeys > w.j.lo && x < w.j.hi);
      }
  };
  look_up();
  for (uint32_t n = 0; w.more(); ++n) {
    int32_t y[2][kBoxes];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int b = 0; b < kBoxes; ++b) y[i][b] = spot[i][b].row(a);
    first = w.j.key0 + w.tile() * kSpaKeys; lo = w.j.lo; hi = w.j.hi;
    w.next_tile();
    look_up();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = n * 4 + o.u0 + 2 * i, use = v / kSpaVUnits, slot = v - use * kSpaVUnits;
      const int32_t pos = first + (o.u0 + 2 * i) * 32;
      if (!ptx::mbar_spin(&o.empty[slot], (use & 1) ^ 1, o.abort_flag)) return;
      if (o.rank == 0) ptx::mbar_arrive_expect_tx(&o.full[slot], 2 * kSpaVUnit);
      const uint32_t dst = o.dst + slot * kSpaVUnit, bar = o.full_lead + slot * 8;
      if (pos >= lo && pos + 32 <= hi) {
#pragma unroll
        for (int b = 0; b < kBoxes; ++b)
          ptx::tma_load_5d_pair(dst + b * (kKeys / 8) * 4096, o.box, bar, o.rank * 128, 0, 0, 0, (y[i][b] + 7) >> 3);
        continue;
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int32_t x = pos + g * 8, row = y[i][g * kBoxes / 4] == a.key_rows ? a.key_rows : y[i][g * kBoxes / 4] + (g * 8) % kKeys;
        if ((x >= lo && x + 8 <= hi) || x + 8 <= lo || x >= hi) {
          const int32_t yy = x >= lo && x < hi ? row : a.key_rows;
          ptx::tma_load_5d_pair(dst + g * 4096, o.box8, bar, o.rank * 128, 0, 0, 0, (yy + 7) >> 3);
          continue;
        }
#pragma unroll 1
        for (int q = 0; q < 2; ++q) {
          int32_t z[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int32_t k = q * 4 + e;
            z[e] = x + k >= lo && x + k < hi && row != a.key_rows ? row + k : a.key_rows;
          }
#pragma unroll 1
          for (int c = 0; c < 4; ++c)
            ptx::tma_gather4_2d_pair(dst + g * 4096 + c * 1024 + q * 512, o.gather, bar, (c >> 1) * 256 + o.rank * 128 + (c & 1) * 64,
                                     z[0], z[1], z[2], z[3]);
        }
      }
    }
  }
}

// Pages that are no multiple of 8: rows are gathered, four a load.  Lane i holds the positions 4 i .. 4 i + 3 of the CTA's 64 (K) or
// of the tile's 128 (V); one elected lane issues.
template <bool kV>
__device__ __forceinline__ void spa_gather(const SpaArgs& a, const SpaLoads& o) {
  const int lane = threadIdx.x & 31;
  SpaWalk w;
  w.start(o.jobs, o.start);
  SpaSpot spot[4];
  auto look_up = [&]() {
    if (!w.more()) return;
    const int32_t pos = w.j.key0 + w.tile() * kSpaKeys + (kV ? lane * 4 : o.rank * 64 + (lane & 15) * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) spot[i].look_up(a, w.j, pos + i, pos + i >= w.j.lo && pos + i < w.j.hi);
  };
  look_up();
  for (uint32_t n = 0; w.more(); ++n) {
    int32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = spot[i].row(a);
    w.next_tile();
    look_up();
    const int units = kV || o.u0 != 0 ? 2 : 3;
#pragma unroll 1
    for (int i = 0; i < units; ++i) {
      const int u = kV ? o.u0 + 2 * i : i == 2 ? 4 : o.u0 + i;
      const uint32_t use = kV ? (n * 4 + u) / kSpaVUnits : n, slot = kV ? n * 4 + u - use * kSpaVUnits : u;
      if (!ptx::mbar_spin_warp(&o.empty[slot], (use & 1) ^ 1, o.abort_flag)) return;
      if (o.rank == 0 && lane == 0)
        ptx::mbar_arrive_expect_tx(&o.full[slot], kV ? 2 * kSpaVUnit : u < 4 ? 2 * kSpaKUnit : kSpaKUnit);
      const uint32_t dst = o.dst + slot * (kV ? kSpaVUnit : kSpaKUnit), bar = o.full_lead + slot * 8;
#pragma unroll 4
      for (int q = 0; q < (kV ? 8 : 16); ++q) {
        const int l = kV ? u * 8 + q : q;
        const int32_t x0 = __shfl_sync(0xffffffffu, r[0], l), x1 = __shfl_sync(0xffffffffu, r[1], l),
                      x2 = __shfl_sync(0xffffffffu, r[2], l), x3 = __shfl_sync(0xffffffffu, r[3], l);
        if (ptx::elect_one()) {
          if (kV) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              ptx::tma_gather4_2d_pair(dst + (q >> 1) * 4096 + c * 1024 + (q & 1) * 512, o.gather, bar,
                                       (c >> 1) * 256 + o.rank * 128 + (c & 1) * 64, x0, x1, x2, x3);
          } else if (u < 4) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              ptx::tma_gather4_2d_pair(dst + (q >> 1) * 2048 + e * 1024 + (q & 1) * 512, o.gather, bar, u * 128 + e * 64, x0, x1, x2, x3);
          } else {
            ptx::tma_gather4_2d_pair(dst + q * 512, o.rope_gather, bar, 0, x0, x1, x2, x3);
          }
        }
        __syncwarp();
      }
      __syncwarp();
    }
  }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kSpaThreads, 1)
spa_fwd_sm100_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_qr,
                     const __grid_constant__ CUtensorMap tmap_kh, const __grid_constant__ CUtensorMap tmap_rh,
                     const __grid_constant__ CUtensorMap tmap_k1, const __grid_constant__ CUtensorMap tmap_r1,
                     const __grid_constant__ CUtensorMap tmap_vh, const __grid_constant__ CUtensorMap tmap_v8,
                     const __grid_constant__ SpaArgs a) {
  extern __shared__ __align__(1024) unsigned char spa_sm[];
  unsigned char* q_s = spa_sm + kSpaOffQ;
  unsigned char* k_s = spa_sm + kSpaOffK;
  unsigned char* v_s = spa_sm + kSpaOffV;
  unsigned char* p_s = spa_sm + kSpaOffP;
  float* xm = reinterpret_cast<float*>(spa_sm + kSpaOffX);      // [2 turns][4 threads of a row][64 rows]
  uint64_t* bars = reinterpret_cast<uint64_t*>(spa_sm + kSpaOffBar);
  uint64_t* k_full = bars;         // [5] even CTA: both CTAs' parts of the unit have landed (bytes)
  uint64_t* k_empty = bars + 5;    // [5] the products that read the unit are done (commit, both CTAs)
  uint64_t* v_full = bars + 10;    // [3] (ring)
  uint64_t* v_empty = bars + 13;   // [3]
  uint64_t* q_full = bars + 20;    // even CTA: both CTAs' rows have landed
  uint64_t* q_empty = bars + 21;   // the job's last score products are done (commit of both issuers, both CTAs)
  uint64_t* s_full = bars + 22;    // [2] scores of a tile are done (commit of both issuers, both CTAs)
  uint64_t* s_empty = bars + 24;   // [2] even CTA: the softmax warps of both CTAs hold them in registers
  uint64_t* p_full = bars + 16;    // [2] even CTA: P stored in both CTAs, O rescaled where it had to be
  uint64_t* p_empty = bars + 18;   // [2] the tile's value products are done (commit, both CTAs)
  uint64_t* o_free = bars + 26;    // even CTA: the softmax warps of both CTAs have read O
  uint64_t* x_bar = bars + 27;     // [2] xm written: the four warps that hold the same 32 rows
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 29);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 30);
  static_assert(31 * 8 <= 512, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const int32_t cluster = blockIdx.x >> 1;

  const bool misaligned = (ptx::smem_u32(spa_sm) & 1023u) != 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 5; ++i) { ptx::mbar_init(&k_full[i], 1); ptx::mbar_init(&k_empty[i], 1); }
    for (uint32_t i = 0; i < kSpaVUnits; ++i) { ptx::mbar_init(&v_full[i], 1); ptx::mbar_init(&v_empty[i], 1); }
    ptx::mbar_init(q_full, 1);
    ptx::mbar_init(q_empty, 2);
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&s_full[i], 2); ptx::mbar_init(&s_empty[i], 16); ptx::mbar_init(&x_bar[i], 4);
    }
    for (int i = 0; i < 2; ++i) { ptx::mbar_init(&p_full[i], 16); ptx::mbar_init(&p_empty[i], 1); }
    ptx::mbar_init(o_free, 16);
    *abort_flag = misaligned ? 1 : 0;
    ptx::mbar_fence_init();
  }
  if (warp == 2) {
    ptx::tmem_alloc_pair(tmem_slot, 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::cluster_arrive();     // the peer's barriers must exist before anything is sent to it
  ptx::cluster_wait();
  grid_dep_launch();
  grid_dep_wait();           // (nothing before this touches global memory)
  const uint32_t tmem = *tmem_slot;
  const SpaJob* jobs = a.p.job;
  const SpaStart* start = a.p.start + cluster;
  if (a.p.places_each > 0) {
    SpaStart* own_start = reinterpret_cast<SpaStart*>(spa_sm + kSpaOffBar + 256);
    SpaJob* own_jobs = a.p.job + (int64_t)a.p.places_each * (1 + blockIdx.x);
    static_assert(sizeof(SpaPlanSmem) <= 2048 && sizeof(SpaStart) <= 256, "in place of the maxima, and behind the barriers");
    spa_plan(a.p, *reinterpret_cast<SpaPlanSmem*>(spa_sm + kSpaOffX), cluster, own_start, own_jobs, blockIdx.x == 0);
    __syncthreads();
    jobs = own_jobs;
    start = own_start;
  }

  if (*abort_flag) {
    // nothing started
  } else if (warp == 0 || warp == kSpaKWarp1) {
    // ------------------------------------------------------------------ K loads
    // two warps: 0 has the units 0, 1 and the rope, 14 the units 2 and 3
    SpaLoads o;
    o.box = &tmap_kh; o.box8 = nullptr; o.rope = &tmap_rh; o.gather = &tmap_k1; o.rope_gather = &tmap_r1;
    o.full = k_full; o.empty = k_empty; o.full_lead = ptx::map_to_rank(&k_full[0], 0);
    o.dst = ptx::smem_u32(k_s); o.rank = (int32_t)rank; o.jobs = jobs; o.start = start; o.u0 = warp == 0 ? 0 : 2; o.abort_flag = abort_flag;
    if (a.box_keys == 0) spa_gather<false>(a, o);
    else if (ptx::elect_one()) {
      if (a.box_keys == 64) spa_k_boxes<1>(a, o);
      else if (a.box_keys == 32) spa_k_boxes<2>(a, o);
      else if (a.box_keys == 16) spa_k_boxes<4>(a, o);
      else spa_k_boxes<8>(a, o);
    }
  } else if (warp == 1 || warp == kSpaVWarp1) {
    // ------------------------------------------------------------------ V loads
    // two warps: 1 has the units 0 and 2, 15 the units 1 and 3
    SpaLoads o;
    o.box = &tmap_vh; o.box8 = &tmap_v8; o.rope = nullptr; o.gather = &tmap_k1; o.rope_gather = nullptr;
    o.full = v_full; o.empty = v_empty; o.full_lead = ptx::map_to_rank(&v_full[0], 0);
    o.dst = ptx::smem_u32(v_s); o.rank = (int32_t)rank; o.jobs = jobs; o.start = start; o.u0 = warp == 1 ? 0 : 1; o.abort_flag = abort_flag;
    if (a.box_keys == 0) spa_gather<true>(a, o);
    else if (ptx::elect_one()) {
      if (a.box_keys >= 32) spa_v_boxes<1>(a, o);
      else if (a.box_keys == 16) spa_v_boxes<2>(a, o);
      else spa_v_boxes<4>(a, o);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ Q loads
    if (lane == 0) {
      SpaWalk w;
      w.start(jobs, start);
      bool ok = true;
      const uint32_t bar = ptx::map_to_rank(q_full, 0);
      for (uint32_t n = 0; w.more() && ok; ++n, w.next_job()) {
        ok = ptx::mbar_wait(q_empty, (n & 1) ^ 1, abort_flag);
        if (!ok) break;
        if (rank == 0) ptx::mbar_arrive_expect_tx(q_full, 2 * kSpaQBytes);
#pragma unroll 1
        for (int f = 0; f < 9; ++f)
          ptx::tma_load_2d_pair(ptx::smem_u32(q_s) + f * kSpaQBlk, f < 8 ? &tmap_q : &tmap_qr, bar, f < 8 ? f * 64 : 0,
                                w.j.row0 + (int32_t)rank * 64);
      }
    }
  } else if (warp == kSpaQkWarp0 || warp == kSpaQkWarp1) {
    // ------------------------------------------------------------------ QK^T issuers
    // Two, each with its units and its partial score.  (One elected thread: chosen by its number in place of elect, it takes twice
    // as long per product; a warp-uniform loop 2 % of the whole.)
    if (rank == 0 && ptx::elect_one()) {
      const bool second = warp == kSpaQkWarp1;      // units 2 and 3; the first: 0, 1 and the rope
      const int units = second ? 2 : 3;
      SpaWalk w;
      w.start(jobs, start);
      bool ok = true;
      const uint64_t qd = ptx::desc_kmajor_sw128(ptx::smem_u32(q_s)), kd = ptx::desc_kmajor_sw128(ptx::smem_u32(k_s), 2048);
      const uint64_t rd = ptx::desc_kmajor_sw128(ptx::smem_u32(k_s));
      const uint32_t q_hi = (uint32_t)(qd >> 32);
      const uint32_t tm = tmem + kSpaTmS + (second ? 64 : 0);
      uint32_t n = 0;
      for (uint32_t n_job = 0; w.more() && ok; ++n_job, w.next_job()) {
        ok = ptx::mbar_spin(q_full, n_job & 1, abort_flag);
        const int32_t stop = w.stop();
        for (int32_t t = w.tile(); t < stop && ok; ++t, ++n) {
          const uint32_t b = n & 1;
          ok = ptx::mbar_spin_cluster(&s_empty[b], ((n >> 1) & 1) ^ 1, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after();
#pragma unroll 1
          for (int i = 0; i < units; ++i) {
            const int u = second ? 2 + i : (i == 2 ? 4 : i);
            ok = ptx::mbar_spin(&k_full[u], n & 1, abort_flag);
            if (!ok) break;
            const uint32_t ql = (uint32_t)qd + u * (2 * kSpaQBlk / 16), kl = (uint32_t)kd + u * (kSpaKUnit / 16);
            const uint32_t k_hi = (uint32_t)((u < 4 ? kd : rd) >> 32);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)   // (addresses in a descriptor count 16 bytes)
              if (kk < 4 || u < 4)
                ptx::mma_ss_pair_lo(tm + b * 128, ql + (kk >> 2) * (kSpaQBlk / 16) + (kk & 3) * 2, q_hi,
                                    kl + (kk >> 2) * (1024 / 16) + (kk & 3) * 2, k_hi, a.idesc_qk, (i > 0 || kk > 0) ? 1u : 0u);
            ptx::mma_commit_pair(&k_empty[u]);
            if (i == units - 1) ptx::mma_commit_pair(&s_full[b]);
          }
        }
        if (ok) ptx::mma_commit_pair(q_empty);
      }
    }
  } else if (warp == kSpaPvWarp) {
    // ------------------------------------------------------------------ PV issuer
    if (rank == 0 && ptx::elect_one()) {
      SpaWalk w;
      w.start(jobs, start);
      bool ok = true;
      const uint64_t pd = ptx::desc_kmajor_sw128(ptx::smem_u32(p_s)), vd = ptx::desc_mnmajor_sw128(ptx::smem_u32(v_s), 1024, 4096);
      const uint32_t p_hi = (uint32_t)(pd >> 32), v_hi = (uint32_t)(vd >> 32);
      uint32_t n = 0;
      for (uint32_t n_job = 0; w.more() && ok; ++n_job, w.next_job()) {
        ok = ptx::mbar_spin_cluster(o_free, (n_job & 1) ^ 1, abort_flag);
        const int32_t first = w.tile(), stop = w.stop();
        for (int32_t t = first; t < stop && ok; ++t, ++n) {
          ok = ptx::mbar_spin_cluster(&p_full[n & 1], (n >> 1) & 1, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after();
#pragma unroll 1
          for (int u = 0; u < 4; ++u) {
            const uint32_t v = n * 4 + u, use = v / kSpaVUnits, slot = v - use * kSpaVUnits;
            ok = ptx::mbar_spin(&v_full[slot], use & 1, abort_flag);
            if (!ok) break;
            const uint32_t pl = (uint32_t)pd + (n & 1) * (kSpaPBuf / 16) + (u >> 1) * (kSpaPBlk / 16) + (u & 1) * 4;
            const uint32_t vl = (uint32_t)vd + slot * (kSpaVUnit / 16);
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
              for (int c = 0; c < 2; ++c)
                ptx::mma_ss_pair_lo(tmem + kSpaTmO + c * 128, pl + kk * 2, p_hi, vl + c * (2048 / 16) + kk * (8192 / 16), v_hi,
                                    a.idesc_pv, (t > first || u > 0 || kk > 0) ? 1u : 0u);
            ptx::mma_commit_pair(&v_empty[slot]);
            if (u == 3) ptx::mma_commit_pair(&p_empty[n & 1]);
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue
    const int g = (warp - kSpaSoftWarp0) >> 2;    // takes keys 32 g .. 32 g + 31 of its half
    const int quarter = warp & 3;
    const int L = quarter * 32 + lane;            // tensor-memory lane
    const int hl = L & 63, half = L >> 6;         // row of this CTA; half of N
    const int trow = (int)rank * 64 + hl;         // row of the tile
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_empty_lead0 = ptx::map_to_rank(&s_empty[0], 0), s_empty_lead1 = ptx::map_to_rank(&s_empty[1], 0);
    const uint32_t p_full_lead = ptx::map_to_rank(&p_full[0], 0), o_free_lead = ptx::map_to_rank(o_free, 0);
    uint64_t* xb = &x_bar[quarter & 1];
    const float lift = a.is_bf16 ? 0.f : kSpaLiftFp16;
    uint32_t n = 0, n_x = 0;
    bool ok = true;
    auto signal_lead = [&](uint64_t* local, uint32_t remote, bool publish) {
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) ptx::mbar_arrive(local);
        else if (publish) ptx::mbar_arrive_remote_release(remote);
        else ptx::mbar_arrive_remote_relaxed(remote, 0u);
      }
    };
    // The values of the row's four threads (two buffers: a warp writes one of them again only after all four have arrived
    // for the other, which they do after reading this one).
    auto exchange = [&](float v, float4& all) -> bool {
      float* x = xm + (n_x & 1) * 256;
      x[(half * 2 + g) * 64 + hl] = v;
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(xb);
      const bool got = ptx::mbar_spin_warp(xb, n_x & 1, abort_flag);
      all = make_float4(x[hl], x[64 + hl], x[128 + hl], x[192 + hl]);
      ++n_x;
      return got;
    };
    SpaWalk w;
    w.start(jobs, start);
    for (; w.more() && ok; w.next_job()) {
      const SpaJob& j = w.j;
      const int32_t first = w.tile(), stop = w.stop();
      const int32_t slot = spa_slot(j, first, stop, cluster);
      // positions that this thread's row sees.  Rows that nobody reads (behind the tile's last one, and in a prefix job those of
      // sequences that are not packed) count as seeing all: masked, they would cost every tile the masks (a tile of 32
      // rows 20 % more time, and with it the whole call where its pair was the last).
      int32_t vis = j.hi;
      if (!j.packed && trow < j.nrows && a.p.seq.sparse_mode == 3) vis = min(j.vis0 + (j.head0 + trow) / a.p.n1, j.hi);
      float m_ref = -INFINITY, m_true = -INFINITY, l = 0.f;
      bool tainted = false;
      for (int32_t t = first; t < stop && ok; ++t, ++n) {
        const uint32_t b = n & 1;
        ok = ptx::mbar_spin_warp(&s_full[b], (n >> 1) & 1, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after();
        float sc[32];
        {
          float s1[32];
          ptx::tmem_ld_x32(lane_addr + kSpaTmS + b * 128 + g * 32, reinterpret_cast<uint32_t*>(sc));
          ptx::tmem_ld_x32(lane_addr + kSpaTmS + b * 128 + 64 + g * 32, reinterpret_cast<uint32_t*>(s1));
          ptx::tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) sc[k] += s1[k];
        }
        ptx::tc_fence_before();
        signal_lead(&s_empty[b], b ? s_empty_lead1 : s_empty_lead0, false);
        const int32_t k0 = j.key0 + t * kSpaKeys + half * 64 + g * 32;    // position of sc[0]
        if (__any_sync(0xffffffffu, k0 < j.lo || k0 + 32 > vis)) {
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const bool seen = k0 + k >= j.lo && k0 + k < vis;
            // (a hidden key that another row of the tile sees)
            if (!seen && k0 + k >= j.lo && k0 + k < j.hi && !(fabsf(sc[k]) < INFINITY)) tainted = true;
            sc[k] = seen ? sc[k] * a.scale_log2 : -INFINITY;
          }
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) sc[k] *= a.scale_log2;
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          mx4[0] = fmaxf(mx4[0], sc[k]); mx4[1] = fmaxf(mx4[1], sc[k + 1]);
          mx4[2] = fmaxf(mx4[2], sc[k + 2]); mx4[3] = fmaxf(mx4[3], sc[k + 3]);
        }
        float4 all;
        ok = exchange(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), all);
        if (!ok) break;
        const float mx = fmaxf(fmaxf(all.x, all.y), fmaxf(all.z, all.w));
        m_true = fmaxf(m_true, mx);
        // The reference follows the maximum where that has risen by more than the guard (or where the row had none yet: the
        // difference is infinite).  A difference of neighbours is exact; the reference plus the guard would be rounded, for
        // scores of millions by more than what fp16 has left above P.
        const bool raise = mx - m_ref > kSpaGuard + lift;
        if (__any_sync(0xffffffffu, raise)) {
          const float m_new = raise ? mx - lift : m_ref;
          const float f = raise ? (m_ref == -INFINITY ? 0.f : ex2(m_ref - m_new)) : 1.f;
          l *= f;
          m_ref = m_new;
          if (t > first) {
            ok = ptx::mbar_spin_warp(&p_empty[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag);     // O is complete up to the tile before
            if (!ok) break;
            ptx::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              const uint32_t at = lane_addr + kSpaTmO + g * 128 + c * 32;
              ptx::tmem_ld_x32(at, o);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              ptx::tmem_st_x32(at, o);
            }
            ptx::tmem_st_wait();
          }
        }
        const float ref = m_ref == -INFINITY ? 0.f : m_ref;       // (a row without a key yet: every sc is -inf, P = 0)
        float sum4[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pw[16];
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float e0 = ex2(sc[k] - ref), e1 = ex2(sc[k + 1] - ref), e2 = ex2(sc[k + 2] - ref), e3 = ex2(sc[k + 3] - ref);
          sum4[0] += e0; sum4[1] += e1; sum4[2] += e2; sum4[3] += e3;
          pw[k / 2] = pack2(e0, e1, a.is_bf16);
          pw[k / 2 + 1] = pack2(e2, e3, a.is_bf16);
        }
        l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
        // P once the value products of the tile before the last have read theirs
        ok = ptx::mbar_spin_warp(&p_empty[b], ((n >> 1) & 1) ^ 1, abort_flag);
        if (!ok) break;
        {
          unsigned char* prow = p_s + b * kSpaPBuf + half * kSpaPBlk + hl * 128;   // keys half * 64 .. are the first or second 64
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4*>(prow + (((g * 4 + c) ^ (hl & 7)) << 4)) =
                make_uint4(pw[4 * c], pw[4 * c + 1], pw[4 * c + 2], pw[4 * c + 3]);
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before();
        signal_lead(&p_full[b], p_full_lead + b * 8, true);
      }
      if (!ok) break;
      // ---- the row's sum, then O
      float4 ls;
      ok = exchange(l, ls);
      if (!ok) break;
      const float l_row = (ls.x + ls.y) + (ls.z + ls.w);
      if (tainted && a.p.redo != nullptr) {
        const int32_t tok = (j.row0 + trow) / a.p.n1;
        if (trow < j.nrows && !j.packed && atomicExch(&a.p.redo[tok], 1) == 0) a.p.redo_list[atomicAdd(a.p.redo_count, 1)] = tok;
      }
      ok = ptx::mbar_spin_warp(&p_empty[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag);
      if (!ok) break;
      ptx::tc_fence_after();
      // A row that sees no key here leaves nothing.  One whose scores here are all minus infinity has the sum 0: as a result it
      // is no number (0 / 0); as a partial it has the sum 1 beside its maximum, so that it weighs nothing beside others, and
      // O as it is (0 x infinity of a value is NaN in the value's column).  A sum that is not a number stays none.
      const bool any = max(j.lo, j.key0 + first * kSpaKeys) < vis;
      const bool low = slot >= 0 && l_row == 0.f;
      const float inv = any ? (low ? 1.f : 1.f / l_row) : 0.f;
      const float total = any ? (low ? 1.f : l_row * ex2(m_ref - m_true)) : 0.f;     // relative to the row's maximum
      const int32_t col0 = g * 256 + half * 128;     // this lane's columns
      if (slot >= 0) {
        float* o_row = a.p.part_o + ((int64_t)slot * 64 + col0 / 8) * (kSpaRows * 8) + trow * 8;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          ptx::tmem_ld_x32(lane_addr + kSpaTmO + g * 128 + c * 32, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
          if (any && trow < j.nrows) {       // (nobody reads the others: 8 x 8 heads 22.0 us with their stores, 20.4 without)
#pragma unroll
            for (int i = 0; i < 4; ++i) ptx::st_global_v8(o_row + (c * 4 + i) * (kSpaRows * 8), o + i * 8);
          }
        }
        if (g == 0 && half == 0 && trow < j.nrows) {
          a.p.part_m[(int64_t)slot * kSpaRows + trow] = m_true;
          a.p.part_l[(int64_t)slot * kSpaRows + trow] = total;
        }
      } else {
        unsigned char* o_row = (unsigned char*)a.p.out + (((int64_t)j.row0 + trow) * 512 + col0) * 2;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32], wd[16];
          ptx::tmem_ld_x32(lane_addr + kSpaTmO + g * 128 + c * 32, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            wd[i] = any ? pack2(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv, a.is_bf16) : 0u;
          if (trow < j.nrows) {
            ptx::st_global_v8(o_row + c * 64, wd);
            ptx::st_global_v8(o_row + c * 64 + 32, wd + 8);
          }
        }
        if (g == 0 && half == 0 && trow < j.nrows && a.p.softmax_max != nullptr) {
          const bool give = a.p.return_lse && any;
          // (a row whose sum is not a number has no maximum either)
          a.p.softmax_max[(int64_t)j.row0 + trow] = give ? (total == total ? m_true * 0.6931471805599453f : total) : 0.f;
          a.p.softmax_sum[(int64_t)j.row0 + trow] = give ? total : 0.f;
        }
      }
      ptx::tc_fence_before();
      signal_lead(o_free, o_free_lead, false);
    }
  }

  // ---------------------------------------------------------------------- teardown
  __syncwarp();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);  // let copies / products in flight land
  }
  ptx::tc_fence_before();
  __syncthreads();
  // neither CTA may leave while its peer can still signal it or run a pair product on its memory
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (warp == 2) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem, 512);
  }
  if (threadIdx.x == 0) {
    if (a.p.places_each > 0) a.p.fail[blockIdx.x] = *abort_flag;
    else if (*abort_flag) atomicExch(a.p.status, misaligned ? 2 : 1);
  }
}

// ---- join: the rows whose result is in parts, or that see nothing ----------------------------------
// A block works on a row tile: where the parts are is the same for all its rows (but for the prefix tile of a packed sequence,
// one of two), and a tile that its job has written itself is left at once.  A warp joins 16 columns of 32 rows, a row per
// lane (8 columns of 32 rows are 1 KB in one piece), with four parts' loads in flight; the warps of a block have the same rows
// and look the parts' maxima and sums up together, while the first O are on their way.
// kSplit, for few row tiles (whose rows may have a part from every pair): the eight warps have the same columns too and take
// every eighth part each; their sums meet in shared memory.  The whole call, in us, without and with it: one sequence of 60000
// keys 62 and 39 (128 heads: 4 groups of 32 rows); 4 such of 16000 keys 40 and 36 (16 groups); 6 and 8 of them 46 and 46, 51
// and 54 (24 and 32 groups); 8 heads behind a prefix of 8192 keys, 16 sequences 32 and 29, 20 of them 31 and 33 (20 groups).
constexpr int kSpaJoinThreads = 256;
constexpr int kSpaJoinWarps = kSpaJoinThreads / 32;
constexpr int kSpaJoinFew = 16;                                 // row groups of 32 up to which parts are split over warps
constexpr int kSpaJoinTasks = (kSpaRows / 32) * (512 / 16);     // of 32 rows x 16 columns in a row tile
struct SpaParts { int32_t first, count, uncut; };      // first share, number of shares, partial of a job in one share
__device__ __forceinline__ SpaParts spa_parts(const SpaDev& p, int32_t job, int32_t share) {
  SpaParts w = {0, 0, -1};
  if (job >= 0) {
    const int32_t t0 = p.job[job].tile0, n = p.job[job].tiles;
    w.uncut = p.job[job].slot;
    w.first = t0 / share;
    w.count = (t0 + n - 1) / share - w.first + 1;
  }
  return w;
}
template <bool kSplit>
__global__ void __launch_bounds__(kSpaJoinThreads, 2) spa_join_kernel(const SpaDev p, int32_t is_bf16) {
  __shared__ float2 ml_s[2 * kSpaClusters + 2][32];      // (maximum, sum) of part, row
  static_assert(sizeof(ml_s) >= kSpaJoinWarps * 17 * 32 * 4, "the warps' sums");
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31;
  if (p.places_each > 0 && blockIdx.x == 0 && blockIdx.y == 0) {     // (otherwise the plan kernel and the main one have seen to it)
    const int bad = __syncthreads_or(threadIdx.x < 2 * kSpaClusters && p.fail[threadIdx.x] != 0);
    if (threadIdx.x < 64) p.status[threadIdx.x] = threadIdx.x == 0 && bad ? 1 : 0;
  }
  const int32_t share = p.plan->share, prefix = p.plan->prefix;
  const int2 mine = p.place[p.prefix_tiles + blockIdx.x];
  const SpaSeq s = spa_seq(p, mine.y, prefix);
  const int32_t i = (int32_t)blockIdx.x - spa_own_place(p, mine.y, s.start);
  const int32_t tokens = p.seq.layout_q != DSA_LAYOUT_TND ? p.seq.s1 : (mine.y < p.seq.batch ? s.act_q : p.rows - s.start);
  if (i < 0) return;
  const int32_t row0 = s.start * p.n1 + i * kSpaRows;
  const int32_t total = min(kSpaRows, tokens * p.n1 - i * kSpaRows), active = min(total, s.act_q * p.n1 - i * kSpaRows);
  const SpaParts own = spa_parts(p, mine.x, share);
  const bool written = own.count == 1 && own.uncut < 0;      // the job wrote its rows itself
  if (total <= 0 || (written && total == active)) return;
  SpaParts pre[2] = {{0, 0, -1}, {0, 0, -1}};
  const int32_t pre0 = row0 / kSpaRows;
  if (s.packed) {
    pre[0] = spa_parts(p, p.place[pre0].x, share);
    if ((row0 + total - 1) / kSpaRows > pre0) pre[1] = spa_parts(p, p.place[pre0 + 1].x, share);
  }
  const int warp = threadIdx.x >> 5;
  for (int32_t y = blockIdx.y; y < kSpaJoinTasks / (kSplit ? 1 : kSpaJoinWarps); y += gridDim.y) {
    const int32_t task = kSplit ? y : y * kSpaJoinWarps + warp;
    const int32_t r = (task >> 5) * 32 + lane, cols = (task & 31) * 16;
    if ((task >> 5) * 32 >= total) break;
    constexpr int kStep = kSplit ? kSpaJoinWarps : 1;     // from a part of this warp to its next
    const int32_t part0 = kSplit ? warp : 0;
    const bool todo = r < total && !(written && r < active);
    const int32_t row = row0 + min(r, total - 1), prow = row % kSpaRows;
    const bool second = row / kSpaRows > pre0;
    const int32_t p_first = second ? pre[1].first : pre[0].first, p_uncut = second ? pre[1].uncut : pre[0].uncut;
    const int32_t p_count = todo && r < active ? (second ? pre[1].count : pre[0].count) : 0;
    const int32_t o_count = todo && r < active ? own.count : 0, parts = o_count + p_count;
    // row of the partials for part k: a job's first share leaves it in slot 2 c + 1, the later ones in 2 c
    auto at = [&](int32_t k, int32_t& tr) -> int64_t {
      const bool o = k < o_count;
      if (!o) k -= o_count;
      const int32_t m = o ? o_count : p_count, c0 = o ? own.first : p_first;
      tr = o ? r : prow;
      return m == 1 ? (o ? own.uncut : p_uncut) : 2 * (c0 + k) + (k == 0 ? 1 : 0);
    };
    float v[4][16];
    auto load = [&](int32_t k0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int32_t k = k0 + e * kStep;
        if (k >= parts) continue;
        int32_t tr;
        const int64_t slot = at(k, tr);
        const float* o = p.part_o + ((slot * 64 + cols / 8) * kSpaRows + tr) * 8;
        ptx::ld_global_v8(o, v[e]);
        ptx::ld_global_v8(o + kSpaRows * 8, v[e] + 8);
      }
    };
    load(part0);
    __syncthreads();               // (the turn before has read ml_s)
    for (int32_t k = warp; k < parts; k += kSpaJoinWarps) {
      int32_t tr;
      const int64_t i = at(k, tr) * kSpaRows + tr;
      ml_s[k][lane] = make_float2(p.part_m[i], p.part_l[i]);
    }
    __syncthreads();
    float mx = -INFINITY;
    for (int32_t k = 0; k < parts; ++k) {
      const float2 ml = ml_s[k][lane];
      if (ml.y != 0.f) mx = fmaxf(mx, ml.x);
    }
    float acc[16] = {}, den = 0.f;
    for (int32_t k0 = part0; k0 < parts; k0 += 4 * kStep) {
      if (k0 > part0) load(k0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (k0 + e * kStep >= parts) continue;
        const float2 ml = ml_s[k0 + e * kStep][lane];
        if (ml.y == 0.f) continue;           // (its O may never have been written)
        const float f = ml.y * ex2(ml.x - mx);
        den += f;
#pragma unroll
        for (int c = 0; c < 16; ++c) acc[c] += f * v[e][c];
      }
    }
    if (kSplit) {
      float* sum = reinterpret_cast<float*>(ml_s);        // [8 warps][17][32]
      __syncthreads();                                    // (everybody has read the weights)
#pragma unroll
      for (int c = 0; c < 16; ++c) sum[(warp * 17 + c) * 32 + lane] = acc[c];
      sum[(warp * 17 + 16) * 32 + lane] = den;
      __syncthreads();
      if (warp != 0) continue;
#pragma unroll 1
      for (int w = 1; w < kSpaJoinWarps; ++w) {
#pragma unroll
        for (int c = 0; c < 16; ++c) acc[c] += sum[(w * 17 + c) * 32 + lane];
        den += sum[(w * 17 + 16) * 32 + lane];
      }
    }
    if (!todo) continue;
    const bool any = den != 0.f;
    const float inv = any ? 1.f / den : 0.f;
    uint32_t out[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) out[c] = pack2(acc[2 * c] * inv, acc[2 * c + 1] * inv, is_bf16);
    ptx::st_global_v8((unsigned char*)p.out + (int64_t)row * 1024 + cols * 2, out);
    if (cols == 0 && p.softmax_max != nullptr) {
      const bool give = p.return_lse && any;
      p.softmax_max[row] = give ? (den == den ? mx * 0.6931471805599453f : den) : 0.f;
      p.softmax_sum[row] = give ? den : 0.f;
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------
struct SpaWs {
  size_t plan, job, place, start, fail, redo, redo_list, redo_count, part_m, part_l, part_o, total;
  int64_t prefix_tiles, own_tiles, own_tiles_per_seq, slots, places_each;
  bool pack, redo_used;
};
inline SpaWs spa_ws_layout(const DsaSpaParams* p, int64_t rows) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  auto tiles = [](int64_t r) { return (r + kSpaRows - 1) / kSpaRows; };
  SpaWs w;
  const bool tnd = p->layout_q == DSA_LAYOUT_TND;
  // packing needs a prefix and sequences of at most kSpaPackRows rows
  w.pack = (p->prefix_device != nullptr || p->prefix >= kSpaPackKeys) && p->n1 <= kSpaPackRows;
  w.prefix_tiles = w.pack ? tiles(rows * p->n1) : 0;
  w.own_tiles_per_seq = tnd ? 0 : std::max<int64_t>(1, tiles((int64_t)p->s1 * p->n1));
  w.own_tiles = tnd ? rows * p->n1 / kSpaRows + p->batch + 1 : p->batch * w.own_tiles_per_seq;
  // a packed sequence has one tile of its own and touches two prefix tiles at most
  w.slots = 2 * kSpaClusters + (w.pack ? std::min<int64_t>(w.own_tiles, p->batch) + std::min<int64_t>(w.prefix_tiles, 2ll * p->batch) : 0);
  // rows of a tile see different keys only when it holds several tokens of a sequence under the causal mask
  w.redo_used = p->sparse_mode == 3 && p->n1 % kSpaRows != 0 && (tnd || p->s1 > 1);
  const size_t places = (size_t)(w.prefix_tiles + w.own_tiles);
  w.plan = 0;
  w.job = 256;
  w.places_each = places <= kSpaPlanEach && !w.redo_used ? (int64_t)places : 0;
  w.place = w.job + up(places * sizeof(SpaJob) * (w.places_each > 0 ? 1 + 2 * kSpaClusters : 1));
  w.start = w.place + up(places * 8);
  w.fail = w.start + up(kSpaClusters * sizeof(SpaStart));
  w.redo_count = w.fail + up(2 * kSpaClusters * 4);
  w.redo = w.redo_count + 256;
  w.redo_list = w.redo + (w.redo_used ? up((size_t)rows * 4) : 0);
  w.part_m = w.redo_list + (w.redo_used ? up((size_t)rows * 4) : 0);
  w.part_l = w.part_m + up((size_t)w.slots * kSpaRows * 4);
  w.part_o = w.part_l + up((size_t)w.slots * kSpaRows * 4);
  w.total = w.part_o + (size_t)w.slots * kSpaRows * 512 * 4;
  return w;
}

inline bool spa_sm100_eligible(const DsaSpaParams* p, int64_t rows) {
  if (((uintptr_t)p->query & 15u) || ((uintptr_t)p->query_rope & 15u) || ((uintptr_t)p->out & 31u)) return false;
  if (p->key_rows >= 0x7FFFFFFF - 256 || rows < 1) return false;
  const SpaWs w = spa_ws_layout(p, rows);
  // tiles of all jobs are counted in 32 bits
  const int64_t key_tiles = ((int64_t)p->max_blocks * p->block_size + kSpaKeys - 1) / kSpaKeys + 1 + kSpaJobTiles;
  return (w.prefix_tiles + w.own_tiles) * key_tiles < (1ll << 30);
}

// The first call on a device raises the kernels' shared-memory limits there.  Safe to call from several host threads.
inline bool spa_sm100_prepare(int dev) {
  static std::atomic<int> ready[64];
  static std::mutex setup_lock;
  if (dev < 0 || dev >= 64) return false;
  if (ready[dev].load(std::memory_order_acquire)) return true;
  std::lock_guard<std::mutex> g(setup_lock);
  const int redo_smem = (kSfaSimtHeads + kSfaSimtKeys) * (512 + 64 + kSfaSimtPad) * 2;
  if (cudaFuncSetAttribute(spa_fwd_sm100_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSpaSmemBytes) != cudaSuccess ||
      cudaFuncSetAttribute(sfa_redo_kernel<__nv_bfloat16, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, redo_smem) != cudaSuccess ||
      cudaFuncSetAttribute(sfa_redo_kernel<__half, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, redo_smem) != cudaSuccess)
    return false;
  ready[dev].store(1, std::memory_order_release);
  return true;
}

// The latent cache [keys, 512] as [keys / 8][2 blocks][8 keys][features] (a box of 64 features from 128 u on, both blocks and n
// groups is n groups of K unit u), or as [keys / 8][2 halves][2 blocks][8 keys][columns] (64 columns from 128 c on, both
// blocks of both halves: n groups of a V unit of CTA c).
inline bool spa_tmap(CUtensorMap* m, const void* base, uint64_t keys, uint32_t box_keys, bool v, bool bf16) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t groups = std::max<uint64_t>(keys / 8, 1);
  const cuuint64_t k_dims[4] = {512, 8, 2, groups}, k_strides[3] = {1024, 128, 8192};
  const cuuint64_t v_dims[5] = {512, 8, 2, 2, groups}, v_strides[4] = {1024, 128, 512, 8192};
  const cuuint32_t k_box[4] = {64, 8, 2, box_keys / 8}, v_box[5] = {64, 8, 2, 2, box_keys / 8}, estr[5] = {1, 1, 1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, v ? 5 : 4, const_cast<void*>(base),
             v ? v_dims : k_dims, v ? v_strides : k_strides, v ? v_box : k_box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// `dense`: the call for the row-by-row kernel.
inline int spa_sm100_launch(const DsaSpaParams* p, const SfaDev& dense, int32_t* status, void* scratch, cudaStream_t st) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return DSA_ERR_CUDA;
  if (!spa_sm100_prepare(dev)) return DSA_ERR_CUDA;
  const bool bf16 = p->dtype == DSA_DTYPE_BF16;
  const SpaWs w = spa_ws_layout(p, dense.rows);
  char* ws = (char*)scratch;
  SpaArgs a;
  SpaDev& d = a.p;
  d.seq = dense.seq;
  d.prefix_device = p->prefix_device; d.prefix = p->prefix;
  d.rows = dense.rows; d.n1 = p->n1;
  d.prefix_tiles = (int32_t)w.prefix_tiles; d.own_tiles = (int32_t)w.own_tiles; d.own_tiles_per_seq = (int32_t)w.own_tiles_per_seq;
  d.pack_rows = w.pack ? kSpaPackRows : 0;
  d.clusters = kSpaClusters;
  d.places_each = (int32_t)w.places_each;
  d.plan = (SpaPlan*)(ws + w.plan); d.job = (SpaJob*)(ws + w.job); d.place = (int2*)(ws + w.place);
  d.start = (SpaStart*)(ws + w.start); d.fail = (int32_t*)(ws + w.fail);
  d.redo = w.redo_used ? (int32_t*)(ws + w.redo) : nullptr;
  d.redo_list = (int32_t*)(ws + w.redo_list); d.redo_count = (int32_t*)(ws + w.redo_count);
  d.status = status;
  d.part_o = (float*)(ws + w.part_o); d.part_m = (float*)(ws + w.part_m); d.part_l = (float*)(ws + w.part_l);
  d.out = p->out; d.softmax_max = p->softmax_max; d.softmax_sum = p->softmax_sum; d.return_lse = p->return_lse != 0;
  a.idesc_qk = ptx::idesc_f16(bf16 ? 1u : 0u, 128, kSpaKeys, 0, 0);
  a.idesc_pv = ptx::idesc_f16(bf16 ? 1u : 0u, 128, 256, 0, 1);
  a.scale_log2 = (float)((double)p->scale * 1.4426950408889634);
  a.is_bf16 = bf16 ? 1 : 0;
  a.key_rows = (int32_t)p->key_rows;
  a.blocks = (int32_t)(p->key_rows / p->block_size);
  // mul = ceil(2^(31 + l) / size) with 2^l >= size: the error is below 2^31 size / 2^(31 + l) <= 1 step of the quotient
  uint32_t l = 0;
  while ((1ll << l) < p->block_size) ++l;
  a.page_shift = 31 + l;
  a.page_mul = (uint32_t)(((1ull << (31 + l)) + p->block_size - 1) / (uint64_t)p->block_size);
  const uint64_t rows = (uint64_t)dense.rows * p->n1, keys = (uint64_t)p->key_rows;
  a.box_keys = 64;
  while (a.box_keys >= 8 && p->block_size % a.box_keys != 0) a.box_keys /= 2;
  if (a.box_keys < 8) a.box_keys = 0;
  const uint32_t box_keys = std::max(a.box_keys, 8);
  CUtensorMap q, qr, kh, rh, k1, r1, vh, v8;
  if (!make_tmap_2d_16bit(&q, p->query, rows, 512, 1024, 64, 64, bf16) ||
      !make_tmap_2d_16bit(&qr, p->query_rope, rows, 64, 128, 64, 64, bf16) ||
      !spa_tmap(&kh, p->key, keys, box_keys, false, bf16) ||
      !make_tmap_2d_16bit(&rh, p->key_rope, keys, 64, 128, box_keys, 64, bf16) ||
      !make_tmap_gather4_16bit(&k1, p->key, keys, 512, 1024, 64, bf16) ||
      !make_tmap_gather4_16bit(&r1, p->key_rope, keys, 64, 128, 64, bf16) ||
      !spa_tmap(&vh, p->key, keys, std::min(box_keys, 32u), true, bf16) || !spa_tmap(&v8, p->key, keys, 8, true, bf16))
    return DSA_ERR_CUDA;
  // (barriers of 8 warps are cheaper than those of 32)
  const int plan_threads = w.prefix_tiles + w.own_tiles <= 256 ? 256 : kSpaPlanThreads;
  if (w.places_each == 0 && launch_after(spa_plan_kernel, dim3(1), dim3(plan_threads), 0, st, d) != cudaSuccess) return DSA_ERR_CUDA;
  if (launch_after(spa_fwd_sm100_kernel, dim3(2 * kSpaClusters), dim3(kSpaThreads), kSpaSmemBytes, st, q, qr, kh, rh, k1, r1,
                   vh, v8, a) !=
      cudaSuccess)
    return DSA_ERR_CUDA;
  // a task per warp, more where there are so many tiles that most are written by their jobs
  const int64_t seq_rows = w.own_tiles_per_seq > 0 ? (int64_t)p->s1 * p->n1 : (int64_t)rows;
  const int64_t tile_rows = std::min<int64_t>(kSpaRows, seq_rows);
  const int64_t groups = (tile_rows + 31) / 32;              // of 32 rows in a tile, at most
  const bool few = w.own_tiles * groups <= kSpaJoinFew;
  const dim3 join_grid((unsigned)w.own_tiles,
                       few ? (unsigned)groups * (512 / 16) : w.own_tiles <= 512 ? kSpaJoinTasks / kSpaJoinWarps : 1);
  if ((few ? launch_after(spa_join_kernel<true>, dim3(join_grid), dim3(kSpaJoinThreads), 0, st, d, a.is_bf16)
           : launch_after(spa_join_kernel<false>, dim3(join_grid), dim3(kSpaJoinThreads), 0, st, d, a.is_bf16)) != cudaSuccess)
    return DSA_ERR_CUDA;
  count_launch(w.places_each > 0 ? 2 : 3);
  if (w.redo_used) {
    const size_t smem = (size_t)(kSfaSimtHeads + kSfaSimtKeys) * (p->d + p->d_rope + kSfaSimtPad) * 2;
    const int64_t work = (int64_t)d.rows * ((p->n1 + kSfaSimtHeads - 1) / kSfaSimtHeads);
    const dim3 grid((unsigned)std::min<int64_t>(work, 296));
    const cudaError_t rc = bf16 ? launch_after(sfa_redo_kernel<__nv_bfloat16, true>, dim3(grid), dim3(kSfaSimtThreads), smem, st,
                                               dense, d.redo_list, d.redo_count)
                                : launch_after(sfa_redo_kernel<__half, true>, dim3(grid), dim3(kSfaSimtThreads), smem, st, dense,
                                               d.redo_list, d.redo_count);
    if (rc != cudaSuccess) return DSA_ERR_CUDA;
    count_launch();
  }
  return DSA_OK;
}

}  // namespace dsa
