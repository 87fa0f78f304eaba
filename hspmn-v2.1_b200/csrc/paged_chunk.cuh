// Sparse-query dense-key causal attention over a paged K/V cache, for requests
// with many query rows (prompt chunks, whole or router-selected): the products
// of sqdk_fwd_kernel on tcgen05 / TMEM / TMA with the keys fetched page by page.
//
// Tile: one request, one K/V head, QT = 128 / G consecutive query rows of the
// packed batch with the G heads that read that K/V head (128 rows), against
// 64-key blocks. S = Q K^T and O += P V as in sqdk.cuh (two S buffers, P over
// S in tensor memory, optimistic running maximum, O in tensor memory for the
// whole tile); K and V blocks land through TMA boxes of min(page_size, 64)
// rows, one box a page, found through the block table by the producer warp.
//
// Schedule: requests have any lengths, the host knows none of them, and a tile
// costs from one block to thousands. The tiles form one list (request, head,
// tile) with an estimated cost each, linear in the tile's number between the
// request's first and last position; the list is cut into equal runs, one a
// CTA (two CTAs an SM). A CTA takes the tiles that lie in its run whole, in
// order, then the pieces that its run's two ends cut off: their O goes to the
// workspace and a merge kernel adds the pieces in run order. Whole tiles first,
// because the tiles of a head then start together at its first key and stream
// the same K/V blocks out of L2. Estimates only set the balance: which keys a
// piece covers is computed from the cut and the tile's true key count, the same
// way by every CTA that holds a piece.
//
// Warp roles (192 threads): warp 0 requests Q, K and V (one lane a page box),
// warp 1 allocates tensor memory and issues the products, warps 2..5 do the
// softmax and the epilogue (one thread a row). The K, V and S rings run on
// across tiles, so the next tile's keys load while this one ends.
//
// Bound: the chain of softmax and products of an SM's two CTAs (a block takes a
// CTA about 1,700 cycles; tensor pipe and exponentials 43 % busy each), at the
// card's 1 kW. Calls in a row for seconds: a fifth of 8192 new tokens over 24576
// cached, three requests of 16/4 heads of 128, 1.24 to 1.30 ms, 890 to 927 TFLOP/s
// (SM at 1.40 GHz); seven whole prompts of 511 to 4096 tokens 279 to 286 us, 754 to
// 774 TFLOP/s (1.70 GHz; tiles of 23 blocks on average, each 5 blocks' time to open
// and close). The prompts in bursts of 20 ms, before the power limit lowers the
// clock: 245 to 247 us; there, eight softmax warps took 258 (against 249 then) and
// 128-key blocks with one S buffer 283.
#pragma once

#include "paged_attn.cuh"

namespace hspmn {

constexpr int kChunkThreads = 192;
constexpr int kChunkCtasPerSm = 2;
constexpr int kChunkUnit = 16;           // cost units of a 64-key block
constexpr int kChunkTileCost = 5;        // blocks' worth of time to open and close a tile (seven prompts in bursts of 20 ms: 247 us; at 3 256, 6 250, 7 252, 9 262)
constexpr int kChunkMinPiece = 8;        // blocks of work below which another run is not opened
constexpr int kChunkEpilogueBar = 1;     // named barrier of the four softmax warps
constexpr int kChunkTilt = 3;            // see ChunkRuns, in 64ths
constexpr float kChunkFmaMax = 512.0f;   // largest maximum (log2 units) of which the rounding may be left in P

template <int HD>
struct ChunkLayout {
  static constexpr int kChunks = HD / 64;
  static constexpr int kQChunkBytes = kSqdkBM * 128;
  static constexpr int kKVChunkBytes = kSqdkBN * 128;
  static constexpr int kKVBytes = kChunks * kKVChunkBytes;
  static constexpr int kQOff = 0;
  static constexpr int kKOff = kChunks * kQChunkBytes;
  static constexpr int kVOff = kKOff + 2 * kKVBytes;
  static constexpr int kOOff = kVOff + 2 * kKVBytes;  // epilogue staging: 32 rows x 64 bytes a warp
  static constexpr int kBytes = kOOff + 4 * 32 * 64;
  static constexpr int kAlloc = kBytes + 1024;
  static constexpr uint32_t kTmemCols = 256;  // S0 | S1 | O
  static constexpr int kOCol = 2 * kSqdkBN;
};

struct ChunkParams {
  PagedAttnParams a;  // part_o / part_ml: [2 * runs][128] rows here
  int QT, box_rows;
};

// One piece of work as the producer posts it to the other warps.
struct ChunkJob {
  int row0, queries;  // first query row of q, queries of the tile
  int r, head, kv;
  int lo, hi;      // smallest and largest last key that the tile's rows see, over rows that see any
  int j0, nblk;    // key blocks; nblk -1: no more work
  int slot;        // workspace slot, or -1 for a tile done whole
  int holes;       // some page of these blocks does not exist
  int lim[kSqdkBM];  // last key each query sees, -1 for none
};

// A request's tiles. Costs are linear in the tile number: first + t * slope.
struct ChunkRequest {
  int q0, len, kv, tiles;
  int first, slope, head;  // head: the sum over a head's tiles
  __device__ __forceinline__ int before(int n) const {
    return first * n + static_cast<int>(static_cast<int64_t>(n) * (n - 1) / 2 * slope);
  }
};

__device__ __forceinline__ ChunkRequest chunk_request(const ChunkParams& p, int split, int r) {
  ChunkRequest c;
  const PagedRequest q = paged_rows(p.a, paged_raw(p.a, r));
  c.q0 = q.q0;
  c.len = q.rows / p.a.G;
  c.kv = q.kv;
  c.tiles = 0;
  c.first = c.slope = c.head = 0;
  if (q.rows <= split) return c;  // the 16-row kernel's
  c.tiles = (c.len + p.QT - 1) / p.QT;
  const int64_t top = max(c.kv - 1, 0);
  const int lo = static_cast<int>(min(max(load_now(p.a.pos + c.q0 + min(p.QT, c.len) - 1), static_cast<int64_t>(0)), top));
  const int hi = static_cast<int>(min(max(load_now(p.a.pos + c.q0 + c.len - 1), static_cast<int64_t>(0)), top));
  constexpr int kShift = 2;  // 64 keys = kChunkUnit units
  static_assert(kSqdkBN >> kShift == kChunkUnit, "cost units");
  const int sh = kShift + p.a.cost_shift;
  c.first = (lo >> sh) + ((kChunkUnit * (1 + kChunkTileCost)) >> p.a.cost_shift) + 1;
  c.slope = c.tiles > 1 ? static_cast<int>(static_cast<unsigned>(max(hi - lo, 0) >> sh) / static_cast<unsigned>(c.tiles - 1)) : 0;
  c.head = c.before(c.tiles);
  return c;
}

struct ChunkTile {
  ChunkRequest req;
  int split, r, head, t;
  int start, cost;  // place in the list
  // Only called while a next tile exists.
  __device__ __forceinline__ void next(const ChunkParams& p) {
    start += cost;
    if (++t == req.tiles) {
      t = 0;
      if (++head == p.a.Hkv) {
        head = 0;
        do req = chunk_request(p, split, ++r);
        while (req.tiles == 0 && r + 1 < p.a.R);
      }
    }
    cost = req.first + req.slope * t;
  }
};

// The list of tiles, as one warp sees it: the first 32 requests' shares stay in
// its lanes, later ones are read again.
struct ChunkList {
  const ChunkParams& p;
  int split, lane;
  int mine, upto;  // cost of request `lane`, and with all before it
  __device__ __forceinline__ ChunkList(const ChunkParams& p_, int split_, int lane_)
      : p(p_), split(split_), lane(lane_) {
    mine = cost(lane);
    upto = warp_scan(mine, lane);
  }
  __device__ __forceinline__ int cost(int r) const { return r < p.a.R ? chunk_request(p, split, r).head * p.a.Hkv : 0; }
  __device__ __forceinline__ int total() const {
    int n = mine;
    for (int r = lane + 32; r < p.a.R; r += 32) n += cost(r);
    return __reduce_add_sync(0xFFFFFFFFu, n);
  }
  // The tile that holds list place w (below the total).
  __device__ __forceinline__ ChunkTile locate(int w) const {
    ChunkTile c;
    int base = 0, own = mine, sum = upto;
    c.r = p.a.R - 1;
    for (int r0 = 0; r0 < p.a.R; r0 += 32) {
      if (r0 > 0) own = cost(r0 + lane), sum = warp_scan(own, lane);
      const unsigned past = __ballot_sync(0xFFFFFFFFu, base + sum > w);
      if (past) {
        const int l = __ffs(past) - 1;
        base += __shfl_sync(0xFFFFFFFFu, sum - own, l);
        c.r = r0 + l;
        break;
      }
      base += __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    c.split = split;
    c.req = chunk_request(p, split, c.r);
    const unsigned rel = w - base;
    c.head = static_cast<int>(rel / static_cast<unsigned>(c.req.head));
    const int in_head = static_cast<int>(rel) - c.head * c.req.head;
    // the last tile t with first t + slope t (t - 1) / 2 <= in_head: the root
    // in float, set right in integers
    const float b = static_cast<float>(c.req.first) - 0.5f * static_cast<float>(c.req.slope);
    const float x = static_cast<float>(in_head), root = sqrtf(b * b + 2.0f * static_cast<float>(c.req.slope) * x);
    int t = min(max(static_cast<int>(__fdividef(2.0f * x, b + root)), 0), c.req.tiles - 1);
    while (t > 0 && c.req.before(t) > in_head) --t;
    while (t + 1 < c.req.tiles && c.req.before(t + 1) <= in_head) ++t;
    c.t = t;
    c.start = base + c.head * c.req.head + c.req.before(t);
    c.cost = c.req.first + c.req.slope * t;
    return c;
  }
};

// Runs of the list. Of the two CTAs that share an SM, the one launched first (the
// first half of a full grid) is 10 % faster while both are at work, so its run is
// longer: with a tilt of 0, 3, 5, 7 64ths, 285.0, 280.5, 280.6, 284.6 us for seven
// prompts, 131.2, 128.5, 129.4, 130.2 for 52 requests of chunks and single tokens
// (calls in a row for seconds).
struct ChunkRuns {
  int share, rem, tilt, n;
  __device__ __forceinline__ ChunkRuns(int total, int runs, int most) {
    const Runs even(total, runs);
    n = runs;
    share = even.share;
    rem = even.rem;
    tilt = runs == most && (runs & 1) == 0 ? share / 64 * kChunkTilt : 0;
  }
  __device__ __forceinline__ int start(int c) const { return share * c + tilt * min(c, n - c) + min(c, rem); }
  // The run that holds list place w.
  __device__ __forceinline__ int of(int w) const {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start(mid) <= w) lo = mid;
      else hi = mid;
    }
    return lo;
  }
};

// The list cut into runs. A cut so near to an end of its tile that the piece
// would not be worth its merge is moved to that end.
struct ChunkCuts {
  ChunkRuns run;
  int total, near;
  __device__ __forceinline__ ChunkCuts(const ChunkParams& p, int total_, int most)
      : run(total_, min(most, max(total_ / max((kChunkUnit * kChunkMinPiece) >> p.a.cost_shift, 1), 1)), most),
        total(total_),
        near(min(run.share >> 4, (8 * kChunkUnit) >> p.a.cost_shift)) {}
  // The first run that begins behind list place w (the start of a tile that a cut divides).
  __device__ __forceinline__ int first_inside(int w) const {
    int c = run.of(w) + 1;
    while (run.start(c) - w <= near) ++c;
    return c;
  }
};

// Walks a run's pieces: the whole tiles in order, then the piece at the run's
// start, then the one at its end.
struct ChunkWalk {
  ChunkTile first, cur;
  int w0, w1;
  int stage;  // 0: whole tiles, 1: piece at the start, 2: piece at the end, 3: done
  bool started;
  __device__ __forceinline__ void open(const ChunkList& list, const ChunkCuts& cuts, int c) {
    stage = 3;
    started = false;
    w0 = w1 = 0;
    if (c >= cuts.run.n || cuts.total == 0) return;
    // the two ends, the start last: its tile is where the walk begins
    w1 = cuts.total;
#pragma unroll 1
    for (int k = c + 1 < cuts.run.n ? 1 : 0; k >= 0; --k) {
      w0 = cuts.run.start(c + k);
      cur = list.locate(w0);
      const int behind = cur.start + cur.cost;
      if (w0 - cur.start <= cuts.near) w0 = cur.start;
      else if (behind - w0 <= cuts.near) w0 = behind;
      if (k == 1) w1 = w0;
    }
    if (w0 >= w1) return;
    if (w0 == cur.start + cur.cost) cur.next(list.p);
    first = cur;
    stage = 0;
  }
  // The next piece's tile; slot and merge say what it is.
  __device__ __forceinline__ bool next(const ChunkParams& p, ChunkTile& tile, int& slot) {
    while (stage == 0) {
      if (started) {
        if (cur.start + cur.cost >= w1) {
          stage = 1;
          break;
        }
        cur.next(p);
      }
      started = true;
      if (cur.start < w0) continue;
      if (cur.start + cur.cost > w1) {
        stage = 1;
        break;
      }
      tile = cur;
      slot = -1;
      return true;
    }
    // cur is the run's last tile now
    if (stage == 1) {
      stage = 2;
      if (first.start < w0) {
        tile = first;
        slot = 2 * static_cast<int>(blockIdx.x);
        if (first.start + first.cost >= w1) stage = 3;  // the run lies inside one tile
        return true;
      }
    }
    if (stage == 2) {
      stage = 3;
      if (cur.start + cur.cost > w1) {
        tile = cur;
        slot = 2 * static_cast<int>(blockIdx.x) + 1;
        return true;
      }
    }
    return false;
  }
};

// Key block at list place w of a tile with nblk blocks.
__device__ __forceinline__ int chunk_block_at(const ChunkTile& c, int w, int nblk) {
  const int64_t x = static_cast<int64_t>(min(max(w - c.start, 0), c.cost)) * nblk;
  // (64-bit divisions are slow, and most lists are short)
  if ((x >> 32) == 0) return static_cast<int>(static_cast<unsigned>(x) / static_cast<unsigned>(c.cost));
  return static_cast<int>(x / c.cost);
}

// Fills in a job for list places [a, b) of a tile (the whole warp).
__device__ __forceinline__ void chunk_job(const ChunkParams& p, const ChunkTile& c, int a, int b, int slot,
                                          volatile ChunkJob& job, int lane) {
  int lo = 0x7FFFFFFF, hi = -1;
  const int n = min(p.QT, c.req.len - c.t * p.QT);
  bool beyond = false;
  for (int i = lane; i < n; i += 32) {
    const int64_t ps = load_now(p.a.pos + c.req.q0 + c.t * p.QT + i);
    const int lim = static_cast<int>(min(max(ps, static_cast<int64_t>(-1)), static_cast<int64_t>(c.req.kv) - 1));
    beyond |= ps >= c.req.kv;
    job.lim[i] = lim;
    if (lim >= 0) lo = min(lo, lim);
    hi = max(hi, lim);
  }
  if (beyond) raise_device_error(HSPMN_DEVERR_POSITION);
  lo = __reduce_min_sync(0xFFFFFFFFu, lo);
  hi = __reduce_max_sync(0xFFFFFFFFu, hi);
  const int all = hi < 0 ? 0 : hi / kSqdkBN + 1;
  const int j0 = chunk_block_at(c, a, all), nblk = chunk_block_at(c, b, all) - j0;
  bool holes = false;
  if (nblk > 0) {
    const int* row = p.a.table + static_cast<int64_t>(c.r) * p.a.table_rs;
    const int last = (min((j0 + nblk) * kSqdkBN, c.req.kv) - 1) >> p.a.shift;
    for (int pg = ((j0 * kSqdkBN) >> p.a.shift) + lane; pg <= last; pg += 32) {
      const int x = load_now(row + pg);
      holes |= x < 0 || x >= p.a.num_pages;
    }
    holes = __any_sync(0xFFFFFFFFu, holes);
    if (holes && lane == 0) raise_device_error(HSPMN_DEVERR_PAGE);
  }
  if (lane == 0) {
    job.row0 = c.req.q0 + c.t * p.QT;
    job.queries = n;
    job.r = c.r;
    job.head = c.head;
    job.kv = c.req.kv;
    job.lo = lo;
    job.hi = hi;
    job.j0 = j0;
    job.nblk = nblk;
    job.slot = slot;
    job.holes = holes;
  }
  __syncwarp();
}

constexpr int kNoKey = 0x7FFFFFFF;

// Notes in keys ([2][HD]: +inf, -inf) what element `h` of a key's V is, if it is an
// infinity or NaN.
template <bool kBF16, int HD>
__device__ __forceinline__ void note_wild(int (&keys)[2][HD], int col, uint32_t h, int key) {
  if (!not_finite2<kBF16>(h)) return;
  const bool nan = (h & (kBF16 ? 0x7Fu : 0x3FFu)) != 0, negative = (h & 0x8000u) != 0;
  if (nan || !negative) atomicMin(&keys[0][col], key);
  if (nan || negative) atomicMin(&keys[1][col], key);
}

template <int HD, bool kBF16>
__global__ void __launch_bounds__(kChunkThreads, kChunkCtasPerSm)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ ChunkParams p) {
  using L = ChunkLayout<HD>;
  extern __shared__ uint8_t chunk_smem_raw[];
  // Blocks are numbered through the whole run: block n uses S buffer, K stage
  // and V stage n & 1, and phase n >> 1 of their barriers. One thread issues
  // every product and they complete in order, so bar_sfull (Q K^T of block n
  // done) also frees K stage n & 1 and, after a tile's last block, the Q tile.
  __shared__ __align__(8) uint64_t bar_q, bar_kfull[2], bar_vfull[2], bar_vempty[2], bar_sfull[2], bar_pfull[2];
  __shared__ __align__(8) uint64_t bar_ofinal, bar_drain, bar_job[2], bar_jobdone[2];
  __shared__ volatile ChunkJob jobs[2];  // by the job's number: the next is posted while one is worked on
  __shared__ int64_t row_off[kSqdkBM];  // of a tile's row in o, from the tile's first query and head; -1: no row
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile uint32_t abort_flag;
  // an infinity or NaN was taken out of V for rows that do not see it, and the
  // first key of each column at which a +inf, a -inf was (a NaN is both): rows see
  // a prefix of the keys, so that is all they need to know, however many there are
  // (both by the job's parity: one is cleared while the other is in use)
  __shared__ volatile uint32_t wild_flag[2];
  __shared__ int wild_key[2][2][HD];

  const uint32_t sbase = (smem_u32(chunk_smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_enter();  // (the 16-row kernel counts on it too)
  // no request for this kernel, or bad offsets (the 16-row kernel says so):
  // nothing to set up
  const int split = paged_split<PagedLayout<HD>::kKeys>(p.a, lane);
  bool any = false, bad = false;
  for (int r = lane; r <= p.a.R; r += 32) {
    const PagedRaw x = paged_raw(p.a, r);
    bad |= paged_offsets_bad(x, r);
    any |= r < p.a.R && paged_rows(p.a, x).rows > split;
  }
  if (!__any_sync(0xFFFFFFFFu, any) || __any_sync(0xFFFFFFFFu, bad)) {
    if (threadIdx.x == 0) p.a.merges[blockIdx.x] = make_int4(0, 0, 0, -1);
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(&bar_q, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar_kfull[s], 1);
      mbar_init(&bar_vfull[s], 1);
      mbar_init(&bar_vempty[s], 1);
      mbar_init(&bar_sfull[s], 1);
      mbar_init(&bar_pfull[s], 4);  // one arrival per softmax warp
      mbar_init(&bar_job[s], 1);
      mbar_init(&bar_jobdone[s], 5);  // the MMA warp and the softmax warps
    }
    mbar_init(&bar_ofinal, 1);
    mbar_init(&bar_drain, 1);
    abort_flag = 0u;
    wild_flag[0] = wild_flag[1] = 0u;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, L::kTmemCols);
    tmem_relinquish();
  }
  if (threadIdx.x >= 64) {
    const int rr = threadIdx.x - 64, ql = rr / p.a.G;
    row_off[rr] = ql < p.QT ? ql * p.a.o_sn + (rr - ql * p.a.G) * p.a.o_sh : -1;
    for (int x = 0; x < 2; ++x)
      if (rr < HD) wild_key[x][0][rr] = wild_key[x][1][rr] = kNoKey;
    // rows behind the G * QT that the copies of Q fill: zeros, since what shared
    // memory happens to hold there would share its warp's choice of a maximum
    if (ql >= p.QT) {
      for (int c = 0; c < L::kChunks * 8; ++c)
        st_shared_v4(sbase + L::kQOff + (c >> 3) * L::kQChunkBytes + rr * 128 + (c & 7) * 16, make_uint4(0u, 0u, 0u, 0u));
      fence_proxy_async_smem();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const int boxes = kSqdkBN / p.box_rows;
    const ChunkList list(p, split, lane);
    const ChunkCuts cuts(p, list.total(), static_cast<int>(gridDim.x));
    ChunkWalk walk;
    walk.open(list, cuts, blockIdx.x);
    uint32_t nk = 0, nv = 0, segs = 0, posted = 0;
    bool live = true;
    bool goes_on = false;
    ChunkTile tile;
    int slot;
    while (live) {
      const bool more = walk.next(p, tile, slot);
      volatile ChunkJob& job = jobs[posted & 1];
      if (posted > 1 && !__all_sync(0xFFFFFFFFu, mbar_wait(&bar_jobdone[posted & 1], ((posted >> 1) - 1) & 1, &abort_flag)))
        break;
      if (more) {
        chunk_job(p, tile, slot < 0 ? tile.start : walk.w0, slot < 0 ? tile.start + tile.cost : walk.w1, slot, job, lane);
      } else if (lane == 0) {
        job.nblk = -1;
      }
      if (lane == 0) mbar_arrive(&bar_job[posted & 1]);
      ++posted;
      __syncwarp();
      if (!more) break;
      if (slot >= 0 && tile.start + tile.cost > walk.w1) {
        // the tile goes on behind this run: its runs from the one in which it
        // begins to the last that begins inside it share its merge
        const int end = tile.start + tile.cost;
        const int first = slot & 1 ? static_cast<int>(blockIdx.x) : cuts.first_inside(tile.start) - 1;
        int last = cuts.run.of(end - 1);
        if (end - cuts.run.start(last) <= cuts.near) --last;
        goes_on = true;
        if (lane == 0)
          p.a.merges[blockIdx.x] = make_int4(tile.req.q0 + tile.t * p.QT, min(p.QT, tile.req.len - tile.t * p.QT),
                                             tile.head, first << 16 | last);
      }
      const int nblk = job.nblk, j0 = job.j0;
      if (nblk == 0) continue;
      if (nk > 0) live = __all_sync(0xFFFFFFFFu, mbar_wait(&bar_sfull[(nk - 1) & 1], ((nk - 1) >> 1) & 1, &abort_flag));
      if (!live) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bar_q, static_cast<uint32_t>(L::kChunks * p.a.G * p.QT * 128));
        for (int c = 0; c < L::kChunks; ++c)
          tma_load_4d(sbase + L::kQOff + c * L::kQChunkBytes, &tmQ, &bar_q, c * 64, tile.head * p.a.G,
                      tile.req.q0 + tile.t * p.QT, 0);
      }
      ++segs;
      const int* row = p.a.table + static_cast<int64_t>(tile.r) * p.a.table_rs;
      const int mask = (1 << p.a.shift) - 1;
      // this lane's page of block j; a page that does not exist (and a box
      // behind the cached tokens) is read from behind the last page: zeros
      auto page_at = [&](int j) -> int {
        const int key = (j0 + j) * kSqdkBN + lane * p.box_rows;
        if (lane >= boxes || key >= tile.req.kv) return p.a.num_pages;
        const int pg = load_now(row + (key >> p.a.shift));
        return pg >= 0 && pg < p.a.num_pages ? pg : p.a.num_pages;
      };
      auto load = [&](const CUtensorMap* map, uint64_t* bar, uint32_t dst, int j, int page) {
        if (lane == 0) mbar_arrive_expect_tx(bar, L::kKVBytes);
        __syncwarp();
        if (lane < boxes) {
          const int off = ((j0 + j) * kSqdkBN + lane * p.box_rows) & mask;
          for (int c = 0; c < L::kChunks; ++c)
            tma_load_4d(dst + c * L::kKVChunkBytes + lane * p.box_rows * 128, map, bar, c * 64, tile.head, off, page);
        }
      };
      int page_k = page_at(0), page_v = page_k;
      auto load_k = [&](int j) -> bool {
        const uint32_t st = nk & 1, ph = nk >> 1;
        if (ph > 0 && !__all_sync(0xFFFFFFFFu, mbar_wait(&bar_sfull[st], (ph - 1) & 1, &abort_flag))) return false;
        load(&tmK, &bar_kfull[st], sbase + L::kKOff + st * L::kKVBytes, j, page_k);
        ++nk;
        return true;
      };
      live = load_k(0);
      for (int j = 0; live && j < nblk; ++j) {
        if (j + 1 < nblk) {
          page_k = page_at(j + 1);
          live = load_k(j + 1);
          if (!live) break;
        }
        const uint32_t st = nv & 1, ph = nv >> 1;
        if (ph > 0 && !__all_sync(0xFFFFFFFFu, mbar_wait(&bar_vempty[st], (ph - 1) & 1, &abort_flag))) {
          live = false;
          break;
        }
        load(&tmV, &bar_vfull[st], sbase + L::kVOff + st * L::kKVBytes, j, page_v);
        page_v = page_k;
        ++nv;
      }
    }
    if (lane == 0 && !goes_on) p.a.merges[blockIdx.x] = make_int4(0, 0, 0, -1);
    // every copy this warp issued has landed before the CTA may exit
    if (lane == 0) {
      if (segs > 0) mbar_wait_drain(&bar_q, (segs - 1) & 1);
      for (uint32_t st = 0; st < 2; ++st) {
        if (nk > st) mbar_wait_drain(&bar_kfull[st], ((nk - 1 - st) >> 1) & 1);
        if (nv > st) mbar_wait_drain(&bar_vfull[st], ((nv - 1 - st) >> 1) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issue
    constexpr int kAB = kBF16 ? 1 : 0;
    constexpr uint32_t idesc_s = umma_idesc_f16(kSqdkBM, kSqdkBN, kAB, false, false);
    constexpr uint32_t idesc_o = umma_idesc_f16(kSqdkBM, HD, kAB, false, true);
    const uint32_t tO = tmem + L::kOCol;
    const uint64_t qdesc = sw128_desc(sbase + L::kQOff, 16, 1024);
    const uint64_t kdesc = sw128_desc(sbase + L::kKOff, 16, 1024);
    const uint64_t vdesc = sw128_desc(sbase + L::kVOff, L::kKVChunkBytes, 1024);
    uint32_t n = 0, segs = 0;
    bool ok = true;
    auto issue_pv = [&](uint32_t m, bool first) -> bool {
      const uint32_t sb = m & 1, ph = (m >> 1) & 1;
      if (!__all_sync(0xFFFFFFFFu, mbar_wait2(&bar_pfull[sb], ph, &bar_vfull[sb], ph, &abort_flag))) return false;
      tc_fence_after();
      const uint64_t vd = vdesc + static_cast<uint64_t>((sb * L::kKVBytes) >> 4);
      const uint32_t ta = tmem + sb * kSqdkBN;
      umma_ts_warp(tO, ta, vd, idesc_o, first ? 0u : 1u);
#pragma unroll
      for (int kk = 1; kk < kSqdkBN / 16; ++kk)
        umma_ts_warp(tO, ta + kk * 8, vd + static_cast<uint64_t>((kk * 16 * 128) >> 4), idesc_o, 1u);
      umma_commit_warp(&bar_vempty[sb]);
      return true;
    };
    for (uint32_t i = 0; ok; ++i) {
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(&bar_job[i & 1], (i >> 1) & 1, &abort_flag));
      if (!ok) break;
      const int nblk = jobs[i & 1].nblk;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_jobdone[i & 1]);
      if (nblk < 0) break;
      if (nblk == 0) continue;
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(&bar_q, segs & 1, &abort_flag));
      ++segs;
      if (!ok) break;
      tc_fence_after();
      for (int j = 0; ok && j < nblk; ++j, ++n) {
        const uint32_t sb = n & 1;
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(&bar_kfull[sb], (n >> 1) & 1, &abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t kd = kdesc + static_cast<uint64_t>((sb * L::kKVBytes) >> 4);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const int c = kk >> 2, w = kk & 3;
          umma_ss_warp(tmem + sb * kSqdkBN, qdesc + static_cast<uint64_t>((c * L::kQChunkBytes + w * 32) >> 4),
                       kd + static_cast<uint64_t>((c * L::kKVChunkBytes + w * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit_warp(&bar_sfull[sb]);
        if (j >= 1) ok = issue_pv(n - 1, j == 1);
      }
      if (ok) ok = issue_pv(n - 1, nblk == 1);
      if (ok) umma_commit_warp(&bar_ofinal);
    }
    umma_commit_warp(&bar_drain);
    if (lane == 0) mbar_wait_drain(&bar_drain, 0);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    const int sw = warp & 3;  // tensor memory lanes 32 * sw ..
    const uint32_t lane_base = static_cast<uint32_t>(32 * sw) << 16;
    const uint32_t tS = tmem + lane_base;
    const uint32_t tO = tmem + lane_base + L::kOCol;
    const int r = 32 * sw + lane;
    const int qloc = r / p.a.G;
    const float c2 = p.a.scale_log2;
    uint32_t n = 0, segs = 0, walked = 0;
    while (true) {
      // The four warps agree on each job, so that all of them meet at the barrier
      // of its epilogue even if some wait gives up; behind this one, every warp
      // has left the job before.
      const bool posted = __all_sync(0xFFFFFFFFu, mbar_wait(&bar_job[walked & 1], (walked >> 1) & 1, &abort_flag));
      if (!named_bar_and(kChunkEpilogueBar, 128, posted)) break;
      if (threadIdx.x == 64) wild_flag[(walked + 1) & 1] = 0u;
      if (r < HD) wild_key[(walked + 1) & 1][0][r] = wild_key[(walked + 1) & 1][1][r] = kNoKey;
      bool ok = true;
      volatile ChunkJob& job = jobs[walked & 1];
      const int nblk = job.nblk, j0 = job.j0;
      if (nblk < 0) break;
      const bool row_valid = qloc < p.QT && qloc < job.queries;
      // rows that see nothing run along like the tile's last row; what they
      // compute is not stored
      const int tile_hi = job.hi, tile_lo = job.lo;
      const bool holes = job.holes != 0;
      int lim = row_valid ? job.lim[qloc] : -1;
      const bool blind = lim < 0;
      if (blind) lim = tile_hi;
      bool seen = !blind && lim >= j0 * kSqdkBN && nblk > 0 && !holes;
      float m_run = -INFINITY, l_run = 0.0f;
      for (int j = 0; j < nblk; ++j, ++n) {
        const uint32_t sb = n & 1;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&bar_sfull[sb], (n >> 1) & 1, &abort_flag));
        if (!ok) break;
        tc_fence_after();
        float sv[kSqdkBN];
        {
          uint32_t r0[32], r1[32];
          tmem_ld32(tS + sb * kSqdkBN, r0);
          tmem_ld32(tS + sb * kSqdkBN + 32, r1);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            sv[i] = __uint_as_float(r0[i]);
            sv[32 + i] = __uint_as_float(r1[i]);
          }
        }
        const int key0 = (j0 + j) * kSqdkBN;
        const int left = lim - key0;  // columns <= left are visible to this row
        // the same for every warp: does any row of the tile not see all of this block?
        const bool edge = key0 + kSqdkBN - 1 > tile_lo;
        if (edge) {
#pragma unroll
          for (int c = 0; c < kSqdkBN; ++c) sv[c] = (c <= left) ? sv[c] : -INFINITY;
        }
        if (holes) {
          const int* row = p.a.table + static_cast<int64_t>(job.r) * p.a.table_rs;
          for (int c0 = 0; c0 < kSqdkBN; c0 += 8) {
            const int x = key0 + c0 < job.kv ? load_now(row + ((key0 + c0) >> p.a.shift)) : -1;
            const bool gone = x < 0 || x >= p.a.num_pages;
            seen |= !gone && !blind && c0 <= left;
#pragma unroll
            for (int c = 0; c < kSqdkBN; ++c)
              if ((c & ~7) == c0 && gone) sv[c] = -INFINITY;
          }
        }
        uint32_t pk[kSqdkBN / 2];
        // p = 2^((s - m) c2), packed in the operands' type (as in the 16-row kernel, for
        // the same reason: half a step, the size of the output's own rounding; the row
        // sum takes p before it); returns the block's row sum. kFma: as
        // s c2 - (m c2), one operation instead of two, with the rounding of m c2
        // (2^-15 at kChunkFmaMax) in every p.
        auto exponentiate = [&](auto kFma, float m) -> float {
          const float neg = (m == -INFINITY) ? 0.0f : kFma ? -(m * c2) : -m;
          const uint64_t cc = f2_pack(c2, c2), nm = f2_pack(neg, neg);
          uint64_t acc0 = f2_pack(0.0f, 0.0f), acc1 = acc0;
#pragma unroll
          for (int c = 0; c < kSqdkBN; c += 2) {
            float x0, x1;
            const uint64_t s2 = f2_pack(sv[c], sv[c + 1]);
            if constexpr (kFma) f2_unpack(f2_fma(s2, cc, nm), x0, x1);
            else f2_unpack(f2_mul(f2_add(s2, nm), cc), x0, x1);
            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
            if ((c >> 1) & 1) acc1 = f2_add(acc1, f2_pack(p0, p1));
            else acc0 = f2_add(acc0, f2_pack(p0, p1));
            pk[c >> 1] = pack2<kBF16>(p0, p1);
          }
          float a0, a1, b0, b1;
          f2_unpack(acc0, a0, a1);
          f2_unpack(acc1, b0, b1);
          return (a0 + a1) + (b0 + b1);
        };
        bool done = false;
        if (__all_sync(0xFFFFFFFFu, fabsf(m_run) * c2 <= kChunkFmaMax)) {
          const float lb = exponentiate(std::true_type{}, m_run);
          if (__all_sync(0xFFFFFFFFu, lb < kSqdkSumBound<kBF16>)) {
            l_run += lb;
            done = true;
          }
        }
        if (!done) {
          float mq[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
          for (int c = 4; c < kSqdkBN; c += 4) {
#pragma unroll
            for (int u = 0; u < 4; ++u) mq[u] = fmaxf(mq[u], sv[c + u]);
          }
          const float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]));
          const float m_new = fmaxf(m_run, mx);
          const bool need_o = j > 0 && (m_run != -INFINITY) && (m_new > m_run);
          if (__any_sync(0xFFFFFFFFu, need_o)) {
            // P V of the block before must have landed in O
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&bar_vempty[(n - 1) & 1], ((n - 1) >> 1) & 1, &abort_flag));
            if (!ok) break;
            tc_fence_after();
            const float alpha = need_o ? fast_exp2((m_run - m_new) * c2) : 1.0f;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t x[32];
              tmem_ld32(tO + c, x);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * alpha);
              tmem_st32(tO + c, x);
            }
            tmem_wait_st();
          }
          if (m_new != m_run) {
            l_run = (m_run == -INFINITY) ? 0.0f : l_run * fast_exp2((m_run - m_new) * c2);
            m_run = m_new;
          }
          l_run += exponentiate(std::false_type{}, m_run);
        }
        tmem_st32(tS + sb * kSqdkBN, pk);
        tmem_wait_st();
        tc_fence_before();
        if (edge) {
          // P is zero where a row does not see a key, but 0 * inf is not: V
          // rows that no row sees (the page's unwritten end) become zeros, and
          // infinities and NaN leave the rows that only some see (they are noted,
          // and the epilogue gives them back to those that do). 16 keys a warp.
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(&bar_vfull[sb], (n >> 1) & 1, &abort_flag));
          if (!ok) break;
          const uint32_t vst = sbase + L::kVOff + sb * L::kKVBytes;
          bool found = false;
          if (key0 + 16 * sw + 15 > tile_lo) {
#pragma unroll 4
            for (int i = lane; i < 16 * 8 * L::kChunks; i += 32) {
              const int kr = 16 * sw + (i >> 3) % 16, key = key0 + kr;
              const uint32_t addr = vst + (i >> 7) * L::kKVChunkBytes + kr * 128 + (i & 7) * 16;
              if (key > tile_hi) {
                st_shared_v4(addr, make_uint4(0u, 0u, 0u, 0u));
              } else if (key > tile_lo) {
                uint4 w;
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                             : "r"(addr));
                if (not_finite2<kBF16>(w.x) || not_finite2<kBF16>(w.y) || not_finite2<kBF16>(w.z) ||
                    not_finite2<kBF16>(w.w)) {
                  found = true;
                  // (the tile's 16-byte chunks lie swizzled by their row)
                  const int col = (i >> 7) * 64 + (((i & 7) ^ (kr & 7)) << 3);
                  const uint32_t pair[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                  for (int u = 0; u < 4; ++u) {
                    note_wild<kBF16>(wild_key[walked & 1], col + 2 * u, pair[u] & 0xFFFFu, key);
                    note_wild<kBF16>(wild_key[walked & 1], col + 2 * u + 1, pair[u] >> 16, key);
                  }
                  w.x = finite2<kBF16>(w.x), w.y = finite2<kBF16>(w.y), w.z = finite2<kBF16>(w.z), w.w = finite2<kBF16>(w.w);
                  st_shared_v4(addr, w);
                }
              }
            }
          }
          if (found) wild_flag[walked & 1] = 1u;
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_pfull[sb]);
      }
      // ---------------------------------------------------------- epilogue
      if (ok && nblk > 0) ok = __all_sync(0xFFFFFFFFu, mbar_wait(&bar_ofinal, segs & 1, &abort_flag));
      if (nblk > 0) ++segs;
      const bool live = named_bar_and(kChunkEpilogueBar, 128, ok);  // every warp has set this job's flag
      const int parity = walked & 1;
      const bool wild = wild_flag[parity] != 0u;
      ++walked;
      if (!live) break;
      tc_fence_after();
      const bool none = !seen;
      const int slot = job.slot, head = job.head;
      const int64_t row0 = job.row0;
      const float inv_l = 1.0f / l_run;
      char* base = p.a.o + row0 * p.a.o_sn + static_cast<int64_t>(head) * p.a.G * p.a.o_sh + (lane & 3) * 16;
      const int rows = job.queries * p.a.G;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float o[32];
        if (nblk > 0) {
          uint32_t x[32];
          tmem_ld32(tO + c, x);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(x[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.0f;
        }
        if (wild && row_valid && !blind) {
          // the infinities and NaN that this row does see
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (wild_key[parity][0][c + i] <= lim) o[i] += INFINITY;
            if (wild_key[parity][1][c + i] <= lim) o[i] -= INFINITY;
          }
        }
        if (slot >= 0) {
          // unnormalised O of this piece, rows side by side in groups of four
          // columns: a warp's stores are whole lines
          float4* dst = reinterpret_cast<float4*>(p.a.part_o) + (static_cast<int64_t>(slot) * (HD / 4) + c / 4) * kSqdkBM + r;
          if (row_valid)
#pragma unroll
            for (int v = 0; v < 8; ++v) dst[v * kSqdkBM] = make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
          continue;
        }
        // 32 columns of the warp's 32 rows through shared memory, so that a
        // row's 64 bytes leave together
        const uint32_t stage = sbase + L::kOOff + sw * 32 * 64;
        const uint32_t keep = none ? 0u : 0xFFFFFFFFu;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a, b;
            f2_unpack(f2_mul(f2_pack(o[8 * v + 2 * i], o[8 * v + 2 * i + 1]), f2_pack(inv_l, inv_l)), a, b);
            w[i] = pack2<kBF16>(a, b) & keep;
          }
          st_shared_v4(stage + lane * 64 + ((v ^ ((lane >> 1) & 3)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int lr = i * 8 + (lane >> 2), rr = 32 * sw + lr;
          uint4 w;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                       : "r"(stage + lr * 64 + (((lane & 3) ^ ((lr >> 1) & 3)) << 4)));
          if (rr < rows && c + (lane & 3) * 8 < p.a.hd) *reinterpret_cast<uint4*>(base + row_off[rr] + c * 2) = w;
        }
        __syncwarp();
      }
      if (slot >= 0 && row_valid)
        reinterpret_cast<float2*>(p.a.part_ml)[static_cast<int64_t>(slot) * kSqdkBM + r] =
            make_float2(m_run, none ? kUnseen : l_run);
      tc_fence_before();  // O has been read: the next tile's first P V (behind this warp's arrival) may write it
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_jobdone[parity]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// Adds the pieces of the tile that goes on behind run `run`, as that run noted:
// O = sum w_c O_c / sum w_c l_c, w_c = 2^(c2 (m_c - M)), over the runs in order. Every run
// that the tile goes on behind gives kChunkMergeBlocks blocks to it. A warp takes
// 8 rows by 16 columns at a time (128-byte reads of the pieces); where there are
// more warps than that needs, several share the pieces.
constexpr int kChunkMergeBlocks = 4;

template <int HD, bool kBF16>
__device__ __forceinline__ void chunk_merge(const ChunkParams& p, int run, int share) {
  __shared__ float s_m[kMergeWarps][32], s_l[kMergeWarps][32];
  __shared__ float4 s_o[kMergeWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 note = p.a.merges[run];
  if (note.w < 0) return;
  const int c0 = note.w >> 16, c1 = note.w & 0xFFFF, pieces = c1 - c0 + 1;
  const float2* ml = reinterpret_cast<const float2*>(p.a.part_ml);
  const float4* part = reinterpret_cast<const float4*>(p.a.part_o);
  const int rows = note.y * p.a.G;
  const int units = (rows + 7) / 8 * (HD / 16), blocks = (c1 - c0) * kChunkMergeBlocks;
  // warps a unit: a power of two up to 16, two pieces a warp at least
  int k = 1;
  while (k < kMergeWarps && 2 * k * units <= blocks * kMergeWarps && 4 * k <= pieces) k *= 2;
  const int per = (pieces + k - 1) / k, from = c0 + warp % k * per, to = min(c1 + 1, from + per);
  const int step = blocks * (kMergeWarps / k);
  // every warp of the block takes as many turns
  for (int i0 = ((run - c0) * kChunkMergeBlocks + share) * (kMergeWarps / k); i0 < units; i0 += step) {
    const int i = i0 + warp / k;
    const int r = i / (HD / 16) * 8 + (lane >> 2), q4 = i % (HD / 16) * 4 + (lane & 3);  // row, group of 4 columns
    const bool live = i < units && r < rows && q4 * 4 < p.a.hd;
    float M = -INFINITY, l = 0.0f;
    bool none = true;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float m, float s, const float4& v) {
      if (s == kUnseen) return;
      none = false;
      const float top = fmaxf(M, m);
      const float f = m == top ? 1.0f : fast_exp2((m - top) * p.a.scale_log2);
      const float g = M == top ? 1.0f : fast_exp2((M - top) * p.a.scale_log2);
      M = top;
      l = g * l + f * s;
      o.x = g * o.x + f * v.x, o.y = g * o.y + f * v.y, o.z = g * o.z + f * v.z, o.w = g * o.w + f * v.w;
    };
    if (live) {
      // four pieces' loads in flight
      for (int c = from; c < to; c += 4) {
        float2 x[4];
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (c + u >= to) continue;
          // run c0's piece is its last, the others' their first
          const int64_t slot = 2 * static_cast<int64_t>(c + u) + (c + u == c0 ? 1 : 0);
          x[u] = ml[slot * kSqdkBM + r];
          v[u] = part[(slot * (HD / 4) + q4) * kSqdkBM + r];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (c + u < to) add(x[u].x, x[u].y, v[u]);
      }
    }
    if (k > 1) {
      __syncthreads();
      s_m[warp][lane] = M;
      s_l[warp][lane] = none ? kUnseen : l;
      s_o[warp][lane] = o;
      __syncthreads();
      if (warp % k == 0)
        for (int w = warp + 1; w < warp + k; ++w) add(s_m[w][lane], s_l[w][lane], s_o[w][lane]);
    }
    if (!live || warp % k != 0) continue;
    const float inv = 1.0f / l;
    const int ql = r / p.a.G;
    uint2 w;
    w.x = none ? 0u : pack2<kBF16>(o.x * inv, o.y * inv);
    w.y = none ? 0u : pack2<kBF16>(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(p.a.o + static_cast<int64_t>(note.x + ql) * p.a.o_sn +
                              static_cast<int64_t>(note.z * p.a.G + r - ql * p.a.G) * p.a.o_sh + q4 * 8) = w;
  }
}

// Both kernels' merges in one launch: blocks [0, paged_runs) those of the 16-row
// kernel, then kChunkMergeBlocks a run of the chunks'.
template <int HD, bool kBF16>
__global__ void __launch_bounds__(32 * kMergeWarps, 2)
    paged_both_merge_kernel(const __grid_constant__ PagedAttnParams p, const __grid_constant__ ChunkParams c, int paged_runs) {
  grid_dependency_enter();
  const int block = static_cast<int>(blockIdx.x) - paged_runs;
  if (block < 0) paged_merge<HD, kBF16>(p, static_cast<int>(blockIdx.x));
  else chunk_merge<HD, kBF16>(c, block / kChunkMergeBlocks, block % kChunkMergeBlocks);
}

}  // namespace hspmn
