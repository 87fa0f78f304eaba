// Sparse-query dense-key causal attention over a paged K/V cache, for requests
// whose query rows are few: single tokens and short runs of them.
//
//   o[i,h,:] = sum_m softmax_m(scale q[i,h,:].K[m,g,:]) V[m,g,:],  g = h / (H / Hkv),
//   m over the positions of the query's request with m <= pos[i], m < kv_len
//   and a page in the table
//
// Work unit: 64 keys (128 for head_dim <= 64) of one (request, K/V head, 16 query
// rows) item; the rows of a request and K/V head are numbered query * G + head,
// so a single token's G heads share the keys that are read. All units of a call
// form one list (requests, then row tiles, then heads, then keys) which is cut
// into as many equal contiguous runs as there are CTAs: ragged lengths cost no
// idle CTA and need no plan from the host, which knows neither lengths nor
// offsets. An item that a cut divides leaves one partial result a run in the
// workspace (a run has two at most: its first item and its last), and the merge
// kernel adds them in run order, so results do not depend on timing.
//
// Bound: reading K and V once (4 query heads a key: 4 flops a byte). Each of a
// CTA's four warps owns 16 (32) keys of every unit and runs on its own: its K and
// V rows come by cp.async into a private ring (kPagedStages deep), Q K^T and P V are
// m16n8k16 products with the softmax between them in registers, and the warps
// meet only at the end of an item. Sums, maxima and O are fp32; the maximum is
// kept in the products' own units and subtracted before the scale, so that scores
// of any size weigh right. The products fill a fifth of the tensor pipe, so
// 128-row tiles would not be faster; three stages of two CTAs an SM keep 192 KB
// an SM on the way (three CTAs with two stages: 178 -> 221 us). 64 tokens over
// 1.15 GB of K and V (contexts to 32768, 16/4 heads of 128) take 176 us, 6.5 TB/s
// (175 to 184 in calls in a row for seconds, at the card's 1 kW, by the card); one
// token over 262144 keys 92 us (5.8 TB/s: the start and the merge of 74 runs
// an item take 9 us); 37 tokens of 16 heads of 64 over up to 8192 keys 63 us (4.9
// TB/s: 592 short items). One token over 500 keys takes 7.7 us, two launches and a
// few rounds of loads.
#pragma once

#include "sqdk.cuh"

namespace hspmn {

constexpr int kPagedRows = 16;     // query rows of an item
constexpr int kPagedWarps = 4;     // a quarter of a unit's keys each
constexpr int kPagedThreads = 32 * kPagedWarps;
constexpr int kPagedStages = 3;
// What opening and closing an item takes, in units (68.0 us against 86.3 at 0,
// 68.7 at 1, 69.6 at 3: 37 x 16 items of 1 to 64 units).
constexpr int kPagedItemCost = 2;
constexpr int kPagedCtasPerSm = 2;
constexpr int kPagedMidRows = 128;      // see paged_split
constexpr int kPagedMidScore = 14200;   // quarters of a microsecond: 12 us of 296 CTAs (148 SMs)

// Row sum of a part that holds no key its row sees (a true sum is not negative).
constexpr float kUnseen = -1.0f;

struct PagedAttnParams {
  const char* q;
  const char* k;
  const char* v;
  char* o;
  int64_t q_sn, q_sh, o_sn, o_sh;   // bytes
  unsigned k_sp, k_ss, v_sp, v_ss;  // bytes: page, slot in the page
  int64_t k_sh, v_sh;               // bytes: head
  const int* table;  // [R,P], row stride table_rs
  int64_t table_rs;
  const int* kv_lens;
  const int* cu_q;
  const int64_t* pos;
  float* part_o;   // [2 * runs][16][HD] unnormalised O
  float* part_ml;  // [2 * runs][16][2] maximum (of q.k, not scaled), row sum
  int4* merges;    // [runs] the item that goes on behind this run, for the merge; .w < 0: none
  int64_t N;
  int R, P, num_pages, shift, H, Hkv, G, hd;
  int has_chunks;  // the chunk kernel takes part in the call
  int cost_shift;  // the list is counted in 2^cost_shift units, so that 32 bits hold any
  float scale_log2;
};

// A request's share of the list. Request R stands for the rows behind the last
// sequence, which see nothing and are written as zeros.
struct PagedRequest {
  int q0, rows;    // first query row of q, rows = queries * G
  int kv;          // visible keys at most
  int tiles;       // 16-row tiles
  int nb;          // units of an item (one at least: it writes the rows)
};

// A request as it lies in memory.
struct PagedRaw {
  int a, b, kv;
};

__device__ __forceinline__ PagedRaw paged_raw(const PagedAttnParams& p, int r) {
  PagedRaw x;
  x.a = r <= p.R ? p.cu_q[r] : 0;
  x.b = r < p.R ? p.cu_q[r + 1] : static_cast<int>(p.N);
  x.kv = r < p.R ? p.kv_lens[r] : 0;
  return x;
}

// Whether offsets do not begin at 0, descend or end behind q. Requests would
// share rows and the lists outgrow their bounds: such a call computes nothing.
__device__ __forceinline__ bool paged_offsets_bad(const PagedRaw& x, int r) { return x.a > x.b || (r == 0 && x.a != 0); }

// The request's rows and keys (its tiles not counted).
__device__ __forceinline__ PagedRequest paged_rows(const PagedAttnParams& p, const PagedRaw& x) {
  PagedRequest q;
  const int N = static_cast<int>(p.N);
  const int a = min(max(x.a, 0), N), b = min(max(x.b, 0), N);
  const int64_t cap = static_cast<int64_t>(p.P) << p.shift;
  q.q0 = a;
  q.rows = max(b - a, 0) * p.G;
  q.kv = static_cast<int>(min(static_cast<int64_t>(max(x.kv, 0)), cap));
  return q;
}

// Rows (queries * G) of a request up to which the 16-row kernel takes it; the
// chunk kernel takes the others. Up to one tile is always the former's. Requests
// of two to eight tiles are read by it once a tile, at about 1.5 us a unit and
// CTA, and by the chunk kernel once, at about 1.75 us a unit and CTA but 12 us
// later (its setup and the merge of 128-row pieces), so they stay here while
// that is less in all: 16 us against 27 for one request of 32 rows and 8192 keys,
// 171 against 118 for 64 requests of 32 rows and 4096 keys. A batch with larger
// requests has the chunk kernel's setup anyway. Both kernels work this out from
// the same lengths.
template <int kKeys>
__device__ __forceinline__ int paged_split(const PagedAttnParams& p, int lane) {
  if (!p.has_chunks) return 0x7FFFFFFF;
  constexpr int kMost = 1 << 24;
  int score = 0;  // quarters of a microsecond and CTA
  bool large = false;
  for (int r = lane; r < p.R; r += 32) {
    const PagedRequest q = paged_rows(p, paged_raw(p, r));
    large |= q.rows > kPagedMidRows;
    if (q.rows <= kPagedRows || q.rows > kPagedMidRows) continue;
    const int64_t units = static_cast<int64_t>(p.Hkv) * ((q.kv + kKeys - 1) / kKeys);
    const int tiles = (q.rows + kPagedRows - 1) / kPagedRows;
    score = static_cast<int>(min(score + units * (6 * tiles - 7), static_cast<int64_t>(kMost)));
  }
  if (__any_sync(0xFFFFFFFFu, large)) return kPagedRows;
  return __reduce_add_sync(0xFFFFFFFFu, score) < kPagedMidScore ? kPagedMidRows : kPagedRows;
}

template <int kKeys>
__device__ __forceinline__ PagedRequest paged_request(const PagedAttnParams& p, int split, const PagedRaw& x, int r) {
  PagedRequest q = paged_rows(p, x);
  q.tiles = r < p.R && q.rows > split ? 0 : (q.rows + kPagedRows - 1) / kPagedRows;
  q.nb = max(1, (q.kv + kKeys - 1) / kKeys);
  return q;
}

// An item's share of the list, and a request's.
__device__ __forceinline__ int item_cost(const PagedAttnParams& p, int nb) {
  return ((nb + kPagedItemCost - 1) >> p.cost_shift) + 1;
}
template <int kKeys>
__device__ __forceinline__ int paged_cost(const PagedAttnParams& p, int split, int r, bool& bad) {
  if (r > p.R) return 0;
  const PagedRaw x = paged_raw(p, r);
  bad |= paged_offsets_bad(x, r);
  const PagedRequest q = paged_request<kKeys>(p, split, x, r);
  return q.tiles * p.Hkv * item_cost(p, q.nb);
}

__device__ __forceinline__ int warp_scan(int x, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xFFFFFFFFu, x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// The list of items, as one warp sees it: the first 32 requests' costs stay in
// its lanes, later ones are read again. (Everything that a CTA does before its
// first load is done with few instructions, in 32 bits: they are fetched cold,
// and that took longer than the loads.)
template <int kKeys>
struct PagedList {
  const PagedAttnParams& p;
  int split, lane;
  int own, upto;  // cost of request `lane`, and with all before it
  bool bad = false;
  __device__ __forceinline__ PagedList(const PagedAttnParams& p_, int split_, int lane_)
      : p(p_), split(split_), lane(lane_) {
    own = paged_cost<kKeys>(p, split, lane, bad);
    upto = warp_scan(own, lane);
  }
  // Its length; 0, and a device error, where the offsets are bad.
  __device__ __forceinline__ int total() {
    unsigned n = own;
    for (int r = lane + 32; r <= p.R; r += 32) n += paged_cost<kKeys>(p, split, r, bad);
    n = __reduce_add_sync(0xFFFFFFFFu, n);
    if (!__any_sync(0xFFFFFFFFu, bad)) return static_cast<int>(n);
    if (blockIdx.x == 0 && threadIdx.x == 0) raise_device_error(HSPMN_DEVERR_POSITION);
    return 0;
  }
  // The request that holds list place w (below the total) and the cost before it.
  __device__ __forceinline__ int locate(int w, int& before) {
    int base = 0, mine = own, sum = upto;
    for (int r0 = 0; r0 <= p.R; r0 += 32) {
      if (r0 > 0) mine = paged_cost<kKeys>(p, split, r0 + lane, bad), sum = warp_scan(mine, lane);
      const unsigned past = __ballot_sync(0xFFFFFFFFu, base + sum > w);
      if (past) {
        const int l = __ffs(past) - 1;
        before = base + __shfl_sync(0xFFFFFFFFu, sum - mine, l);
        return r0 + l;
      }
      base += __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    before = base;
    return p.R;  // not reached for w below the total
  }
};

// A list of `total` units cut into n runs whose lengths differ by one at most.
struct Runs {
  int share, rem, n;
  __device__ __forceinline__ Runs(int total, int runs) {
    n = runs;
    share = static_cast<int>(static_cast<unsigned>(total) / static_cast<unsigned>(runs));
    rem = total - share * runs;
  }
  __device__ __forceinline__ int start(int c) const { return share * c + min(c, rem); }
  // The run that holds unit u.
  __device__ __forceinline__ int of(int u) const {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start(mid) <= u) lo = mid;
      else hi = mid;
    }
    return lo;
  }
};

// A unit of a run: request, row tile, head and key unit. The next request is
// read ahead, so that coming to it costs no wait.
template <int kKeys>
struct PagedCursor {
  PagedRequest req;
  PagedRaw ahead;
  int split, r, tile, head;
  int j, jend;  // unit, and the end of this run's units of the item
  int a, end;   // the item's place in the list, the run's end
  // The item's unit at list place w: an item's fixed cost comes before its units.
  __device__ __forceinline__ int unit_at(const PagedAttnParams& p, int w) const {
    return min(max((min(w - a, item_cost(p, req.nb)) << p.cost_shift) - kPagedItemCost, 0), req.nb);
  }
  // To the run [w0, w1), whose start lies in request `request` with `before` before it.
  __device__ __forceinline__ void open(const PagedAttnParams& p, int split_, int request, int before, int w0, int w1) {
    split = split_;
    r = request;
    req = paged_request<kKeys>(p, split, paged_raw(p, r), r);
    ahead = paged_raw(p, r + 1);
    const unsigned cost = item_cost(p, req.nb), item = static_cast<unsigned>(w0 - before) / cost;
    tile = static_cast<int>(item / static_cast<unsigned>(p.Hkv));
    head = static_cast<int>(item) - tile * p.Hkv;
    a = before + static_cast<int>(item * cost);
    end = w1;
    j = unit_at(p, w0);
    jend = unit_at(p, w1);
  }
  __device__ __forceinline__ bool valid() const { return j < jend; }
  // Whether the run ends in front of the first unit of the item behind this one.
  __device__ __forceinline__ bool last_item(const PagedAttnParams& p) const {
    return end - a - item_cost(p, req.nb) <= kPagedItemCost >> p.cost_shift;
  }
  // To the run's next unit, if there is one (valid() tells).
  __device__ __forceinline__ void next(const PagedAttnParams& p) {
    if (++j < jend) return;
    if (last_item(p)) {
      jend = 0;
      return;
    }
    a += item_cost(p, req.nb);
    j = 0;
    if (++head == p.Hkv) {
      head = 0;
      if (++tile == req.tiles) {
        tile = 0;
        do {
          req = paged_request<kKeys>(p, split, ahead, ++r);
          ahead = paged_raw(p, r + 1);
        } while (req.tiles == 0 && r < p.R);
      }
    }
    jend = unit_at(p, end);
  }
};

// Byte offset of query row `row` (q0 * G + ...) of K/V head `head`.
__device__ __forceinline__ int64_t paged_row(int q0, int row, int head, int G, int64_t sn, int64_t sh) {
  const int qi = row / G;
  return (static_cast<int64_t>(q0) + qi) * sn + static_cast<int64_t>(head * G + (row - qi * G)) * sh;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool full) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// c += a b, 16 x 8 x 16, fp32 accumulation.
template <bool kBF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Whether a 32-bit word of two 16-bit elements holds an infinity or a NaN.
template <bool kBF16>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  constexpr uint32_t e = kBF16 ? 0x7F80u : 0x7C00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

// The word with infinities and NaN replaced by zero.
template <bool kBF16>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  constexpr uint32_t e = kBF16 ? 0x7F80u : 0x7C00u;
  if ((w & e) == e) w &= 0xFFFF0000u;
  if (((w >> 16) & e) == e) w &= 0x0000FFFFu;
  return w;
}

template <bool kBF16>
__device__ __forceinline__ float half_to_float(uint16_t h) {
  if constexpr (kBF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  else return __half2float(__ushort_as_half(h));
}

template <int HD>
struct PagedLayout {
  static constexpr int kRow = HD * 2;                             // bytes of a key's K or V in shared memory
  static constexpr int kWarpKeys = HD == 64 ? 32 : 16;            // a warp's keys of a unit: 8 KB of K and V
  static constexpr int kKeys = kPagedWarps * kWarpKeys;
  static constexpr int kWarpStage = 2 * kWarpKeys * kRow;
  static constexpr int kStage = kPagedWarps * kWarpStage;
  static constexpr int kQSlot = kPagedRows * HD * 2;              // a tile's query rows
  static constexpr int kQOff = kPagedStages * kStage;
  static constexpr int kBytes = kQOff + kPagedStages * kQSlot;
  // at the end of an item a warp leaves its 16 x HD fp32 O in the stage it has just consumed
  static_assert(kWarpStage >= kPagedRows * HD * 4, "an O tile fits a warp's stage");
};

// Word index of O element (row, col) in a warp's stage: 8-column groups are
// permuted by the row so the accumulator layout's writes spread over the banks.
template <int HD>
__device__ __forceinline__ int paged_o_word(int row, int col) {
  return row * HD + ((((col >> 3) ^ row) & (HD / 8 - 1)) << 3) + (col & 7);
}

template <int HD, bool kBF16>
__global__ void __launch_bounds__(kPagedThreads, kPagedCtasPerSm) paged_attn_kernel(const PagedAttnParams p) {
  using L = PagedLayout<HD>;
  extern __shared__ __align__(128) uint8_t paged_smem[];
  __shared__ float s_m[kPagedWarps][kPagedRows], s_l[kPagedWarps][kPagedRows];
  __shared__ __align__(8) int64_t s_pos[kPagedStages][kPagedRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t2 = (lane & 3) * 2;  // accumulator row and first column of this lane
  // the chunk kernel in front of this one has entered: see grid_dependency_enter
  if (p.has_chunks) grid_dependency_behind();
  else grid_dependency_enter();
  const int split = paged_split<L::kKeys>(p, lane);
  PagedList<L::kKeys> list(p, split, lane);
  const int total = list.total();
  const int runs = min(static_cast<int>(gridDim.x), total);
  PagedCursor<L::kKeys> cur, ahead;
  const Runs run(total, max(runs, 1));
  if (static_cast<int>(blockIdx.x) < runs) {
    const int w0 = run.start(blockIdx.x), w1 = run.start(blockIdx.x + 1);
    int before;
    const int r0 = list.locate(w0, before);
    cur.open(p, split, r0, before, w0, w1);
  } else {
    cur.j = cur.jend = 0;
  }
  if (!cur.valid()) {
    if (threadIdx.x == 0) p.merges[blockIdx.x] = make_int4(0, 0, 0, -1);
    grid_dependency_wait();
    return;
  }
  ahead = cur;
  const uint32_t wbase = smem_u32(paged_smem) + warp * L::kWarpStage;
  constexpr int kChunks = HD / 8;           // 16-byte chunks of a row
  constexpr int kPerIter = 32 / kChunks;    // rows a warp-wide copy covers
  const int ld_row = lane / kChunks, ld_chunk = lane % kChunks;
  const bool ld_col = ld_chunk * 8 < p.hd;  // columns past head_dim are zero

  constexpr int kGroups = L::kWarpKeys / 8;  // of 8 keys: each lies in one page
  const int mask = (1 << p.shift) - 1;
  uint32_t gone_ring = 0;  // kGroups bits a stage: the group's page does not exist

  // With an item's first unit come its query rows (a quarter a warp) and their
  // positions, into slot q_ahead.
  const uint32_t qbase = smem_u32(paged_smem) + L::kQOff;
  int q_ahead = 0, q_cur = 0;
  auto request_rows = [&]() {
#pragma unroll
    for (int i = 0; i < 4 / kPerIter; ++i) {
      const int lr = warp * 4 + i * kPerIter + ld_row, row = ahead.tile * kPagedRows + lr;
      const bool there = row < ahead.req.rows && ld_col;
      const char* src = p.q + paged_row(ahead.req.q0, there ? row : 0, ahead.head, p.G, p.q_sn, p.q_sh) +
                        (there ? ld_chunk * 16 : 0);
      cp_async16(qbase + q_ahead * L::kQSlot + lr * L::kRow + ((ld_chunk ^ (lr & 7)) << 4), src, there);
    }
    const int row = ahead.tile * kPagedRows + lane;
    if (warp == 0 && lane < kPagedRows && row < ahead.req.rows)
      cp_async8(smem_u32(&s_pos[q_ahead][lane]), p.pos + ahead.req.q0 + row / p.G);
    q_ahead = q_ahead + 1 == kPagedStages ? 0 : q_ahead + 1;
  };
  // This warp's keys of the unit `ahead` points at, into ring stage s. Keys past
  // the visible range or in a page that does not exist arrive as zeros: no byte
  // is read for them.
  const int ld_byte = ld_col ? ld_chunk * 16 : 0;
  const uint32_t ld_dst = ld_row * L::kRow;
  auto request = [&](int s) {
    const int key0 = ahead.j * L::kKeys + warp * L::kWarpKeys, left = ahead.req.kv - key0;
    const uint32_t kdst = wbase + s * L::kStage + ld_dst, vdst = kdst + L::kWarpKeys * L::kRow;
    const int* row = p.table + static_cast<int64_t>(ahead.r) * p.table_rs;
    const char* kh = p.k + static_cast<int64_t>(ahead.head) * p.k_sh + ld_byte;
    const char* vh = p.v + static_cast<int64_t>(ahead.head) * p.v_sh + ld_byte;
    int page[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) page[i] = 8 * i < left ? row[(key0 + 8 * i) >> p.shift] : 0;
    uint32_t gone = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) gone |= (static_cast<unsigned>(page[i]) >= static_cast<unsigned>(p.num_pages) ? 1u : 0u) << i;
    const bool full = left >= L::kWarpKeys && gone == 0 && p.hd == HD;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const unsigned pg = gone >> i & 1 ? 0u : static_cast<unsigned>(page[i]);
      const unsigned off = ((key0 + 8 * i) & mask) + ld_row;
      const char* ks = kh + static_cast<uint64_t>(pg) * p.k_sp + static_cast<uint64_t>(off) * p.k_ss;
      const char* vs = vh + static_cast<uint64_t>(pg) * p.v_sp + static_cast<uint64_t>(off) * p.v_ss;
      const int rows = gone >> i & 1 || !ld_col ? 0 : left - 8 * i - ld_row;  // rows from here on that count
#pragma unroll
      for (int x = 0; x < 8 / kPerIter; ++x) {
        const int kr = 8 * i + x * kPerIter;
        const uint32_t d = kr * L::kRow + ((ld_chunk ^ ((kr & 7) + ld_row)) << 4);
        if (full) {
          cp_async16(kdst + d, ks);
          cp_async16(vdst + d, vs);
        } else {
          cp_async16(kdst + d, ks, x * kPerIter < rows);
          cp_async16(vdst + d, vs, x * kPerIter < rows);
        }
        ks += kPerIter * p.k_ss, vs += kPerIter * p.v_ss;
      }
    }
    if (gone && lane == 0) raise_device_error(HSPMN_DEVERR_PAGE);
    gone_ring = (gone_ring & ~(((1u << kGroups) - 1) << (kGroups * s))) | gone << (kGroups * s);
  };

#pragma unroll
  for (int s = 0; s < kPagedStages - 1; ++s) {
    if (ahead.valid()) {
      if (s == 0 || ahead.j == 0) request_rows();
      request(s);
      ahead.next(p);
    }
    cp_async_commit();
  }

  uint32_t qa[HD / 16][4];
  float acc[HD / 8][4];
  float m_run[2] = {}, l_run[2] = {};
  bool seen[2] = {};  // the row has met a key that it sees
  int lim[2] = {}, lim_min = 0, lim_max = 0;
  bool fresh = true;  // the next unit opens an item (or this run's part of one)
  int seg_j = 0;      // the part's first unit
  int stage = 0;
  while (cur.valid()) {
    cp_async_wait<kPagedStages - 2>();
    if (fresh) {
      // every warp's share of the query rows has arrived, and every warp has
      // left the item before (its O in a stage, its maxima and sums)
      __syncthreads();
      fresh = false;
      seg_j = cur.j;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const int lr = (lane & 7) + (((lane >> 3) & 1) << 3), chunk = kk * 2 + (lane >> 4);
        ldmatrix_x4(qa[kk], qbase + q_cur * L::kQSlot + lr * L::kRow + ((chunk ^ (lr & 7)) << 4));
      }
      // the last key that each row sees
      lim_min = 0x7FFFFFFF;
      lim_max = -1;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lim[i] = -1;
        if (cur.tile * kPagedRows + g + 8 * i < cur.req.rows) {
          const int64_t ps = s_pos[q_cur][g + 8 * i];
          if (ps >= cur.req.kv && cur.r < p.R) raise_device_error(HSPMN_DEVERR_POSITION);
          lim[i] = static_cast<int>(min(max(ps, static_cast<int64_t>(-1)), static_cast<int64_t>(cur.req.kv) - 1));
          if (lim[i] >= 0) lim_min = min(lim_min, lim[i]);
          lim_max = max(lim_max, lim[i]);
        }
        m_run[i] = -INFINITY;
        l_run[i] = 0.0f;
        seen[i] = false;
      }
      lim_min = __reduce_min_sync(0xFFFFFFFFu, lim_min);
      lim_max = __reduce_max_sync(0xFFFFFFFFu, lim_max);
      q_cur = q_cur + 1 == kPagedStages ? 0 : q_cur + 1;
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
    } else {
      __syncwarp();
    }
    const int key0 = cur.j * L::kKeys + warp * L::kWarpKeys;
    const uint32_t kst = wbase + stage * L::kStage, vst = kst + L::kWarpKeys * L::kRow;
    if (key0 <= lim_max) {
      // S = Q K^T, 16 rows by the warp's keys, in 8-key tiles
      float s[kGroups][4] = {};
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const int chunk = kk * 2 + ((lane >> 3) & 1);
#pragma unroll
        for (int n = 0; n < kGroups; n += 2) {
          const int kr = n * 8 + ((lane >> 4) << 3) + (lane & 7);
          uint32_t b[4];
          ldmatrix_x4(b, kst + kr * L::kRow + ((chunk ^ (kr & 7)) << 4));
          mma16816<kBF16>(s[n], qa[kk], b[0], b[1]);
          mma16816<kBF16>(s[n + 1], qa[kk], b[2], b[3]);
        }
      }
      const uint32_t gone = (gone_ring >> (kGroups * stage)) & ((1u << kGroups) - 1);
      const bool masked = key0 + L::kWarpKeys - 1 > lim_min || gone != 0;
      if (masked) {
#pragma unroll
        for (int n = 0; n < kGroups; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 8 * n + t2 + (e & 1);
            if (key > lim[e >> 1] || (gone >> n & 1)) s[n][e] = -INFINITY;
          }
      }
      // online softmax of rows g and g + 8
      float alpha[2];
      bool grew = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = fmaxf(s[0][2 * i], s[0][2 * i + 1]);
#pragma unroll
        for (int n = 1; n < kGroups; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
        const float m_new = fmaxf(m_run[i], mx);
        alpha[i] = m_new > m_run[i] ? fast_exp2((m_run[i] - m_new) * p.scale_log2) : 1.0f;
        grew |= m_new > m_run[i];
        const float base = m_new == -INFINITY ? 0.0f : m_new;
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float e = fast_exp2((s[n][2 * i + c] - base) * p.scale_log2);
            s[n][2 * i + c] = e;
            sum += e;
          }
          seen[i] |= key0 + 8 * n <= lim[i] && !(gone >> n & 1);
        }
        l_run[i] = l_run[i] * alpha[i] + sum;
        m_run[i] = m_new;
      }
      if (__any_sync(0xFFFFFFFFu, grew)) {
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          acc[n][0] *= alpha[0], acc[n][1] *= alpha[0];
          acc[n][2] *= alpha[1], acc[n][3] *= alpha[1];
        }
      }
      // Where some row sees a key and another does not, an infinity or NaN in
      // that key's V must not reach the other (0 * inf): such a step adds its
      // products one by one (with P as it is: no operand to round it for).
      bool wild = false;
      if (masked) {
        bool mine = false;
#pragma unroll
        for (int i = 0; i < L::kWarpKeys / kPerIter; ++i) {
          const int kr = i * kPerIter + ld_row;
          uint4 w;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                       : "r"(vst + kr * L::kRow + ((ld_chunk ^ (kr & 7)) << 4)));
          mine |= not_finite2<kBF16>(w.x) || not_finite2<kBF16>(w.y) || not_finite2<kBF16>(w.z) ||
                  not_finite2<kBF16>(w.w);
        }
        wild = __any_sync(0xFFFFFFFFu, mine);
      }
      if (!wild) {
#pragma unroll
        for (int k = 0; k < kGroups; k += 2) {
          // P in the operands' type: its rounding (half a step) is of the size of
          // the output's own. (A second product with what the rounding leaves took
          // the error to the output's alone, and 6 % more time for 64 requests.)
          const uint32_t pa[4] = {pack2<kBF16>(s[k][0], s[k][1]), pack2<kBF16>(s[k][2], s[k][3]),
                                  pack2<kBF16>(s[k + 1][0], s[k + 1][1]), pack2<kBF16>(s[k + 1][2], s[k + 1][3])};
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            const int kr = k * 8 + (((lane >> 3) & 1) << 3) + (lane & 7), chunk = n * 2 + (lane >> 4);
            uint32_t b[4];
            ldmatrix_x4_trans(b, vst + kr * L::kRow + ((chunk ^ (kr & 7)) << 4));
            mma16816<kBF16>(acc[2 * n], pa, b[0], b[1]);
            mma16816<kBF16>(acc[2 * n + 1], pa, b[2], b[3]);
          }
        }
      } else {
#pragma unroll
        for (int k8 = 0; k8 < kGroups; ++k8) {
#pragma unroll 1
          for (int kr = 0; kr < 8; ++kr) {
            const int src = (lane & ~3) | (kr >> 1);  // the lane of this quad that holds the key's column
            float w[2];
            bool sees[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              w[i] = __shfl_sync(0xFFFFFFFFu, kr & 1 ? s[k8][2 * i + 1] : s[k8][2 * i], src);
              sees[i] = key0 + 8 * k8 + kr <= lim[i] && !(gone >> k8 & 1);
            }
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
              uint32_t two;
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(two) : "r"(vst + (8 * k8 + kr) * L::kRow + ((n ^ kr) << 4) + t2 * 2));
              const float x = half_to_float<kBF16>(static_cast<uint16_t>(two)), y = half_to_float<kBF16>(two >> 16);
#pragma unroll
              for (int i = 0; i < 2; ++i)
                if (sees[i]) acc[n][2 * i] = fmaf(w[i], x, acc[n][2 * i]), acc[n][2 * i + 1] = fmaf(w[i], y, acc[n][2 * i + 1]);
            }
          }
        }
      }
    }
    if (cur.j + 1 == cur.jend) {
      // the warps' results of this item: O in the stage each has just
      // consumed, maxima and sums beside it
      __syncwarp();
      float* mine = reinterpret_cast<float*>(paged_smem + warp * L::kWarpStage + stage * L::kStage);
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<float2*>(mine + paged_o_word<HD>(g + 8 * i, n * 8 + t2)) =
              make_float2(acc[n][2 * i], acc[n][2 * i + 1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float l = l_run[i];
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
        if ((lane & 3) == 0) s_m[warp][g + 8 * i] = m_run[i], s_l[warp][g + 8 * i] = seen[i] ? l : kUnseen;
      }
      const bool item_end = cur.jend == cur.req.nb, whole = item_end && seg_j == 0;
      // the last item of this run: if it goes on behind it, its runs from the one
      // in which it opens to this one share its merge
      if (threadIdx.x == 0 && (!item_end || cur.last_item(p))) {
        const int first = run.of(cur.a + (kPagedItemCost >> p.cost_shift));
        const int last = run.of(cur.a + ((kPagedItemCost + cur.req.nb - 1) >> p.cost_shift));
        p.merges[blockIdx.x] =
            make_int4(cur.req.q0, cur.tile * kPagedRows,
                      cur.head * kPagedRows + min(kPagedRows, cur.req.rows - cur.tile * kPagedRows) - 1,
                      item_end ? -1 : first << 16 | last);
      }
      __syncthreads();
      // a run holds the last piece of one item at most, and the first of one
      const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (seg_j == 0 ? 1 : 0);
      constexpr int kQuads = HD / 4;  // 4-column groups of a row
      for (int i = threadIdx.x; i < kPagedRows * kQuads; i += kPagedThreads) {
        const int lr = i / kQuads, c = (i % kQuads) * 4;
        const int row = cur.tile * kPagedRows + lr;
        if (row >= cur.req.rows || c >= p.hd) continue;
        float M = s_m[0][lr];
#pragma unroll
        for (int w = 1; w < kPagedWarps; ++w) M = fmaxf(M, s_m[w][lr]);
        float l = 0.0f;
        bool none = true;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) {
          if (s_l[w][lr] == kUnseen) continue;
          none = false;
          const float mw = s_m[w][lr], f = mw == M ? 1.0f : fast_exp2((mw - M) * p.scale_log2);
          const float4 x = *reinterpret_cast<const float4*>(
              reinterpret_cast<const float*>(paged_smem + w * L::kWarpStage + stage * L::kStage) +
              paged_o_word<HD>(lr, c));
          l += f * s_l[w][lr];
          o.x += f * x.x, o.y += f * x.y, o.z += f * x.z, o.w += f * x.w;
        }
        if (whole) {
          const float inv = 1.0f / l;
          uint2 w;
          w.x = none ? 0u : pack2<kBF16>(o.x * inv, o.y * inv);
          w.y = none ? 0u : pack2<kBF16>(o.z * inv, o.w * inv);
          *reinterpret_cast<uint2*>(p.o + paged_row(cur.req.q0, row, cur.head, p.G, p.o_sn, p.o_sh) + c * 2) = w;
        } else {
          *reinterpret_cast<float4*>(p.part_o + (slot * kPagedRows + lr) * HD + c) = o;
          if (c == 0) reinterpret_cast<float2*>(p.part_ml)[slot * kPagedRows + lr] = make_float2(M, none ? kUnseen : l);
        }
      }
      fresh = true;
    }
    // refill the stage that the unit before this one has left
    __syncwarp();
    if (ahead.valid()) {
      if (ahead.j == 0) request_rows();
      request((stage + kPagedStages - 1) % kPagedStages);
      ahead.next(p);
    }
    cp_async_commit();
    stage = stage + 1 == kPagedStages ? 0 : stage + 1;
    cur.next(p);
  }
  cp_async_wait<0>();
  // the kernel before (the chunks' one, or the caller's) is not needed here, but
  // what comes next counts on it when this grid has ended
  grid_dependency_wait();
}

constexpr int kMergeWarps = 16;

// Adds the partial results of the item that goes on behind run `block`, as that
// run noted: O = sum w_c O_c / sum w_c l_c, w_c = 2^(scale_log2 (m_c - M)), over the
// item's runs in order. All runs it goes on behind share its rows; a warp takes a row and a
// share of the runs.
template <int HD, bool kBF16>
__device__ __forceinline__ void paged_merge(const PagedAttnParams& p, int block) {
  __shared__ float4 s_o[kMergeWarps][HD / 4];
  __shared__ float2 s_ml[kMergeWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 note = p.merges[block];
  if (note.w < 0) return;
  const int c0 = note.w >> 16, c1 = note.w & 0xFFFF;
  const int rows = note.z % kPagedRows + 1, head = note.z / kPagedRows;
  const int blocks = min(rows, c1 - c0), slice = block - c0;
  if (slice >= blocks) return;
  const int mine = (rows - slice + blocks - 1) / blocks;  // rows slice, slice + blocks, ..
  const int shares = kMergeWarps / mine;                  // warps of a row
  const int part = warp % shares, lr = slice + warp / shares * blocks;
  const bool live = warp / shares < mine;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  float M = -INFINITY, l = 0.0f;
  bool none = true;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (live) {
    const int per = (c1 - c0 + shares) / shares, lo = c0 + part * per, hi = min(c1 + 1, lo + per);
#pragma unroll 4
    for (int c = lo; c < hi; ++c) {
      // run c0's piece is its last, the others' their first
      const int64_t s = (2 * static_cast<int64_t>(c) + (c == c0 ? 1 : 0)) * kPagedRows + lr;
      const float2 x = ml[s];
      const float4 v = lane < HD / 4 ? *reinterpret_cast<const float4*>(p.part_o + s * HD + lane * 4)
                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (x.y == kUnseen) continue;
      none = false;
      const float top = fmaxf(M, x.x);
      const float f = x.x == top ? 1.0f : fast_exp2((x.x - top) * p.scale_log2);
      const float g = M == top ? 1.0f : fast_exp2((M - top) * p.scale_log2);
      M = top;
      l = g * l + f * x.y;
      o.x = g * o.x + f * v.x, o.y = g * o.y + f * v.y, o.z = g * o.z + f * v.z, o.w = g * o.w + f * v.w;
    }
  }
  if (lane < HD / 4) s_o[warp][lane] = o;
  if (lane == 0) s_ml[warp] = make_float2(M, none ? kUnseen : l);
  __syncthreads();
  if (!live || part != 0) return;
  float top = -INFINITY, sum = 0.0f;
  bool empty = true;
  for (int w = warp; w < warp + shares; ++w)
    if (s_ml[w].y != kUnseen) top = fmaxf(top, s_ml[w].x);
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int w = warp; w < warp + shares; ++w) {
    const float2 x = s_ml[w];
    if (x.y == kUnseen) continue;
    empty = false;
    const float f = x.x == top ? 1.0f : fast_exp2((x.x - top) * p.scale_log2);
    sum += f * x.y;
    if (lane < HD / 4) {
      const float4 v = s_o[w][lane];
      y.x += f * v.x, y.y += f * v.y, y.z += f * v.z, y.w += f * v.w;
    }
  }
  const float inv = 1.0f / sum;
  if (lane * 4 < p.hd && lane < HD / 4) {
    uint2 w;
    w.x = empty ? 0u : pack2<kBF16>(y.x * inv, y.y * inv);
    w.y = empty ? 0u : pack2<kBF16>(y.z * inv, y.w * inv);
    *reinterpret_cast<uint2*>(p.o + paged_row(note.x, note.y + lr, head, p.G, p.o_sn, p.o_sh) + lane * 8) = w;
  }
}

template <int HD, bool kBF16>
__global__ void __launch_bounds__(32 * kMergeWarps) paged_merge_kernel(const __grid_constant__ PagedAttnParams p) {
  grid_dependency_enter();
  paged_merge<HD, kBF16>(p, static_cast<int>(blockIdx.x));
}

}  // namespace hspmn
