// Paged K/V cache: page and slot bookkeeping, and the cache write with the
// rotary embedding of K. The attention that reads the cache is paged_attn.cuh.
//
// A cache is [num_pages, page_size, Hkv, hd]; token `pos` of request r lives in
// page block_table[r, pos / page_size] at offset pos % page_size, and its slot
// is page * page_size + offset. page_size is a power of two.
#pragma once

#include "rows.cuh"

namespace hspmn {

constexpr int kSlotsThreads = 256;
constexpr int kSlotsWarps = kSlotsThreads / 32;
constexpr int kSlotsMaxRequests = 8192;  // two prefix arrays of 4 bytes a request fit in shared memory

// Largest i in [0, n) with pre[i] <= x, for an ascending pre with pre[0] <= x
// (entries that repeat: the last one, i.e. the request that owns x).
__device__ __forceinline__ int last_not_above(const int* pre, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct SlotsParams {
  int* table;  // [R,P], row stride table_rs
  int64_t table_rs;
  const int* seq_lens;
  const int* new_lens;
  const int* free_pages;
  int R, P, F, shift;
  int64_t N;
  int* cu;         // [R+1]
  int* kv_lens;    // [R]
  int64_t* pos;    // [N]
  int64_t* slots;  // [N]
  int* taken;      // [1]
};

// Sum of two counts, held at the largest int (the result of a call whose
// lengths add up to more than that is flagged, and stays in bounds).
__device__ __forceinline__ int add_held(int a, int b) {
  const int s = static_cast<int>(static_cast<unsigned>(a) + static_cast<unsigned>(b));
  return s < 0 ? 0x7FFFFFFF : s;
}

// Pages that hold the first `len` tokens, at most the table's width.
__device__ __forceinline__ int pages_of(int64_t len, int shift, int P) {
  const int64_t n = (len + (1 << shift) - 1) >> shift;
  return static_cast<int>(n < P ? n : P);
}

// Every CTA scans the R lengths (a few loads a thread) into two shared prefix
// arrays, tokens and fresh pages, and then takes its share of the fresh table
// entries and of the tokens; each finds its request by binary search in shared
// memory. No CTA reads what another writes: a token in a fresh page takes the
// page from the free list, a token in an older page from the part of the table
// that nobody writes. Latency bound: one launch and two dependent rounds of
// loads, 3.3 us for 64 requests of one token; 6.5 us for 509 prompts of 1 to 4096
// tokens (251,500 in all, 4 MB).
__global__ void __launch_bounds__(kSlotsThreads) paged_slots_kernel(const SlotsParams p) {
  extern __shared__ int slots_smem[];
  int* s_tok = slots_smem;               // [R+1]
  int* s_page = slots_smem + (p.R + 1);  // [R+1]
  __shared__ int2 warp_sum[kSlotsWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dependency_enter();
  int2 carry = make_int2(0, 0);
  bool bad = false;
  if (threadIdx.x == 0) s_tok[0] = s_page[0] = 0;
  for (int base = 0; base < p.R; base += kSlotsThreads) {
    const int r = base + static_cast<int>(threadIdx.x);
    int2 v = make_int2(0, 0);
    if (r < p.R) {
      const int c = p.seq_lens[r], m = p.new_lens[r];
      bad |= c < 0 || m < 0;
      const int64_t c0 = max(c, 0), kv = c0 + max(m, 0);
      v.x = max(m, 0);
      v.y = pages_of(kv, p.shift, p.P) - pages_of(c0, p.shift, p.P);
      bad |= kv > (static_cast<int64_t>(p.P) << p.shift);
      if (blockIdx.x == 0) p.kv_lens[r] = static_cast<int>(kv < 0x7FFFFFFF ? kv : 0x7FFFFFFF);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xFFFFFFFFu, v.x, d), y = __shfl_up_sync(0xFFFFFFFFu, v.y, d);
      if (lane >= d) v.x = add_held(v.x, x), v.y += y;
    }
    __syncthreads();  // the previous round's warp sums have been read
    if (lane == 31) warp_sum[warp] = v;
    __syncthreads();
    int2 before = carry;
#pragma unroll
    for (int w = 0; w < kSlotsWarps; ++w) {
      const int2 t = warp_sum[w];
      if (w < warp) before.x = add_held(before.x, t.x), before.y += t.y;
      carry.x = add_held(carry.x, t.x), carry.y += t.y;
    }
    if (r < p.R) s_tok[r + 1] = add_held(before.x, v.x), s_page[r + 1] = before.y + v.y;
  }
  __syncthreads();
  const int total = s_tok[p.R], fresh = s_page[p.R];
  const int64_t tid = static_cast<int64_t>(blockIdx.x) * kSlotsThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kSlotsThreads;
  if (blockIdx.x == 0) {
    for (int r = threadIdx.x; r <= p.R; r += kSlotsThreads) p.cu[r] = s_tok[r];
    if (threadIdx.x == 0) *p.taken = fresh;
    if (bad || (threadIdx.x == 0 && total > p.N)) raise_device_error(HSPMN_DEVERR_POSITION);
    if (threadIdx.x == 0 && fresh > p.F) raise_device_error(HSPMN_DEVERR_PAGE);
  }
  for (int64_t j = tid; j < fresh; j += step) {
    const int r = last_not_above(s_page, p.R, static_cast<int>(j));
    const int col = pages_of(max(p.seq_lens[r], 0), p.shift, p.P) + static_cast<int>(j) - s_page[r];
    if (col < p.P) p.table[r * p.table_rs + col] = j < p.F ? p.free_pages[j] : -1;
  }
  const int mask = (1 << p.shift) - 1;
  for (int64_t t = tid; t < p.N; t += step) {
    int64_t pos = -1, slot = -1;
    if (t < total) {
      const int r = last_not_above(s_tok, p.R, static_cast<int>(t));
      const int64_t c0 = max(p.seq_lens[r], 0);
      pos = c0 + t - s_tok[r];
      const int64_t col = pos >> p.shift;
      const int held = pages_of(c0, p.shift, p.P);
      int page = -1;
      if (col < held) page = p.table[r * p.table_rs + col];
      else if (col < p.P && s_page[r] + (col - held) < p.F) page = p.free_pages[s_page[r] + (col - held)];
      if (page >= 0) slot = (static_cast<int64_t>(page) << p.shift) + (pos & mask);
      else if (col < held) raise_device_error(HSPMN_DEVERR_PAGE);  // (the other causes are flagged above)
    }
    p.pos[t] = pos;
    p.slots[t] = slot;
  }
}

// ---------------------------------------------------------------------------
// cache write
// ---------------------------------------------------------------------------

struct PagedWriteParams {
  const char* k;
  const char* v;
  int64_t k_sn, k_sh, v_sn, v_sh;  // bytes
  const char* cos_tab;             // null: K is stored as it is
  const char* sin_tab;
  int64_t tab_ss, tab_rows;  // bytes, rows
  const int64_t* pos;
  const int64_t* slots;
  char* kc;
  char* vc;
  int64_t kc_sp, kc_ss, kc_sh, vc_sp, vc_ss, vc_sh;  // bytes: page, slot in the page, head
  int64_t N, num_pages;
  int shift, Hkv, hd;
};

template <typename T>
__device__ __forceinline__ float elt_to_float(T x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(x);
  else return __bfloat162float(x);
}

template <typename T>
__device__ __forceinline__ T float_to_elt(float x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

// n consecutive table entries as floats (n * sizeof(Tab) is 16 or 32 bytes)
template <typename Tab, int n>
__device__ __forceinline__ void load_table(const char* p, float (&out)[n]) {
  constexpr int per = 16 / sizeof(Tab);
#pragma unroll
  for (int i = 0; i < n / per; ++i) {
    const uint4 w = reinterpret_cast<const uint4*>(p)[i];
    const Tab* e = reinterpret_cast<const Tab*>(&w);
#pragma unroll
    for (int j = 0; j < per; ++j) out[i * per + j] = elt_to_float(e[j]);
  }
}

// kLanes lanes a token (the smallest power of two from 8 to 32 that gives each one
// K unit, where 32 are enough): lanes take the K row in pairs of 16-byte groups
// (a group of a head's low half and its partner in the high half, so x and the
// tables are read once per pair) and the V row in 16-byte groups. The rotation is
// formed in fp32 and rounded once, when it is stored. The slot and position of a
// lane's next token are read one token ahead, and its first K pair and first two
// V groups (the whole rows up to 512 16-bit elements) together with the table
// rows, so that a token waits for memory once. HBM bound: 65,536 tokens of 4 x 128
// bf16 take 46.8 us, 5.85 TB/s (57 us when slots were read with the rows they
// send); 61 tokens take 2.4 us, the launch.
template <typename T, typename Tab, int kLanes>
__global__ void __launch_bounds__(kRowThreads) rope_paged_write_kernel(const PagedWriteParams p) {
  constexpr int n = 16 / sizeof(T);
  constexpr int kTokens = kRowThreads / kLanes;  // of a CTA at a time
  const int lane = threadIdx.x % kLanes;
  const int half = p.hd / 2;
  const bool rope = p.cos_tab != nullptr;
  const int vgroups = p.hd / n, units = p.Hkv * vgroups;  // 16-byte groups of a head, of a row
  const int pairs = half / n, kunits = rope ? p.Hkv * pairs : units;
  const int kg = rope ? pairs : vgroups;
  const int kh = lane / kg, kc = lane - kh * kg;
  const int vh0 = lane / vgroups, vc0 = lane - vh0 * vgroups;
  const int vh1 = (lane + kLanes) / vgroups, vc1 = lane + kLanes - vh1 * vgroups;
  auto source = [](const char* row, int64_t sh, int h, int c) { return reinterpret_cast<const uint4*>(row + h * sh + c * 16); };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTokens;
  grid_dependency_enter();
  int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + threadIdx.x / kLanes;
  int64_t slot = t < p.N ? p.slots[t] : -1, pos = rope && t < p.N ? p.pos[t] : 0;
  for (; t < p.N; t += step) {
    const int64_t slot_now = slot, pos_now = pos;
    if (t + step < p.N) {
      slot = p.slots[t + step];
      if (rope) pos = p.pos[t + step];
    }
    if (slot_now < 0) continue;  // padding
    const int64_t page = slot_now >> p.shift, off = slot_now & ((1 << p.shift) - 1);
    if (page >= p.num_pages || pos_now < 0 || (rope && pos_now >= p.tab_rows)) {
      if (lane == 0) raise_device_error(page >= p.num_pages ? HSPMN_DEVERR_PAGE : HSPMN_DEVERR_POSITION);
      continue;
    }
    const char* krow = p.k + t * p.k_sn;
    const char* vrow = p.v + t * p.v_sn;
    uint4 k_lo = make_uint4(0, 0, 0, 0), k_hi = k_lo, v_0 = k_lo, v_1 = k_lo;
    if (lane < kunits) {
      k_lo = __ldcs(source(krow, p.k_sh, kh, kc));
      if (rope) k_hi = __ldcs(source(krow, p.k_sh, kh, kc + pairs));
    }
    if (lane < units) v_0 = __ldcs(source(vrow, p.v_sh, vh0, vc0));
    if (lane + kLanes < units) v_1 = __ldcs(source(vrow, p.v_sh, vh1, vc1));
    char* kdst = p.kc + page * p.kc_sp + off * p.kc_ss;
    char* vdst = p.vc + page * p.vc_sp + off * p.vc_ss;
    const char* cs = p.cos_tab + pos_now * p.tab_ss;
    const char* sn = p.sin_tab + pos_now * p.tab_ss;
    for (int i = lane; i < kunits; i += kLanes) {
      const int h = i == lane ? kh : i / kg, c = i == lane ? kc : i - h * kg;
      if (i != lane) {
        k_lo = __ldcs(source(krow, p.k_sh, h, c));
        if (rope) k_hi = __ldcs(source(krow, p.k_sh, h, c + pairs));
      }
      uint4 out_lo = k_lo;
      if (rope) {
        float c_lo[n], c_hi[n], s_lo[n], s_hi[n];
        load_table<Tab, n>(cs + c * n * sizeof(Tab), c_lo);
        load_table<Tab, n>(cs + (c * n + half) * sizeof(Tab), c_hi);
        load_table<Tab, n>(sn + c * n * sizeof(Tab), s_lo);
        load_table<Tab, n>(sn + (c * n + half) * sizeof(Tab), s_hi);
        const T* lo = reinterpret_cast<const T*>(&k_lo);
        const T* hi = reinterpret_cast<const T*>(&k_hi);
        uint4 out_hi;
        T* a = reinterpret_cast<T*>(&out_lo);
        T* b = reinterpret_cast<T*>(&out_hi);
#pragma unroll
        for (int j = 0; j < n; ++j) {
          const float x = elt_to_float(lo[j]), y = elt_to_float(hi[j]);
          a[j] = float_to_elt<T>(x * c_lo[j] - y * s_lo[j]);
          b[j] = float_to_elt<T>(y * c_hi[j] + x * s_hi[j]);
        }
        __stcs(reinterpret_cast<uint4*>(kdst + h * p.kc_sh + (c + pairs) * 16), out_hi);
      }
      __stcs(reinterpret_cast<uint4*>(kdst + h * p.kc_sh + c * 16), out_lo);
    }
    if (lane < units) __stcs(reinterpret_cast<uint4*>(vdst + vh0 * p.vc_sh + vc0 * 16), v_0);
    if (lane + kLanes < units) __stcs(reinterpret_cast<uint4*>(vdst + vh1 * p.vc_sh + vc1 * 16), v_1);
    for (int i = lane + 2 * kLanes; i < units; i += kLanes) {
      const int h = i / vgroups, c = i - h * vgroups;
      __stcs(reinterpret_cast<uint4*>(vdst + h * p.vc_sh + c * 16), __ldcs(source(vrow, p.v_sh, h, c)));
    }
  }
}

}  // namespace hspmn
