// Attention over the 8-bit paged cache for many query rows, on the tcgen05 tensor
// cores (the formulas: cache_attn.cu; the softmax's references: cache_attn.cuh).
//
// A unit is one K/V head of one sequence and up to 256 rows (row r is new token
// r / group, head r % group), two M = 128 tiles; its key tiles hold 128 cached
// tokens.  The kernel is persistent, one CTA an SM, and has two streams of
//   S_h = Q K^T (M 128, N 128, K hd),  softmax,  O_h += P V (N hd, K 128 keys)
// so that one stream's products run while the other one's softmax does:
//  - a unit of more than 128 rows: a stream for each tile, sharing every key tile;
//  - otherwise: both streams have the same tile, one the even key tiles and one
//    the odd ones, each with its own reference, sum and O, which the join puts
//    together (half the time a key tile, which is what bounds few rows: a stream
//    alone takes longer over 128 keys than the SM's share of the memory does).
//
//   warps 0-3    queries to f16 (bf16 ones scaled by a power of two per row:
//                exact) and K, V codes to f16 (exact), from the ring of codes to
//                the operands' tiles in shared memory, 128-byte swizzled;
//   warp 4       tensor memory and the MMAs;
//   warp 5       TMA: K and V pages (8 KB of codes) into the ring, four ahead;
//   warps 6-13   softmax of the streams, one row a thread, and the results.
//
// Tokens past a sequence's end become zeros.  0 . NaN is NaN: in key tiles that
// some rows see only part of, NaN codes of V are taken out, and the softmax threads
// put NaN into the results of the rows that do see them.
//
// TMEM: S_h (P_h over it) at 128 h, O_h at 256 + 128 h.
//
// Bound by the softmax's chain and by what an item costs besides its key tiles.
// Measured on a B200: one unit of 256 rows a CTA, nothing masked, takes 21 us and 2.4 us
// (4,800 cycles, where the products need 2,900) a key tile; four sessions of up to 1024
// new tokens over 8192 (16/8 heads of 128) 323 us, 328 TFLOP/s, the join among them (40
// us by itself), with the tensor pipes active for a quarter of the time.
#include <algorithm>

#include "cache_attn.cuh"
#include "gemm_tc.cuh"
#include "tma_host.h"

namespace qa {

namespace {

constexpr int kRows = 128;      // of an MMA tile
constexpr int kUnitRows = 256;
constexpr int kKeys = 128;
constexpr int kConvWarps = 4, kSoftWarps = 8;
constexpr int kConv = kConvWarps * 32;
constexpr int kThreads = (kConvWarps + 2 + kSoftWarps) * 32;
constexpr int kRing = 4;       // pages of codes
constexpr int kScales = 4;     // key tiles whose pages' scales are there
constexpr uint32_t kHalf = kRows * 128;  // 64 f16 columns of a tile
constexpr uint32_t kTmemCols = 512;
constexpr int kMinStep = 8;    // key tiles of a chunk, at least
constexpr int kMaxChunks = 16;

// Key tiles of a chunk of a sequence with `keys` key tiles and `tiles` units a
// head: enough chunks to fill the GPU from one sequence, as few as that takes.  1024
// new tokens over 8192, 16/8 heads: one session 125 us with 16 in kMaxChunks and 185
// with 8, which leaves SMs idle; eight sessions 767 and 704 (no parts).  256 new
// tokens: 71 and 83.  The number of sequences must not decide: a sequence's result
// would depend on the others.
__host__ __device__ __forceinline__ int chunk_step(int keys, int tiles) {
  const int want = kMaxChunks / tiles > 1 ? kMaxChunks / tiles : 1;
  const int step = (keys + want - 1) / want;
  return step > kMinStep ? step : kMinStep;
}

struct TilePlan {
  int tiles, step;
  int chunks;  // of a unit, at most: each unit but the last has place for as many parts, if it is more than one
};
__device__ __forceinline__ TilePlan tile_plan(const CacheAttnParams& ap, const SeqSpan& sp) {
  const int group = ap.nq / ap.nkv;
  TilePlan p;
  p.tiles = sp.ok ? (sp.n * group + kUnitRows - 1) / kUnitRows : 0;
  const int keys = max(1, (sp.len + kKeys - 1) / kKeys);
  p.step = chunk_step(keys, max(1, p.tiles));
  p.chunks = (keys + p.step - 1) / p.step;
  return p;
}

// One unit's tile of rows.
struct Unit {
  int rows, seen;    // rows; tokens that its last row sees
  int keys;          // key tiles, at least one: a row that sees nothing still gets zeros
  int step, chunks;  // key tiles of a chunk, chunks
  int place;         // where its parts are in the sequence's and head's place
  bool pair;         // two tiles of rows, or no place for parts: streams are tiles
};
__device__ __forceinline__ Unit unit_of(const CacheAttnParams& ap, const SeqSpan& sp, const TilePlan& p,
                                        int s, int tile) {
  const int group = ap.nq / ap.nkv;
  Unit u;
  u.rows = min(kUnitRows, sp.n * group - tile * kUnitRows);
  const int last = (tile * kUnitRows + u.rows - 1) / group;
  u.seen = ap.causal ? min(sp.len, max(0, sp.len - sp.n + last + 1)) : sp.len;
  u.keys = max(1, (u.seen + kKeys - 1) / kKeys);
  u.step = p.step;
  u.chunks = (u.keys + u.step - 1) / u.step;
  u.pair = u.rows > kRows;
  // a part of both tiles for each chunk, or one of a tile for each chunk and stream
  u.place = p.chunks > 1 ? tile * p.chunks * ap.part_stride : 0;
  const int floats = !u.pair ? 2 * u.chunks * ap.half_stride : u.chunks > 1 ? u.chunks * ap.part_stride : 0;
  if (u.place + floats > ap.place_floats || (s + 1ll) * ap.nkv > ap.cap_units) {
    u.pair = true;
    u.chunks = 1;
    u.step = u.keys;
  }
  return u;
}

__device__ __forceinline__ PartsAt unit_parts(const CacheAttnParams& ap, const Unit& u, int s, int h) {
  return PartsAt{ap.parts + (static_cast<long long>(s) * ap.nkv + h) * ap.place_floats + u.place,
                 u.pair ? ap.part_stride : ap.half_stride,
                 padded_rows(u.pair ? ap.part_rows : min(kRows, ap.part_rows))};
}

// The parts that this kernel leaves, for the join.
struct TilesPlan {
  static constexpr int kRows = kUnitRows;
  static constexpr bool kAlone = true;
  __device__ static PartsAt place(const CacheAttnParams& ap, const SeqSpan& sp, const UnitAt& at) {
    return unit_parts(ap, unit_of(ap, sp, tile_plan(ap, sp), at.s, at.tile), at.s, at.h);
  }
  __device__ static int parts(const CacheAttnParams& ap, const SeqSpan& sp, int s, int tile) {
    const Unit u = unit_of(ap, sp, tile_plan(ap, sp), s, tile);
    return u.pair ? (u.chunks > 1 ? u.chunks : 0) : 2 * u.chunks;
  }
};

// One piece of work: a chunk of a unit.
struct Item {
  int s, tile, h, chunk;
  int k0, cnt;  // its key tiles
};

// A CTA's share: the chunks that begin in it.
struct TileWalk {
  long long x, hi;  // first key tile (of all units' laid end to end) not looked at, end of the share
  Item it;
  SeqSpan sp;
  TilePlan plan;
  Unit u;

  __device__ __forceinline__ void look(const CacheAttnParams& ap) {
    sp = seq_span(ap.seqs, it.s, ap.T);
    plan = tile_plan(ap, sp);
  }
  __device__ __forceinline__ void begin(const CacheAttnParams& ap, int seq, long long start, long long lo,
                                        long long end) {
    x = lo;
    hi = end;
    it = Item{seq, 0, 0, 0, 0, 0};
    look(ap);
    long long rel = lo - start;
    for (;; ++it.tile) {  // the share begins in this sequence: its units hold it
      u = unit_of(ap, sp, plan, it.s, it.tile);
      const long long c = static_cast<long long>(u.keys) * ap.nkv;
      if (rel < c) break;
      rel -= c;
    }
    it.h = static_cast<int>(rel / u.keys);
    const int in = static_cast<int>(rel % u.keys);
    it.chunk = (in + u.step - 1) / u.step - 1;
    x += min(u.keys, (it.chunk + 1) * u.step) - in;
  }
  __device__ __forceinline__ bool next(const CacheAttnParams& ap) {
    if (x >= hi) return false;
    if (++it.chunk == u.chunks) {
      it.chunk = 0;
      if (++it.h == ap.nkv) {
        it.h = 0;
        ++it.tile;
        while (it.tile >= plan.tiles) {  // x < hi <= all key tiles: there is another unit
          ++it.s;
          it.tile = 0;
          look(ap);
        }
        u = unit_of(ap, sp, plan, it.s, it.tile);
      }
    }
    it.k0 = it.chunk * u.step;
    it.cnt = min(u.step, u.keys - it.k0);
    x += it.cnt;
    return true;
  }
};

// A piece of work as the warps read it, from shared memory.
struct Work {
  long long t0;      // the sequence's first row of q and out
  const int* bt;     // its pages
  float* parts;      // where this chunk's (first) part goes; null: results are final
  int s, tile, h;
  int row0, rows;    // the unit's first row in the sequence, its rows
  int len, past;     // cached tokens; past + i + 1 of them are seen by new token i when causal
  int seen, all;     // tokens seen by the last row, by every row
  int k0, cnt;       // key tiles
  bool pair;
  // jobs of stream h, and the key tile (of the item) of its k-th
  __device__ __forceinline__ int jobs(int st) const {
    return pair ? (st == 0 || rows > kRows ? cnt : 0) : (cnt + 1 - st) / 2;
  }
  __device__ __forceinline__ int key_tile(int st, int k) const { return pair ? k : 2 * k + st; }
  // whether stream st is the last to use a key tile that streams share
  __device__ __forceinline__ bool last_user(int st) const { return st == 1 || rows <= kRows; }
};
constexpr int kBatch = 2;  // pieces of work described at a time

__device__ __forceinline__ Work work_of(const CacheAttnParams& ap, const TileWalk& walk) {
  const int group = ap.nq / ap.nkv;
  const Item& it = walk.it;
  const Unit& u = walk.u;
  Work w;
  w.t0 = walk.sp.t0;
  w.bt = ap.seqs.block_tab + static_cast<long long>(it.s) * ap.seqs.max_pages;
  w.s = it.s;
  w.tile = it.tile;
  w.h = it.h;
  w.row0 = it.tile * kUnitRows;
  w.rows = u.rows;
  w.len = walk.sp.len;
  w.past = walk.sp.len - walk.sp.n;
  w.seen = u.seen;
  w.all = ap.causal ? min(w.len, max(0, w.past + w.row0 / group + 1)) : w.len;
  w.k0 = it.k0;
  w.cnt = it.cnt;
  w.pair = u.pair;
  const PartsAt parts = unit_parts(ap, u, it.s, it.h);
  w.parts = u.pair && u.chunks == 1 ? nullptr : parts.base + (u.pair ? it.chunk : 2 * it.chunk) * parts.stride;
  return w;
}

// Store 16 consecutive 32-bit columns of this warp's 32 TMEM lanes (no wait).
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&w)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]),
      "r"(w[10]), "r"(w[11]), "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15])
      : "memory");
}

// 0x80 in each byte of w that is a NaN code.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}

template <int HD>
struct Mem {
  static constexpr uint32_t kTile = kHalf * (HD / 64);  // Q, K or V
  static constexpr size_t kSmem = 6 * kTile + kRing * kPage * HD + 2 * kUnitRows * 4 + 512 +
                                  kScales * 2 * sizeof(float4) + kBatch * sizeof(Work) + sizeof(TileWalk);
};

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) cache_attn_tiles(const __grid_constant__ CUtensorMap tmK,
                                                                const __grid_constant__ CUtensorMap tmV,
                                                                const __grid_constant__ CacheAttnParams ap) {
  constexpr uint32_t kTile = Mem<HD>::kTile;
  constexpr int kCpr = HD / 16;           // 16-byte units of codes a row
  constexpr uint32_t kPageBytes = kPage * HD;
  extern __shared__ __align__(1024) uint8_t smem[];  // no room to align it by hand
  static_assert(Mem<HD>::kSmem <= 232448, "shared memory of a CTA");
  uint8_t* sQ = smem;              // [tile]
  uint8_t* sK = sQ + 2 * kTile;    // [slot]
  uint8_t* sV = sK + 2 * kTile;    // [slot]
  uint8_t* ring = sV + 2 * kTile;  // [slot] a page of codes
  float* s_undo = reinterpret_cast<float*>(ring + kRing * kPageBytes);  // [item & 1][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_undo + 2 * kUnitRows);
  uint64_t* q_full = bars + 0;   // [item & 1] queries and their factors are there
  uint64_t* q_free = bars + 2;   // the item's last S is done
  uint64_t* k_full = bars + 4;   // [slot]
  uint64_t* k_empty = bars + 6;
  uint64_t* v_full = bars + 8;
  uint64_t* v_empty = bars + 10;
  uint64_t* s_full = bars + 12;  // [stream] S computed
  uint64_t* p_full = bars + 14;  // [stream] P written over S
  uint64_t* o_ready = bars + 16; // [stream] P V done
  uint64_t* o_free = bars + 18;  // [stream] O read
  uint64_t* r_full = bars + 20;  // [ring slot]
  uint64_t* r_empty = bars + 24;
  uint64_t* sc_full = bars + 50;  // [key tile % kScales] scales are there
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + 28);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tslot + 1);
  int* r_ok = reinterpret_cast<int*>(bars + 29);               // [ring slot] the page was loaded
  long long* share = reinterpret_cast<long long*>(bars + 31);  // lo, hi, start, sequence
  long long* scan = share + 4;                                 // [warp]
  int* staged = reinterpret_cast<int*>(scan + kThreads / 32);  // pieces of work described
  // a page's K scale, log2 and reciprocal of its V scale, 1 if it is there
  float4* sc = reinterpret_cast<float4*>(bars + 64);           // [kScales][2]
  Work* work = reinterpret_cast<Work*>(sc + kScales * 2);      // [kBatch]

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int group = ap.nq / ap.nkv, n_seqs = ap.seqs.n_seqs;
  if (smem_u32(smem) & 1023u) {  // the swizzled tiles would not be where the MMA looks for them
    if (threadIdx.x == 0 && ap.status) atomicOr(ap.status, kStatusTimeout);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], kConv);
      mbar_init(&k_full[i], kConv);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], kConv);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kRows);
      mbar_init(&o_ready[i], 1);
      mbar_init(&o_free[i], kRows);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], kConvWarps);
    }
    for (int i = 0; i < kScales; ++i) mbar_init(&sc_full[i], 1);
    mbar_init(q_free, 1);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kConvWarps) tmem_alloc(tslot, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = __shfl_sync(0xFFFFFFFFu, *tslot, 0);
  pdl_wait();
  pdl_trigger();

  // ---- this CTA's share: thread i adds up sequences [i c, (i + 1) c)
  bool any;
  {
    const int c = (n_seqs + kThreads - 1) / kThreads;
    const int s0 = min(n_seqs, static_cast<int>(threadIdx.x) * c), s1 = min(n_seqs, s0 + c);
    auto cost_of = [&](int s) {
      const SeqSpan sp = seq_span(ap.seqs, s, ap.T);
      const TilePlan p = tile_plan(ap, sp);
      long long sum = 0;
      for (int t = 0; t < p.tiles; ++t) sum += unit_of(ap, sp, p, s, t).keys;
      return sum * ap.nkv;
    };
    long long mine = 0;
    for (int s = s0; s < s1; ++s) {
      mine += cost_of(s);
      if (blockIdx.x == 0 && ap.status && !seq_span(ap.seqs, s, ap.T).ok) atomicOr(ap.status, kStatusBadShape);
    }
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xFFFFFFFFu, before, o);
      if (lane >= o) before += y;
    }
    if (lane == 31) scan[warp] = before;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    before -= mine;
    const long long quot = total / gridDim.x, rem = total % gridDim.x, b = blockIdx.x;
    const long long lo = quot * b + min(b, rem), hi = lo + quot + (b < rem ? 1 : 0);
    any = lo < hi;
    if (any && lo >= before && lo < before + mine) {
      share[0] = lo;
      share[1] = hi;
      long long at = before;
      for (int s = s0; s < s1; ++s) {
        const long long cost = cost_of(s);
        if (lo < at + cost) {
          share[2] = at;
          share[3] = s;
          break;
        }
        at += cost;
      }
    }
    __syncthreads();
  }
  auto fail = [&]() {
    *abort_flag = 1;
    if (ap.status) atomicOr(ap.status, kStatusTimeout);
  };
  // bounded wait taken by a whole warp, warp-uniform result
  auto wait = [&](uint64_t* bar, uint32_t par) -> bool {
    if (__all_sync(0xFFFFFFFFu, mbar_try_wait(smem_u32(bar), par & 1u))) return true;
    return __all_sync(0xFFFFFFFFu, !*abort_flag && mbar_wait(bar, par & 1u));
  };
  // a value that is the same in all lanes, known as such to the compiler: operands
  // of the MMAs are then made in uniform registers
  auto same = [](int v) { return __shfl_sync(0xFFFFFFFFu, v, 0); };
  auto good = [&](int page) { return page >= 0 && page < ap.kv_pages; };
  // thread 0's, in shared memory: it would take registers of every thread otherwise
  TileWalk& walk = *reinterpret_cast<TileWalk*>(work + kBatch);
  if (threadIdx.x == 0 && any) walk.begin(ap, static_cast<int>(share[3]), share[2], share[0], share[1]);
  bool ok = true;
  uint32_t n_it = 0;  // pieces of work before this one
  uint32_t g = 0;     // key tiles before this one
  uint32_t pages = 0;  // of codes before this one
  uint32_t uses0 = 0, uses1 = 0, jobs0 = 0, jobs1 = 0;  // of the streams
  for (;;) {
    if (threadIdx.x == 0) {
      int n = 0;
      while (any && n < kBatch && walk.next(ap)) work[n++] = work_of(ap, walk);
      *staged = n;
    }
    __syncthreads();
    const int n_work = *staged;
    if (n_work == 0 || *abort_flag) break;
  if (warp < kConvWarps) {
    // ================================================ conversion
    // A thread has unit c of the rows row0 + i kRowStep.  hd 128: neighbouring rows'
    // lanes 0-3 and 4-7 take opposite halves of their rows, so that the eight lanes
    // of a 16-byte access meet different banks when they read codes and when they
    // write f16 (whose units are XORed with the row's low bits).
    constexpr int kRowStep = kConv / kCpr;
    const int c = HD == 128 ? (lane & 3) + 4 * ((lane >> 2 ^ lane >> 3) & 1) : lane & 3;
    const int row0 = HD == 128 ? warp * 4 + (lane >> 4) * 2 + (lane >> 2 & 1) : warp * 8 + (lane >> 2);
    const uint32_t from0 = row0 * HD + 16 * (c ^ (HD == 128 ? row0 & 7 : (row0 >> 1) & 3));
    // f16 dims 16 c .. 16 c + 15 of row0, as two units; row0 + i kRowStep has the
    // same low bits
    const uint32_t to0 = (c >> 2) * kHalf + row0 * 128 + 16 * ((2 * (c & 3)) ^ (row0 & 7));
    const uint32_t to1 = (c >> 2) * kHalf + row0 * 128 + 16 * ((2 * (c & 3) + 1) ^ (row0 & 7));
    static_assert(kRowStep % 8 == 0, "rows of a thread have the same low bits");
    for (int wi = 0; ok && wi < n_work; ++wi) {
      const Work& it = work[wi];
      const int seen = it.seen, all = it.all, h_kv = it.h;
      // a key tile's two pages from the ring to a tile
      // (the loops over pages are not unrolled, here and in the softmax: the roles' code
      // together has to stay in the instruction cache)
      auto convert = [&](uint8_t* tile, int key0, bool v) -> bool {
#pragma unroll 1
        for (int p = 0; p < 2; ++p, ++pages) {
          const int slot = pages % kRing;
          if (!wait(&r_full[slot], pages / kRing)) return false;
          const bool on = r_ok[slot];
          const uint8_t* from = ring + slot * kPageBytes;
          uint4 d[kPage / kRowStep];
#pragma unroll
          for (int i = 0; i < kPage / kRowStep; ++i)
            d[i] = *reinterpret_cast<const uint4*>(from + from0 + i * (kRowStep * HD));
          if (!on || key0 + (p + 1) * kPage > seen || (v && key0 + (p + 1) * kPage > all)) {
#pragma unroll
            for (int i = 0; i < kPage / kRowStep; ++i) {
              const int key = key0 + p * kPage + row0 + i * kRowStep;
              uint32_t* w = reinterpret_cast<uint32_t*>(&d[i]);
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                if (v && key >= all) w[y] &= ~((nan_codes(w[y]) >> 7) * 0xFFu);
                if (!on || key >= seen) w[y] = 0;
              }
            }
          }
          uint8_t* to = tile + p * kPage * 128;
#pragma unroll
          for (int i = 0; i < kPage / kRowStep; ++i) {
            uint4 lo, hi;
            e4m3x4_f16x2(d[i].x, lo.x, lo.y);
            e4m3x4_f16x2(d[i].y, lo.z, lo.w);
            e4m3x4_f16x2(d[i].z, hi.x, hi.y);
            e4m3x4_f16x2(d[i].w, hi.z, hi.w);
            *reinterpret_cast<uint4*>(to + to0 + i * (kRowStep * 128)) = lo;
            *reinterpret_cast<uint4*>(to + to1 + i * (kRowStep * 128)) = hi;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&r_empty[slot]);
        }
        return true;
      };
      // ---- queries: copied to where their f16 values go (16 bits either way), all on
      // their way at once, then bf16 converted in place.  Short loops: code that runs
      // once a piece of work comes from beyond the instruction cache.
      if (n_it > 0 && !wait(q_free, n_it - 1)) {
        ok = false;
        break;
      }
      const int rows_up = it.rows > kRows ? 2 * kRows : kRows;
      auto q_at = [&](int r, uint32_t unit) { return sQ + (r / kRows) * kTile + (r % kRows - row0) * 128 + unit; };
      {
        int tok = (it.row0 + row0) / group, head = (it.row0 + row0) % group;  // of the row to be read
        const int tok_step = kRowStep / group, head_step = kRowStep % group;
#pragma unroll 1
        for (int r = row0; r < rows_up; r += kRowStep) {
          const bool in = r < it.rows;
          const T* src = static_cast<const T*>(ap.q);
          if (in) src += (it.t0 + tok) * ap.ldq + (h_kv * group + head) * HD + 16 * c;
          if (ap.vec) {
            cp_async16(smem_u32(q_at(r, to0)), src, in ? 16 : 0);
            cp_async16(smem_u32(q_at(r, to1)), src + (in ? 8 : 0), in ? 16 : 0);
          } else {
#pragma unroll 1
            for (int k = 0; k < 16; ++k)
              reinterpret_cast<T*>(q_at(r, k < 8 ? to0 : to1))[k % 8] = in ? src[k] : f2h<T>(0.0f);
          }
          tok += tok_step;
          head += head_step;
          if (head >= group) {
            head -= group;
            ++tok;
          }
        }
        cp_async_commit();
        cp_async_wait_all();
      }
      float* undo_of = s_undo + (n_it & 1) * kUnitRows;
      const bool flip = ap.scale < 0.0f;  // the softmax takes a positive scale
#pragma unroll 2
      for (int r = row0; r < rows_up; r += kRowStep) {
        float undo = 1.0f;
        if (H16Traits<T>::kBf16 || flip) {
          uint4 raw[2] = {*reinterpret_cast<const uint4*>(q_at(r, to0)), *reinterpret_cast<const uint4*>(q_at(r, to1))};
          uint32_t* w = reinterpret_cast<uint32_t*>(raw);
          if constexpr (H16Traits<T>::kBf16) {
            float shift = 1.0f;
            // the largest magnitude, in pairs: of two finite bf16 the larger bits are
            // the larger magnitude, and those of infinities and NaN are larger still
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) top = __vmaxu2(top, w[k] & 0x7FFF7FFFu);
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            if (HD == 128) top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
            const int ex = static_cast<int>(max(top & 0xFFFFu, top >> 16) >> 7) - 127;  // 2^ex <= it
            if (top && ex < 128) {
              const int up = min(14 - ex, 126);
              shift = __int_as_float((up + 127) << 23);
              undo = __int_as_float((127 - up) << 23);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
              w[k] = cvt2_rn<__half>(
                  make_float2(__uint_as_float(w[k] << 16) * shift, __uint_as_float(w[k] & 0xFFFF0000u) * shift));
          }
          if (flip)
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] ^= 0x80008000u;
          *reinterpret_cast<uint4*>(q_at(r, to0)) = raw[0];
          *reinterpret_cast<uint4*>(q_at(r, to1)) = raw[1];
        }
        if (c == 0) undo_of[r] = undo;
      }
      fence_proxy_async_smem();
      mbar_arrive(&q_full[n_it & 1]);
      // ---- key tiles
      for (int j = 0; ok && j < it.cnt; ++j, ++g) {
        const int slot = g & 1;
#pragma unroll 1
        for (int v = 0; v < 2; ++v) {
          if (!wait((v ? v_empty : k_empty) + slot, (g >> 1) + 1) ||
              !convert((v ? sV : sK) + slot * kTile, (it.k0 + j) * kKeys, v)) {
            ok = false;
            break;
          }
          fence_proxy_async_smem();
          mbar_arrive((v ? v_full : k_full) + slot);
        }
      }
      ++n_it;
    }
  } else if (warp == kConvWarps) {
    // ================================================ MMA (the warp together, one lane elected)
    const uint32_t idS = f16_instr_desc(kRows, kKeys, false);
    const uint32_t idPV = f16_instr_desc(kRows, HD, false) | (1u << 16);  // V MN-major
    const uint32_t qa = smem_u32(sQ), ka = smem_u32(sK), va = smem_u32(sV);
    for (int wi = 0; ok && wi < n_work; ++wi) {
      const Work& it = work[wi];
      const int nj0 = same(it.jobs(0)), nj1 = same(it.jobs(1)), cnt = same(it.cnt);
      const bool pair = same(it.pair);
      const uint32_t last = same(it.last_user(0)) ? 0 : 1;  // stream that frees a shared key tile
      const uint64_t dq0 = sw128_kmajor_desc(qa), dq1 = sw128_kmajor_desc(pair ? qa + kTile : qa);
      if (!wait(&q_full[n_it & 1], n_it >> 1)) {
        ok = false;
        break;
      }
      int left = nj0 + nj1;  // S products to be issued
      // S of stream h's k-th job
      auto issue_s = [&](int h, int k) -> bool {
        const uint32_t kt = g + (pair ? k : 2 * k + h);
        if (!wait(&k_full[kt & 1], kt >> 1)) return false;
        tc_fence_after();
        const uint64_t dq = h ? dq1 : dq0, dk = sw128_kmajor_desc(ka + (kt & 1) * kTile);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const uint32_t off = (ks >> 2) * (kHalf >> 4) + (ks & 3) * 2;
          mma_f16_e(tbase + h * 128, dq + off, dk + off, idS, ks > 0 ? 1u : 0u);
        }
        mma_commit_e(&s_full[h]);
        if (!pair || h == last) mma_commit_e(&k_empty[kt & 1]);
        if (--left == 0) mma_commit_e(q_free);
        return true;
      };
      // P V of stream h's k-th job, then S of its next
      auto step = [&](int h, int k, int nj, uint32_t uses, uint32_t& jobs) -> bool {
        if (k >= nj) return true;
        if (k == 0 && uses > 0 && !wait(&o_free[h], uses - 1)) return false;
        const uint32_t kt = g + (pair ? k : 2 * k + h);
        if (!wait(&v_full[kt & 1], kt >> 1) || !wait(&p_full[h], jobs)) return false;
        tc_fence_after();
        const uint64_t dv = sw128_mn_desc(va + (kt & 1) * kTile, kHalf, 1024);
#pragma unroll
        for (int ks = 0; ks < kKeys / 16; ++ks)
          mma_f16_ts_e(tbase + 256 + h * 128, tbase + h * 128 + (ks >> 2) * 64 + (ks & 3) * 8, dv + ks * 128, idPV,
                       (k > 0 || ks > 0) ? 1u : 0u);
        mma_commit_e(&o_ready[h]);
        if (!pair || h == last) mma_commit_e(&v_empty[kt & 1]);
        ++jobs;
        return k + 1 >= nj || issue_s(h, k + 1);
      };
      if (nj0 > 0) ok = issue_s(0, 0);
      if (ok && nj1 > 0) ok = issue_s(1, 0);
      for (int k = 0; ok && k < max(nj0, nj1); ++k)
        ok = step(0, k, nj0, uses0, jobs0) && step(1, k, nj1, uses1, jobs1);
      uses0 += nj0 > 0;
      uses1 += nj1 > 0;
      g += cnt;
      ++n_it;
    }
  } else if (warp == kConvWarps + 1) {
    // ================================================ TMA
    for (int wi = 0; ok && wi < n_work; ++wi) {
      const Work& it = work[wi];
      int next[2] = {0, 0};  // page ids, read a key tile ahead
      auto look = [&](int kt) {
#pragma unroll
        for (int p = 0; p < 2; ++p) next[p] = kt * kKeys + p * kPage < it.seen ? it.bt[2 * kt + p] : -2;
      };
      look(it.k0);
      for (int j = 0; ok && j < it.cnt; ++j) {
        const int now[2] = {next[0], next[1]};
        if (j + 1 < it.cnt) look(it.k0 + j + 1);
        float ks = 0.0f, vs = 1.0f;  // lanes 0 and 1: of their pages
        if (lane < 2 && good(now[lane & 1])) {
          const long long at = static_cast<long long>(now[lane & 1]) * ap.nkv + it.h;
          ks = ap.kscale[at];
          vs = usable_vscale(ap.vscale[at]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i, ++pages) {  // K, K, V, V
          const int slot = pages % kRing, page = now[i & 1];
          if (!wait(&r_empty[slot], pages / kRing + 1)) {
            ok = false;
            break;
          }
          if (i == 1) {
            // Four key tiles back, the softmax is done with this place: the page before
            // this one needed the ring's last K page converted, and with it the V
            // tile before that, whose slot was free only after the P V product two
            // tiles further back.
            if (lane < 2)
              sc[(g % kScales) * 2 + lane] = make_float4(ks, lg2_approx(vs), rcp_approx(vs), good(now[lane & 1]) ? 1.0f : 0.0f);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sc_full[g % kScales]);
            ++g;
          }
          if (lane == 0) {
            r_ok[slot] = good(page);
            if (good(page)) {
              mbar_arrive_expect_tx(&r_full[slot], kPageBytes);
              tma_load_2d(i < 2 ? &tmK : &tmV, &r_full[slot], ring + slot * kPageBytes, 0,
                          (page * ap.nkv + it.h) * kPage);
            } else {
              if (page != -2 && ap.status) atomicOr(ap.status, kStatusBadShape);
              mbar_arrive(&r_full[slot]);
            }
          }
          __syncwarp();
        }
      }
      ++n_it;
    }
  } else {
    // ================================================ softmax and results: stream h, row r
    const int h = (warp - kConvWarps - 2) / 4, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tbase + h * 128 + lane_off, tO = tbase + 256 + h * 128 + lane_off;
    constexpr float kTiny = 1.1754944e-38f;  // a factor of 0 would lose the masks (0 . -inf is NaN)
    const float scale = fabsf(ap.scale) * kLog2e;
    uint32_t& jobs = jobs0;
    for (int wi = 0; ok && wi < n_work; ++wi) {
      const Work& it = work[wi];
      // Dims 32 quarter .. of the results (all of them: any bit, quarter -1) that NaN
      // codes of V of tokens [from, to) below lim spoil.  The warp looks at 32 / kCpr
      // tokens at a time, a unit of 16 dims a lane.
      auto nan_dims = [&](int from, int to, int lim, int quarter) {
        uint32_t mask = 0;
#pragma unroll 1
        for (int key0 = from; key0 < to; key0 += 32 / kCpr) {
          const int key = key0 + lane / kCpr, page = key < to ? it.bt[key / kPage] : -1;
          uint32_t bits = 0;
          if (good(page)) {
            const uint4 d = __ldg(reinterpret_cast<const uint4*>(
                ap.vpool + ((static_cast<long long>(page) * ap.nkv + it.h) * kPage + (key & 63)) * HD +
                16 * (lane % kCpr)));
            auto four = [](uint32_t w) {  // the NaN codes of a word, a bit each
              const uint32_t n = nan_codes(w) >> 7;
              return (n & 1u) | (n >> 7 & 2u) | (n >> 14 & 4u) | (n >> 21 & 8u);
            };
            bits = four(d.x) | four(d.y) << 4 | four(d.z) << 8 | four(d.w) << 12;
          }
          if (!__any_sync(0xFFFFFFFFu, bits != 0)) continue;
#pragma unroll 1
          for (int l2 = 0; l2 < 32; ++l2) {
            const uint32_t b = __shfl_sync(0xFFFFFFFFu, bits, l2);
            const int its_key = __shfl_sync(0xFFFFFFFFu, key, l2), unit = l2 % kCpr;
            if (its_key < lim && (quarter < 0 || unit / 2 == quarter)) mask |= b << (16 * (unit & 1));
          }
        }
        return mask;
      };
      const int nj = it.jobs(h);
      const int ur = it.pair ? h * kRows + r : r;  // the unit's row
      const int row = it.row0 + ur, tok = row / group;
      const bool valid = ur < it.rows;
      if (it.pair && h == 1 && it.rows <= kRows) {  // no such tile
        ++n_it;
        g += it.cnt;
        continue;
      }
      const int lim = !valid ? 0 : ap.causal ? max(0, min(it.len, it.past + tok + 1)) : it.len;  // tokens it sees
      const int h_kv = it.h;
      float m = -INFINITY, l = 0.0f;
      bool spoiled = false;  // some results, by a NaN code of V that was taken out
      float kf = 0.0f;
      if (nj > 0) {
        if (!wait(&q_full[n_it & 1], n_it >> 1)) {
          ok = false;
          break;
        }
        kf = s_undo[(n_it & 1) * kUnitRows + ur] * scale;
      }
      ++n_it;
      for (int k = 0; k < nj; ++k, ++jobs) {
        const int kt = it.k0 + it.key_tile(h, k);
        const uint32_t place = g + it.key_tile(h, k);
        if (!wait(&sc_full[place % kScales], place / kScales)) {
          ok = false;
          break;
        }
        const float4* pg = sc + (place % kScales) * 2;
        if (!wait(&s_full[h], jobs)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t x[64];
        auto fetch = [&](int p) {
          tmem_ld_x64(tS + p * 64, x);
          const int see = pg[p].w != 0.0f ? lim - kt * kKeys - p * kPage : 0;
          if (see < 64)
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (i >= see) x[i] = __float_as_uint(-INFINITY);
        };
        float top = -INFINITY;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          fetch(p);
          float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 64; ++i) t4[i & 3] = fmaxf(t4[i & 3], __uint_as_float(x[i]));
          const float t = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
          top = fmaxf(top, fmaf(t, fmaxf(pg[p].x * kf, kTiny), pg[p].y));
        }
        const bool grow = top > m + kSlack;
        float alpha = 1.0f;
        if (grow) {
          alpha = ex2_approx(m - top);  // 0 the first time
          m = top;
          l *= alpha;
        }
        if (k > 0 && __any_sync(0xFFFFFFFFu, grow)) {
          if (!wait(&o_ready[h], jobs - 1)) {  // the last P V is done
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int q = 0; q < HD / 32; ++q) {
            float o[32];
            tmem_ld32(tO + q * 32, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= alpha;
            tmem_st32(tO + q * 32, o);
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        // page 1 first: its scores are in x; a page's P (32 columns) goes over its scores
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int p = 1 - q;
          if (q == 1) fetch(p);
          const float4 of = pg[p];
          const float up = of.y + (kLift - ref), fp = fmaxf(of.x * kf, kTiny);
          float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float p0 = ex2_approx(fmaf(__uint_as_float(x[32 * half + 2 * e]), fp, up));
              const float p1 = ex2_approx(fmaf(__uint_as_float(x[32 * half + 2 * e + 1]), fp, up));
              s4[e & 3] += p0 + p1;
              w[e] = cvt2_rn<__half>(make_float2(p0, p1));
            }
            tmem_st_x16(tS + p * 64 + half * 16, w);
          }
          l = fmaf((s4[0] + s4[1]) + (s4[2] + s4[3]), of.z, l);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[h]);
        // ---- NaN codes of V that only some rows see
        if ((kt + 1) * kKeys > it.all)
          spoiled |= nan_dims(max(it.all, kt * kKeys), min(it.seen, (kt + 1) * kKeys), lim, -1) != 0;
      }
      if (!ok) break;
      if (nj > 0 && !wait(&o_ready[h], jobs - 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // ---- the row's result, or its part
      const UnitAt at{it.s, it.tile, h_kv, it.t0};
      float inv = 1.0f;
      float* part = it.parts;
      if (part) {
        const int l_at = padded_rows(it.pair ? ap.part_rows : min(kRows, ap.part_rows));
        if (!it.pair) part += h * ap.half_stride;
        if (valid) {
          __stcg(part + ur, m);
          __stcg(part + l_at + ur, l);
        }
        part += 2 * l_at + ur * HD;
      } else if (valid) {
        inv = close_row(ap, at, row, m, l);
      }
      T* dst = static_cast<T*>(ap.out) + (it.t0 + tok) * ap.ldo + static_cast<long long>(h_kv * group + row % group) * HD;
#pragma unroll 1
      for (int q = 0; q < HD / 32; ++q) {
        float o[32];
        if (nj > 0) {
          tmem_ld32(tO + q * 32, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.0f;
        }
        if (__any_sync(0xFFFFFFFFu, spoiled)) {
          // this chunk's tokens of the stream, which the warp has seen to hold some
          uint32_t bad = 0;
#pragma unroll 1
          for (int k = 0; k < nj; ++k) {
            const int kt = it.k0 + it.key_tile(h, k);
            if ((kt + 1) * kKeys > it.all)
              bad |= nan_dims(max(it.all, kt * kKeys), min(it.seen, (kt + 1) * kKeys), lim, q);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (bad >> e & 1) o[e] = NAN;
        }
        if (part) {
          if (valid)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              __stcg(reinterpret_cast<float4*>(part + q * 32) + e,
                     make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]));
        } else if (valid && ap.vec) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(dst + q * 32 + 8 * e) =
                make_uint4(cvt2_rn<T>(make_float2(o[8 * e] * inv, o[8 * e + 1] * inv)),
                           cvt2_rn<T>(make_float2(o[8 * e + 2] * inv, o[8 * e + 3] * inv)),
                           cvt2_rn<T>(make_float2(o[8 * e + 4] * inv, o[8 * e + 5] * inv)),
                           cvt2_rn<T>(make_float2(o[8 * e + 6] * inv, o[8 * e + 7] * inv)));
        } else if (valid) {
#pragma unroll
          for (int e = 0; e < 32; ++e) dst[q * 32 + e] = f2h<T>(o[e] * inv);
        }
      }
      if (nj > 0) {
        tc_fence_before();
        mbar_arrive(&o_free[h]);
      }
      g += it.cnt;
    }
  }
    if (!ok && lane == 0) fail();
    __syncthreads();  // the descriptions have been read
    if (*abort_flag && warp == kConvWarps + 1)  // no copy may be on its way when the CTA ends
      for (uint32_t n = pages > kRing ? pages - kRing : 0; n < pages; ++n)
        mbar_wait_warp(&r_full[n % kRing], (n / kRing) & 1);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kConvWarps) {
    tc_fence_after();
    tmem_dealloc(tbase, kTmemCols);
  }
}

struct PartSizes {
  int tiles, rows, stride, half;
  long long place_floats;  // of a sequence and K/V head
};
PartSizes part_sizes(int nq, int nkv, int hd, int max_q, int max_kv) {
  PartSizes p;
  const long long rows = static_cast<long long>(max_q) * (nq / nkv);
  p.tiles = static_cast<int>((rows + kUnitRows - 1) / kUnitRows);
  p.rows = static_cast<int>(std::min<long long>(kUnitRows, rows));
  p.stride = part_floats(p.rows, hd);
  p.half = part_floats(std::min(kRows, p.rows), hd);
  const int most = (std::max(1, max_kv) - 1) / kKeys / kMinStep + 1;  // chunks of a unit, whatever its tiles
  // the most that a sequence of up to so many tiles asks for: 4096 rows or fewer
  p.place_floats = 0;
  for (int t = 1; t <= std::min(p.tiles, kMaxChunks); ++t) {
    const long long chunks = std::min(kMaxChunks / t, most), whole = chunks > 1 ? chunks * p.stride : 0;
    p.place_floats = std::max(p.place_floats, (t - 1) * whole + std::max(whole, 2 * chunks * p.half));
  }
  return p;
}

template <typename T, int HD>
cudaError_t launch(CacheAttnParams ap, int max_kv, void* ws, long long ws_bytes, cudaStream_t s) {
  const PartSizes ps = part_sizes(ap.nq, ap.nkv, HD, ap.seqs.max_q, max_kv);
  ap.tiles_max = ps.tiles;
  ap.part_rows = ps.rows;
  ap.part_stride = ps.stride;
  ap.half_stride = ps.half;
  ap.parts = static_cast<float*>(ws);
  ap.place_floats = ps.place_floats;
  ap.cap_units = ws ? ws_bytes / (4 * ps.place_floats) : 0;
  CUtensorMap tk, tv;
  const long long rows = static_cast<long long>(ap.kv_pages) * ap.nkv * kPage;
  if (rows > 0x7FFFFFFFll) return cudaErrorInvalidValue;  // TMA row coordinates
  // codes in pairs, as 16-bit elements
  const long long dims[2] = {HD / 2, rows}, stride[1] = {HD};
  const int box[2] = {HD / 2, kPage}, step[2] = {1, 1};
  int rc = make_tmap_nd(&tk, ap.kpool, false, 2, dims, stride, box, step, HD);
  if (!rc) rc = make_tmap_nd(&tv, ap.vpool, false, 2, dims, stride, box, step, HD);
  if (rc) return static_cast<cudaError_t>(rc);
  auto k = cache_attn_tiles<T, HD>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Mem<HD>::kSmem);
  if (e == cudaSuccess) e = launch_pdl(k, dim3(device_sm_count()), dim3(kThreads), Mem<HD>::kSmem, s, tk, tv, ap);
  if (e == cudaSuccess && ap.cap_units > 0) {
    e = launch_join<T, HD, TilesPlan>(ap, s);
  }
  return e;
}

}  // namespace

long long cache_tiles_workspace(int nqh, int nkvh, int hd, int n_seqs, int max_q, int max_kv) {
  const PartSizes p = part_sizes(nqh, nkvh, hd, max_q, max_kv);
  return places_bytes(n_seqs, nkvh, p.place_floats);
}

int cache_attention_tiles(const CacheAttnParams& ap, int hd, bool bf16, int max_kv, void* ws,
                          long long ws_bytes, cudaStream_t s) {
  if (bf16)
    return hd == 128 ? launch<__nv_bfloat16, 128>(ap, max_kv, ws, ws_bytes, s)
                     : launch<__nv_bfloat16, 64>(ap, max_kv, ws, ws_bytes, s);
  return hd == 128 ? launch<__half, 128>(ap, max_kv, ws, ws_bytes, s)
                   : launch<__half, 64>(ap, max_kv, ws, ws_bytes, s);
}

}  // namespace qa
