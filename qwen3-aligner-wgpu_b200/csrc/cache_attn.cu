// Attention over the 8-bit paged cache (codes and scales as kv_append writes
// them).
//
// Query i of sequence s (n new tokens, len cached ones, the new ones among
// them) sees cache indices c < len - n + i + 1 when causal, c < len otherwise:
//   s_c = scale kscale[page(c)] (q . kcode_c),  out = sum_c softmax(s)_c vscale[page(c)] vcode_c,
// lse = log sum_c exp(s_c); a row that sees nothing gets 0 and -inf.
#include <algorithm>
#include <atomic>

#include "cache_attn.cuh"
#include "gemm_tc.cuh"
#include "tma_host.h"

namespace qa {

namespace {

// ------------------------------------------------------------ few query rows
// A query row is one (new token, head of the K/V head's group); row r of a
// sequence is token r / group, head r % group.  A CTA takes up to 8 * NT rows of one
// sequence and K/V head (a unit) at a time.
//
// Bound: the cache's bytes, read once (2 hd a token and head), so what matters
// is that every SM reads all the time, bytes in flight and instructions a byte.
//  - A unit's cached tokens are cut into chunks by the unit's own length alone
//    (the batch it is in does not move a sequence's cuts).  The slabs
//    of 32 tokens of all units, laid end to end, are shared out evenly over the
//    CTAs that the GPU holds; a CTA takes the chunks that begin in its share,
//    which it finds from kv_len and q_start itself.  Its four warps take every
//    fourth slab of a chunk and are joined in shared memory.
//  - A unit of one chunk is finished where it is computed.  Otherwise each chunk
//    leaves its part (m, l, O) in the workspace, and a second kernel joins a
//    unit's parts in their order (joining them in this kernel, by whoever comes
//    last, measured slower: one warp reads 512 parts of 7 rows in 50 us, at the
//    very end).  No atomics, the same bits each time.
//  - Each warp streams its own slabs through a private ring of kStages slabs
//    (TMA, 128-byte swizzle; hd 64: 64-byte), without any CTA-wide barrier in
//    the loop.
//
// Tokens are the M = 16 side of both products, so 8 rows cost one mma.sync
// m16n8k16 a 16x16 block and nothing is padded to 16 rows:
//   S^T [16 tokens][8 rows] = K [16][hd] . Q^T,
//   O^T [hd][8 rows]       += V^T [hd][16 tokens] . P^T.
// The order of the dims inside S^T's sum, and of the dims along O^T's rows, is
// free; it is chosen so that a thread reads its K and V operands as whole
// 16-byte units (16-byte units XOR-swizzled by token: no bank conflicts).
// V's pairs of tokens are formed bytewise before the conversion to f16 (one
// PRMT per two pairs); P^T comes from S^T's layout by movmatrix.
//
// e4m3 codes are exact in f16.  So are bf16 queries once a row is scaled by a
// power of two that brings its largest component to [2^14, 2^15): components up to
// 2^28 smaller keep all their bits, and what is lost of others lies 2^-39 below the
// largest.  P is rounded to f16 (cache_attn.cuh says what that costs).
//
// As M moves rarely, a slab usually needs one vote instead of a maximum across
// lanes.
constexpr int kMaxCtasPerSm = 3;
constexpr int kMaxParts = 1024;  // parts of a unit

constexpr int kWarps = 4;

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 8x8 transpose of 16-bit values across the warp.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}

// Tokens of a chunk of a unit of `tokens` tokens, a multiple of 32.  A short unit is
// one chunk, which needs no part and no second kernel (one row, 16/8 heads of 128,
// against 64- and 128-token chunks of single warps that are joined afterwards: 64
// sessions of 512 tokens 29 against 39 us, one of 128 tokens 10 against 14, of 1024
// the same).  Longer ones: 768 tokens keep the parts few and the shares even (two
// sessions of 131,000 tokens: 46 us, 49 with 512, 60 with 256; 16 of 5000 with 24
// rows: 55, 59 and 77; one of 8192 with 24 rows: 39, 27 and 29).
constexpr int kShort = 1024, kChunk = 768;
__host__ __device__ __forceinline__ int chunk_tokens(int tokens) {
  if (tokens <= kShort) return kShort;
  return tokens <= kMaxParts * kChunk ? kChunk : ((tokens - 1) / (kMaxParts * 32) + 1) * 32;
}

// Shared memory of the few-row kernel besides the ring.
template <int R, int STAGES>
struct RowsShared {
  uint64_t full[kWarps][STAGES][2];  // K, V
  float m[kWarps][R], l[kWarps][R];  // the warps' references and sums
  float cm[R], cl[R];                // of the joined warps
  float inv[R];                      // 1 / sum
  long long scan[kWarps];
  long long lo, hi;                  // the CTA's share of the slabs
  long long start;                   // first slab of the first sequence of the share
  int seq;                           // that sequence
};

// What a sequence asks of the few-row kernel: tiles x K/V heads units of
// `slabs` slabs, each in `chunks` chunks of `step` slabs.
struct SeqPlan {
  int tiles, slabs, step, chunks;
  long long cost;  // slabs of all units
};
__device__ __forceinline__ SeqPlan seq_plan(const CacheAttnParams& ap, const SeqSpan& sp, int s,
                                            int group, int R, int slab) {
  SeqPlan c;
  c.tiles = sp.ok ? (sp.n * group + R - 1) / R : 0;
  c.slabs = max(1, (sp.len + slab - 1) / slab);  // an empty cache still owes its rows zeros
  c.step = chunk_tokens(sp.len) / slab;
  c.chunks = (c.slabs + c.step - 1) / c.step;
  if (c.chunks > ap.cap_parts || static_cast<long long>(s + 1) * ap.tiles_max * ap.nkv > ap.cap_units) {
    c.step = c.slabs;  // no place for the parts
    c.chunks = 1;
  }
  c.cost = static_cast<long long>(c.tiles) * c.slabs * ap.nkv;
  return c;
}

// A CTA's share: the chunks that begin in it.
template <int R, int SLAB>
struct Walk {
  long long x, hi;  // first slab still to be looked at, end of the share
  int s, unit, chunk, run;  // the run: chunks [chunk, run) of a unit of sequence s
  SeqSpan sp;
  SeqPlan plan;

  __device__ __forceinline__ void look(const CacheAttnParams& ap) {
    sp = seq_span(ap.seqs, s, ap.T);
    plan = seq_plan(ap, sp, s, ap.nq / ap.nkv, R, SLAB);
  }
  // the share [lo, hi) begins in sequence `seq`, whose first slab is `start`
  __device__ __forceinline__ void begin(const CacheAttnParams& ap, int seq, long long start, long long lo,
                                        long long end) {
    x = lo;
    hi = end;
    s = seq;
    look(ap);
    const long long rel = lo - start;
    unit = static_cast<int>(rel / plan.slabs);
    const int in = static_cast<int>(rel % plan.slabs);
    run = (in + plan.step - 1) / plan.step;  // the first chunk that begins here
    x += min(plan.slabs, run * plan.step) - in;
  }
  __device__ __forceinline__ bool next(const CacheAttnParams& ap) {
    if (x >= hi) return false;
    if (run == plan.chunks) {
      run = 0;
      ++unit;
    }
    while (unit >= plan.tiles * ap.nkv) {  // x < hi <= all slabs: there is another unit
      ++s;
      unit = run = 0;
      look(ap);
    }
    chunk = run;
    run = chunk + 1;  // shared memory joins the warps chunk by chunk
    x += min(plan.slabs, run * plan.step) - chunk * plan.step;
    return true;
  }
};

__device__ __forceinline__ PartsAt unit_parts(const CacheAttnParams& ap, const UnitAt& at) {
  const long long u = (static_cast<long long>(at.s) * ap.tiles_max + at.tile) * ap.nkv + at.h;
  return PartsAt{ap.parts + u * ap.place_floats, ap.part_stride, padded_rows(ap.part_rows)};
}

// The parts that this kernel leaves, for the join.
template <int R, int SLAB, bool ALONE>
struct RowsPlan {
  static constexpr int kRows = R;
  static constexpr bool kAlone = ALONE;
  __device__ static PartsAt place(const CacheAttnParams& ap, const SeqSpan&, const UnitAt& at) {
    return unit_parts(ap, at);
  }
  __device__ static int parts(const CacheAttnParams& ap, const SeqSpan& sp, int s, int) {
    const int n = seq_plan(ap, sp, s, ap.nq / ap.nkv, R, SLAB).chunks;
    return n > 1 ? n : 0;
  }
};

// Tokens of a slab: the more of them, the more independent work a warp has
// between two waits and the fewer instructions a token, as far as the registers
// reach (S^T takes 4 a 16 tokens and 8 rows).
constexpr int kSlab = 32, kStages = 2;

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2)
    cache_attn_rows(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CacheAttnParams ap) {
  constexpr int R = 8 * NT;          // rows of a tile
  constexpr int kKc = HD / 64;       // 16-byte units of K a thread reads a token
  constexpr int kMt = HD / 16;       // 16-dim blocks of O^T
  constexpr int kMb = kSlab / 16;    // 16-token blocks of S^T
  constexpr int kPart = kSlab * HD;  // bytes of a slab's K (or V)
  extern __shared__ uint8_t smem_raw[];
  __shared__ RowsShared<R, kStages> sh;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tid = threadIdx.x;
  const int group = ap.nq / ap.nkv, n_seqs = ap.seqs.n_seqs;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int i = 0; i < kWarps * kStages * 2; ++i) mbar_init(&sh.full[0][0][0] + i, 1);
    fence_barrier_init();
  }
  pdl_wait();
  pdl_trigger();

  // ---- the teams' shares: thread i adds up sequences [i c, (i + 1) c)
  {
    const int c = (n_seqs + kWarps * 32 - 1) / (kWarps * 32);
    const int s0 = min(n_seqs, static_cast<int>(threadIdx.x) * c), s1 = min(n_seqs, s0 + c);
    long long mine = 0;
    for (int i = s0; i < s1; ++i) {
      const SeqSpan sp = seq_span(ap.seqs, i, ap.T);
      if (!sp.ok && blockIdx.x == 0 && ap.status) atomicOr(ap.status, kStatusBadShape);
      mine += seq_plan(ap, sp, i, group, R, kSlab).cost;
    }
    long long before = mine;  // inclusive scan
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xFFFFFFFFu, before, o);
      if (lane >= o) before += y;
    }
    if (lane == 31) sh.scan[warp] = before;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh.scan[w];
      total += sh.scan[w];
    }
    before -= mine;
    const long long quot = total / gridDim.x, rem = total % gridDim.x, i = blockIdx.x;
    const long long lo = quot * i + min(i, rem), hi = lo + quot + (i < rem ? 1 : 0);
    if (threadIdx.x == 0) {
      sh.lo = lo;
      sh.hi = hi;
    }
    if (lo < hi && lo >= before && lo < before + mine) {  // the share begins in one of mine
      long long at = before;
      for (int q = s0; q < s1; ++q) {
        const long long cost = seq_plan(ap, seq_span(ap.seqs, q, ap.T), q, group, R, kSlab).cost;
        if (lo < at + cost) {
          sh.seq = q;
          sh.start = at;
          break;
        }
        at += cost;
      }
    }
    __syncthreads();
    if (sh.lo >= sh.hi) return;
  }
  Walk<R, kSlab> walk;
  walk.begin(ap, sh.seq, sh.start, sh.lo, sh.hi);
  uint32_t it = 0;  // slabs this warp has taken through its ring
  bool ok = true;   // no wait has run out
  while (walk.next(ap)) {
    const SeqSpan& sp = walk.sp;
    const SeqPlan& plan = walk.plan;
    const int s = walk.s, tile = walk.unit / ap.nkv, h = walk.unit % ap.nkv;
    int chunk = walk.chunk;
    const int run = walk.run, lo = chunk * plan.step, hi = min(plan.slabs, run * plan.step);
    const int rows = min(R, sp.n * group - tile * R);
    const int past = sp.len - sp.n;  // + i + 1: tokens seen by new token i
    const int seen = ap.causal ? min(sp.len, max(0, past + (tile * R + rows - 1) / group + 1)) : sp.len;
    const int end = min(hi, (seen + kSlab - 1) / kSlab);

    // ---- the ring's first slabs
    uint8_t* ring = smem + warp * (kStages * 2 * kPart);
    const int* bt = ap.seqs.block_tab + static_cast<long long>(s) * ap.seqs.max_pages;
    int slab = lo + warp;
    auto page_of = [&](int slab) { return slab < end ? bt[slab / (kPage / kSlab)] : 0; };
    auto good = [&](int page) { return page >= 0 && page < ap.kv_pages; };
    // K (v = 0) or V (v = 1) of a slab, the warp's n-th
    auto fetch = [&](int slab, int page, uint32_t n, int v) {
      if (slab < end && lane == 0) {
        uint64_t* bar = &sh.full[warp][n % kStages][v];
        if (good(page)) {
          const int row = (page * ap.nkv + h) * kPage + slab % (kPage / kSlab) * kSlab;
          mbar_arrive_expect_tx(bar, kPart);
          tma_load_2d(v ? &tmV : &tmK, bar, ring + n % kStages * (2 * kPart) + v * kPart, 0, row);
        } else {
          if (ap.status) atomicOr(ap.status, kStatusBadShape);
          mbar_arrive(bar);
        }
      }
    };
    int pages[kStages + 1];  // of the slabs from the current one on
#pragma unroll
    for (int i = 0; i <= kStages; ++i) pages[i] = page_of(slab + i * kWarps);
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      fetch(slab + i * kWarps, pages[i], it + i, 0);
      fetch(slab + i * kWarps, pages[i], it + i, 1);
    }
    auto scale_at = [&](const float* p, int page) {
      return p[static_cast<long long>(good(page) ? page : 0) * ap.nkv + h];
    };
    float ks_next = scale_at(ap.kscale, pages[0]), vs_next = scale_at(ap.vscale, pages[0]);

    // ---- queries: B operands, f16
    uint32_t qf[NT][HD / 16][2];
    float fac[NT][2];  // scale log2(e), undoing the row's own scaling, of columns 2t, 2t + 1
    int lim[NT][2];    // tokens that they see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g, row = tile * R + r;
      float undo = 1.0f;
      if (r < rows) {
        const T* qr = static_cast<const T*>(ap.q) + (sp.t0 + row / group) * ap.ldq +
                      static_cast<long long>(h * group + row % group) * HD;
        uint4 raw[kKc][2];
#pragma unroll
        for (int i = 0; i < kKc; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const T* src = qr + 16 * (kKc * t + i) + 8 * j;
            if (ap.vec) {
              raw[i][j] = *reinterpret_cast<const uint4*>(src);
            } else {
              T* e = reinterpret_cast<T*>(&raw[i][j]);
#pragma unroll
              for (int k = 0; k < 8; ++k) e[k] = src[k];
            }
          }
        if constexpr (H16Traits<T>::kBf16) {
          float big = 0.0f, shift = 1.0f;
#pragma unroll
          for (int i = 0; i < kKc; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int k = 0; k < 8; ++k)
                big = fmaxf(big, fabsf(h2f<T>(reinterpret_cast<const T*>(&raw[i][j])[k])));
          const unsigned quad = 0xFu << (lane & 28);
          big = fmaxf(big, __shfl_xor_sync(quad, big, 1));
          big = fmaxf(big, __shfl_xor_sync(quad, big, 2));
          const int e = (__float_as_int(big) >> 23) - 127;  // 2^e <= big
          // 2^(14 - e), in reach of a float for every finite row
          if (big > 0.0f && e < 128) {
            const int up = min(14 - e, 126);
            shift = __int_as_float((up + 127) << 23);
            undo = __int_as_float((127 - up) << 23);
          }
#pragma unroll
          for (int i = 0; i < kKc; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t* w = reinterpret_cast<uint32_t*>(&raw[i][j]);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const T* e2 = reinterpret_cast<const T*>(&w[k]);
                w[k] = cvt2_rn<__half>(make_float2(h2f<T>(e2[0]) * shift, h2f<T>(e2[1]) * shift));
              }
            }
        }
#pragma unroll
        for (int i = 0; i < kKc; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            qf[nt][4 * i + 2 * j][0] = raw[i][j].x;
            qf[nt][4 * i + 2 * j][1] = raw[i][j].y;
            qf[nt][4 * i + 2 * j + 1][0] = raw[i][j].z;
            qf[nt][4 * i + 2 * j + 1][1] = raw[i][j].w;
          }
      } else {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) qf[nt][k][0] = qf[nt][k][1] = 0u;
      }
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        fac[nt][c] = __shfl_sync(0xFFFFFFFFu, undo, 8 * t + 4 * c) * (ap.scale * kLog2e);
        const int cr = nt * 8 + 2 * t + c;
        // columns without a row: zeros that nothing masks and nobody reads
        lim[nt][c] = cr >= rows ? 0x7FFFFFFF : ap.causal ? max(0, past + (tile * R + cr) / group + 1) : sp.len;
      }
    }
    int all = 0x7FFFFFFF;  // tokens that every row sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) all = min(all, min(lim[nt][0], lim[nt][1]));
    all = __reduce_min_sync(0xFFFFFFFFu, all);

    for (; chunk < run; ++chunk) {
    float o[kMt][NT][4];
    float m[NT][2], l[NT][2];
    float up[NT][2];  // kLift - m
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      up[nt][0] = up[nt][1] = kLift;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < kMt; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
    }

    for (const int stop = min(end, (chunk + 1) * plan.step); slab < stop; slab += kWarps, ++it) {
      const float ks = ks_next, vs = usable_vscale(vs_next);
      const int have = good(pages[0]) ? min(kSlab, sp.len - slab * kSlab) : 0;
#pragma unroll
      for (int i = 0; i < kStages; ++i) pages[i] = pages[i + 1];
      pages[kStages] = page_of(slab + (kStages + 1) * kWarps);
      ks_next = scale_at(ap.kscale, pages[0]);
      vs_next = scale_at(ap.vscale, pages[0]);
      if (!mbar_wait_warp(&sh.full[warp][it % kStages][0], (it / kStages) & 1)) {
        ok = false;
        break;
      }
      const uint32_t kb = smem_u32(ring) + it % kStages * (2 * kPart), vb = kb + kPart;
      const float lv = lg2_approx(vs), ivs = rcp_approx(vs);

      float c[kMb][NT][4];
#pragma unroll
      for (int b = 0; b < kMb; ++b)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[b][nt][0] = c[b][nt][1] = c[b][nt][2] = c[b][nt][3] = 0.0f;
#pragma unroll
      for (int i = 0; i < kKc; ++i) {
        const int u = (kKc * t + i) ^ (HD == 128 ? g & 7 : (g >> 1) & 3);
#pragma unroll
        for (int b = 0; b < kMb; ++b) {
          const uint4 ka = lds128(kb + (16 * b + g) * HD + 16 * u);
          const uint4 kc = lds128(kb + (16 * b + g + 8) * HD + 16 * u);
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wc[4] = {kc.x, kc.y, kc.z, kc.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a[4];
            e4m3x4_f16x2(wa[j], a[0], a[2]);
            e4m3x4_f16x2(wc[j], a[1], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(c[b][nt], a, qf[nt][4 * i + j][0], qf[nt][4 * i + j][1]);
          }
        }
      }

      __syncwarp();  // K has been read
      fetch(slab + kStages * kWarps, pages[kStages - 1], it + kStages, 0);

      // ---- softmax of tokens 16 b + g, + 8 (c[0..1], c[2..3]) for columns 2t, 2t + 1
      const bool partial = (slab + 1) * kSlab > all || have < kSlab;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float f[2] = {ks * fac[nt][0], ks * fac[nt][1]};
#pragma unroll
        for (int b = 0; b < kMb; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) c[b][nt][e] = fmaf(c[b][nt][e], f[e & 1], lv);
      }
      if (partial) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int b = 0; b < kMb; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int at = 16 * b + g + (e >> 1) * 8;
              if (slab * kSlab + at >= lim[nt][e & 1] || at >= have) c[b][nt][e] = -INFINITY;
            }
      }
      float top[NT][2];  // of this thread's tokens
      bool over = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = fmaxf(c[0][nt][e], c[0][nt][e + 2]);
#pragma unroll
          for (int b = 1; b < kMb; ++b) top[nt][e] = fmaxf(top[nt][e], fmaxf(c[b][nt][e], c[b][nt][e + 2]));
          over |= top[nt][e] > m[nt][e] + kSlack;
        }
      if (__any_sync(0xFFFFFFFFu, over)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float big = top[nt][e];
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, w));
            if (big > m[nt][e]) {
              const float a = ex2_approx(m[nt][e] - big);
              m[nt][e] = big;
              up[nt][e] = kLift - big;
              l[nt][e] *= a;
#pragma unroll
              for (int i = 0; i < kMt; ++i) {
                o[i][nt][e] *= a;
                o[i][nt][e + 2] *= a;
              }
            }
          }
      }
      uint32_t pb[kMb][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < kMb; ++b) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = ex2_approx(c[b][nt][e] + up[nt][e & 1]);
            sum[e & 1] += p[e];
          }
          pb[b][nt][0] = movmatrix_trans(cvt2_rn<__half>(make_float2(p[0], p[1])));
          pb[b][nt][1] = movmatrix_trans(cvt2_rn<__half>(make_float2(p[2], p[3])));
        }
        l[nt][0] = fmaf(sum[0], ivs, l[nt][0]);
        l[nt][1] = fmaf(sum[1], ivs, l[nt][1]);
      }

      // ---- O^T += V^T P^T: tokens 2t, 2t + 1, 2t + 8, 2t + 9 of dims 2 kMt g ..
      if (!mbar_wait_warp(&sh.full[warp][it % kStages][1], (it / kStages) & 1)) {
        ok = false;
        break;
      }
#pragma unroll
      for (int b = 0; b < kMb; ++b) {
        uint32_t v[4][HD / 32];  // the four tokens' codes
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = 16 * b + 2 * t + (k & 1) + (k >> 1) * 8;
          if constexpr (HD == 128) {
            const uint4 d = lds128(vb + row * HD + 16 * (g ^ (row & 7)));
            v[k][0] = d.x;
            v[k][1] = d.y;
            v[k][2] = d.z;
            v[k][3] = d.w;
          } else {
            const uint32_t at = vb + row * HD + 16 * ((g >> 1) ^ ((row >> 1) & 3)) + 8 * (g & 1);
            asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v[k][0]), "=r"(v[k][1]) : "r"(at));
          }
        }
        if (partial) {
          // What lies past the sequence's end is not used, whatever it holds.  And
          // 0 . NaN is NaN: a NaN code that some rows do not see is taken out, and
          // put into the results of the rows that do.
          uint32_t nan[4];  // a bit for each of the thread's dims
          bool any = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            nan[k] = 0;
            const bool in = 16 * b + 2 * t + (k & 1) + (k >> 1) * 8 < have;
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) {
              if (!in) v[k][w] = 0;
#pragma unroll
              for (int y = 0; y < 4; ++y)
                if (((v[k][w] >> (8 * y)) & 0x7Fu) == 0x7Fu) {
                  nan[k] |= 1u << (4 * w + y);
                  v[k][w] &= ~(0xFFu << (8 * y));
                }
            }
            any |= nan[k] != 0;
          }
          if (__any_sync(0xFFFFFFFFu, any)) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              for (int from = 0; from < 4; ++from) {
                const uint32_t bits = __shfl_sync(0xFFFFFFFFu, nan[k], (lane & 28) + from);
                const int at = 16 * b + 2 * from + (k & 1) + (k >> 1) * 8;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if (slab * kSlab + at < lim[nt][e])
#pragma unroll
                      for (int i = 0; i < kMt; ++i) {
                        if (bits >> (2 * i) & 1) o[i][nt][e] = NAN;
                        if (bits >> (2 * i + 1) & 1) o[i][nt][e + 2] = NAN;
                      }
              }
          }
        }
#pragma unroll
        for (int w = 0; w < HD / 32; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t b01 = __byte_perm(v[0][w], v[1][w], half ? 0x7362 : 0x5140);
            const uint32_t b23 = __byte_perm(v[2][w], v[3][w], half ? 0x7362 : 0x5140);
            uint32_t a[4];
            e4m3x4_f16x2(b01, a[0], a[1]);
            e4m3x4_f16x2(b23, a[2], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(o[2 * w + half][nt], a, pb[b][nt][0], pb[b][nt][1]);
          }
      }
      __syncwarp();  // V has been read
      fetch(slab + kStages * kWarps, pages[kStages - 1], it + kStages, 1);
    }

    if (!ok)  // a wait ran out: nothing may still be on its way when the CTA ends
      for (uint32_t n = it; n <= it + kStages; ++n)
        if (slab + static_cast<int>(n - it) * kWarps < end) {
          mbar_wait_warp(&sh.full[warp][n % kStages][0], (n / kStages) & 1);
          mbar_wait_warp(&sh.full[warp][n % kStages][1], (n / kStages) & 1);
        }

    // ---- the warps' m, l and O
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], w);
        if (g == 0) {
          sh.m[warp][nt * 8 + 2 * t + e] = m[nt][e];
          sh.l[warp][nt * 8 + 2 * t + e] = l[nt][e];
        }
      }
    float* obuf = reinterpret_cast<float*>(smem);  // [warp][row][dim] over the ring
    {
      if (__syncthreads_or(!ok)) goto done;  // every slab has been read
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * t + e;
          if (r >= rows) continue;
          float big = sh.m[0][r];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) big = fmaxf(big, sh.m[w][r]);
          const float ref = big == -INFINITY ? 0.0f : big;
          const float a = ex2_approx(m[nt][e] - ref);
          float* dst = obuf + (warp * R + r) * HD + 2 * kMt * g;
#pragma unroll
          for (int i = 0; i < kMt / 2; ++i)
            *reinterpret_cast<float4*>(dst + 4 * i) = make_float4(
                o[2 * i][nt][e] * a, o[2 * i][nt][e + 2] * a, o[2 * i + 1][nt][e] * a, o[2 * i + 1][nt][e + 2] * a);
          if (warp == 0 && g == 0) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) sum += sh.l[w][r] * ex2_approx(sh.m[w][r] - ref);
            sh.cm[r] = big;
            sh.cl[r] = sum;
          }
        }
      __syncthreads();
    }
    // calls put(row, dim, four values) for all of O, f32
    auto each = [&](auto put) {
      {
        for (int i = tid; i < rows * (HD / 4); i += kWarps * 32) {
          float4 v = reinterpret_cast<float4*>(obuf)[i];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) {
            const float4 y = reinterpret_cast<float4*>(obuf + w * R * HD)[i];
            v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
          }
          put(i / (HD / 4), 4 * (i % (HD / 4)), v);
        }
      }
    };
    // calls put(row, m, l) for all rows
    auto each_row = [&](auto put) {
      if (tid < rows) put(tid, sh.cm[tid], sh.cl[tid]);
    };

    // ---- they are all there is, or a part
    const UnitAt at{s, tile, h, sp.t0};
    if (plan.chunks == 1) {
      each_row([&](int r, float big, float sum) { sh.inv[r] = close_row(ap, at, tile * R + r, big, sum); });
      __syncthreads();
      each([&](int r, int dim, float4 v) { finish_row<T, HD>(ap, at, tile * R + r, dim, v, sh.inv[r]); });
      __syncthreads();  // the sums are read before the next chunk's are written
    } else {
      const PartsAt parts = unit_parts(ap, at);
      float* mine = parts.base + static_cast<long long>(chunk) * parts.stride;
      const int l_at = parts.l_at;
      each([&](int r, int dim, float4 v) {
        __stcg(reinterpret_cast<float4*>(mine + 2 * l_at + r * HD + dim), v);
      });
      each_row([&](int r, float big, float sum) {
        __stcg(mine + r, big);
        __stcg(mine + l_at + r, sum);
      });
    }
    fence_proxy_async_smem();  // O is overwritten by the next chunk's copies
    __syncthreads();
    }
  }
done:
  if (!ok && lane == 0 && ap.status) atomicOr(ap.status, kStatusTimeout);
}

// Rows of a tile of the few-row kernel for sequences of up to `rows` rows.
int tile_rows(long long rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : 24; }

// The workspace of a unit, for caches of up to max_kv tokens.
struct PartSizes {
  int tiles, parts, rows, stride;
  long long place_floats;
};
PartSizes part_sizes(int nq, int nkv, int hd, int max_q, int max_kv) {
  PartSizes p;
  const long long rows = static_cast<long long>(max_q) * (nq / nkv);
  const int R = tile_rows(rows);
  const int tokens = std::max(1, max_kv);
  p.tiles = static_cast<int>((rows + R - 1) / R);
  p.parts = (tokens - 1) / chunk_tokens(tokens) + 1;
  if (tokens > kMaxParts * kChunk) p.parts = kMaxParts;  // a shorter cache may have as many
  p.rows = static_cast<int>(std::min<long long>(R, rows));
  p.stride = part_floats(p.rows, hd);
  p.place_floats = static_cast<long long>(p.parts) * p.stride;
  return p;
}

// CTAs of a few-row kernel that the GPU holds at once.
template <typename K>
int resident_ctas(K kern, size_t smem, cudaError_t* err) {
  int per = 0;
  *err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (*err == cudaSuccess) *err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, kWarps * 32, smem);
  return std::min(per, kMaxCtasPerSm) * device_sm_count();
}

template <typename T, int HD, int NT>
cudaError_t launch_rows(CacheAttnParams ap, void* ws, long long ws_bytes, int max_kv, cudaStream_t s) {
  constexpr int R = 8 * NT;
  // the ring, which also takes the warps' O, 4 kWarps R HD bytes; and 1 KB to align it
  constexpr int kSmem = kWarps * kStages * 2 * kSlab * HD + 1024;
  static_assert(kSmem - 1024 >= 4 * kWarps * R * HD, "the warps' O fits the ring");
  CUtensorMap tk, tv;
  const long long rows = static_cast<long long>(ap.kv_pages) * ap.nkv * kPage;
  if (rows > 0x7FFFFFFFll) return cudaErrorInvalidValue;  // TMA row coordinates
  // codes in pairs, as 16-bit elements
  const long long dims[2] = {HD / 2, rows}, stride[1] = {HD};
  const int box[2] = {HD / 2, kSlab}, step[2] = {1, 1};
  int rc = make_tmap_nd(&tk, ap.kpool, false, 2, dims, stride, box, step, HD);
  if (!rc) rc = make_tmap_nd(&tv, ap.vpool, false, 2, dims, stride, box, step, HD);
  if (rc) return static_cast<cudaError_t>(rc);
  auto kern = cache_attn_rows<T, HD, NT>;
  static std::atomic<int> resident[64];  // per instantiation and device
  int dev = 0;
  cudaGetDevice(&dev);
  int grid = resident[dev & 63];
  if (!grid) {
    cudaError_t e;
    grid = resident_ctas(kern, kSmem, &e);
    if (e != cudaSuccess) return e;
    resident[dev & 63] = grid;
  }
  const PartSizes ps = part_sizes(ap.nq, ap.nkv, HD, ap.seqs.max_q, max_kv);
  ap.tiles_max = ps.tiles;
  ap.cap_parts = ps.parts;
  ap.part_rows = ps.rows;
  ap.part_stride = ps.stride;
  ap.parts = static_cast<float*>(ws);
  ap.place_floats = ps.place_floats;
  ap.cap_units = ws ? ws_bytes / (4 * ps.place_floats) : 0;
  // no more CTAs than chunks, as far as max_kv tells
  const long long chunks = static_cast<long long>(ap.seqs.n_seqs) * ps.tiles * ap.nkv * ps.parts;
  grid = static_cast<int>(std::min<long long>(grid, chunks));
  cudaError_t e = launch_pdl(kern, dim3(grid), dim3(kWarps * 32), kSmem, s, tk, tv, ap);
  if (e == cudaSuccess && ps.parts > 1 && ap.cap_units > 0) {
    constexpr bool kMany = R > 8;  // rows enough for a warp each
    e = kMany && ps.parts <= kJoinAlone ? launch_join<T, HD, RowsPlan<R, kSlab, kMany>>(ap, s)
                                        : launch_join<T, HD, RowsPlan<R, kSlab, false>>(ap, s);
  }
  return e;
}

template <typename T, int HD>
cudaError_t launch_any(const CacheAttnParams& ap, void* ws, long long ws_bytes, int max_kv, cudaStream_t s) {
  const int R = tile_rows(static_cast<long long>(ap.seqs.max_q) * (ap.nq / ap.nkv));
  if (R == 8) return launch_rows<T, HD, 1>(ap, ws, ws_bytes, max_kv, s);
  if (R == 16) return launch_rows<T, HD, 2>(ap, ws, ws_bytes, max_kv, s);
  return launch_rows<T, HD, 3>(ap, ws, ws_bytes, max_kv, s);
}

// Rows of a K/V head and sequence up to which the few-row kernel is used: as far as
// its registers reach.  24 rows over 5000 tokens each (16/8 heads of 128), 16 sessions:
// 80 us here, 124 on the tcgen05 kernel, which pads them to 128 rows; 16 rows: 65 and
// 122.  One session of 24 rows over 8192 tokens: 38 and 42, over 131,000: 104 and 156.
constexpr int kFewRows = 24;

}  // namespace

long long cache_rows_workspace(int nqh, int nkvh, int hd, int n_seqs, int max_q, int max_kv) {
  const PartSizes p = part_sizes(nqh, nkvh, hd, max_q, max_kv);
  if (p.parts == 1) return 0;
  return places_bytes(static_cast<long long>(n_seqs) * p.tiles, nkvh, p.place_floats);
}

int cache_attention_rows(const CacheAttnParams& ap, int hd, bool bf16, int max_kv, void* ws,
                         long long ws_bytes, cudaStream_t s) {
  if (bf16)
    return hd == 128 ? launch_any<__nv_bfloat16, 128>(ap, ws, ws_bytes, max_kv, s)
                     : launch_any<__nv_bfloat16, 64>(ap, ws, ws_bytes, max_kv, s);
  return hd == 128 ? launch_any<__half, 128>(ap, ws, ws_bytes, max_kv, s)
                   : launch_any<__half, 64>(ap, ws, ws_bytes, max_kv, s);
}

long long cache_attention_workspace(int nqh, int nkvh, int hd, int n_seqs, int max_q, int max_kv) {
  if (nkvh <= 0 || nqh < nkvh || n_seqs <= 0 || max_q <= 0 || (hd != 64 && hd != 128)) return 0;
  const bool few = static_cast<long long>(max_q) * (nqh / nkvh) <= kFewRows;
  return few ? cache_rows_workspace(nqh, nkvh, hd, n_seqs, max_q, max_kv)
             : cache_tiles_workspace(nqh, nkvh, hd, n_seqs, max_q, max_kv);
}

int cache_attention(const void* q, long long ldq, long long T, int nqh, int nkvh, int hd,
                    const SeqMap& seqs, int max_q, int max_kv, const void* kpool, const void* vpool,
                    int kv_pages, const float* kscale, const float* vscale, float scale, bool causal,
                    void* out, long long ldo, float* lse, void* workspace,
                    long long workspace_bytes, bool bf16, unsigned* status, cudaStream_t s) {
  if (T <= 0 || seqs.n_seqs <= 0 || max_q <= 0) return 0;
  max_q = static_cast<int>(std::min<long long>(max_q, T));  // no sequence has more
  max_kv = static_cast<int>(std::min(static_cast<long long>(max_kv), 64ll * seqs.max_pages));
  CacheAttnParams ap{};
  ap.q = q;
  ap.ldq = ldq;
  ap.T = T;
  ap.nq = nqh;
  ap.nkv = nkvh;
  ap.seqs = seqs;
  ap.seqs.max_q = max_q;
  ap.kpool = static_cast<const uint8_t*>(kpool);
  ap.vpool = static_cast<const uint8_t*>(vpool);
  ap.kv_pages = kv_pages;
  ap.kscale = kscale;
  ap.vscale = vscale;
  ap.scale = scale;
  ap.causal = causal;
  ap.out = out;
  ap.ldo = ldo;
  ap.lse = lse;
  ap.status = status;
  ap.vec = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0) &&
           ((ldq | ldo) % 8 == 0);
  const bool few = static_cast<long long>(max_q) * (nqh / nkvh) <= kFewRows;
  const int rc = few ? cache_attention_rows(ap, hd, bf16, max_kv, workspace, workspace_bytes, s)
                     : cache_attention_tiles(ap, hd, bf16, max_kv, workspace, workspace_bytes, s);
  return rc ? rc : (int)cudaGetLastError();
}

}  // namespace qa
