// Attention over a paged int8 cache where a sequence has many query rows (chunks of a prompt, whole prompts): tiles of 128 rows on tcgen05.
// (Included by intfa_paged_attn.cu inside namespace intfa, after the shared helpers.)
//
// A unit is (sequence, K/V head, 256 rows; 128 at head dim 256): two tiles of 128 rows, each the rows of as many whole tokens as fit, all query heads of the
// K/V head packed.  The units' chunks of 64 keys (those that the last row of a unit sees) are dealt out to the CTAs, one an SM, in equal
// contiguous shares; parts of units that are cut go to scratch and combine_tiles_kernel adds them up, as in the kernel for few rows.
//
// Four sequences of up to 512 new rows, 32 / 8 heads x 128, and up to 8192 keys: 4 * rows * keys * D operations, 94 us at the fp16 rate of P V and S
// (70 with S at the int8 rate, 67 for the exp2 alone), 217 here; six prompts of up to 4096 306 and 695.  Bound by the latency of the chain from
// S to P (scores, exponents, exp2, sums, P) with two softmax warps a scheduler: issue slots 47 %, exp2 40 %, tensor pipe 31 %.  Eight sequences of up to
// 256 rows and 4096 keys: 64 channels, 32 / 8 heads 19 and 115, 256 channels, 16 / 4 heads 38 and 122 (one tile: four of the eight softmax warps have
// no rows).  Spilled: 32 bytes at 128 channels, 40 at 256, 12 at 64.
//
// 512 threads:
//   warp 0       TMA: Q once per unit (heads x tokens boxes), K and V pages of 8 rows and more each
//   warp 1       MMA issuer.  For each tile in turn: P V of a chunk, S = Q K^T of the one after the next
//   warp 2       TMEM; K scales, log2 and reciprocal of the V scales of a chunk into a ring
//   warp 3       goes through the units and publishes them
//   warps 4-7    V from int8 (as TMA left it) to fp16 in the MN-major tiles that P V takes
//   warps 8-11, 12-15   softmax of tile 0 and of tile 1, one thread a row
// TMEM: two S buffers of each tile, P (fp16) over the scores it was made of, two accumulators of D columns.  S is two chunks ahead of P V.
//
// The arithmetic is that of the kernel for few rows: w = p v_scale relative to a reference near its running maximum, P = fp16(w), l = sum p
// relative to a reference of its own.  The reference of w follows only where the sum of p times the largest V scale does not say that all w
// are below 2^15: the accumulator is rescaled in a few chunks of a unit, and w below 2^15 (fp16 ends at 65504) loses no bits in fp16.
// Where a chunk's V scales are within 2^60 of what the references differ by (nearly always: the general way is for zeros and for scales of very
// different sizes; there p is summed up by itself and its reference follows where it gets 2^8 ahead) p = w / v_scale needs no exp2 of its own.
// S starts from the bit pattern of 1.5*2^23, written by a small fp16 MMA, and reads as fp32 1.5*2^23 + dot.
#pragma once

constexpr int kTileRows = 128;
constexpr int kTileKeys = 64;                     // keys of a chunk: two S buffers of two tiles and two accumulators of 128 fill TMEM
constexpr int kTileThreads = 512, kTileLaunch = 128, kTileService = 56, kTileConvert = 72, kTileSoftmax = 192;        // registers
static_assert(128 * (kTileService + kTileConvert) + 256 * kTileSoftmax <= kTileThreads * kTileLaunch, "setmaxnreg budget");

// a unit, or the part of it that a CTA does
struct __align__(16) TileUnit {
  long long lim0;              // causal: the last key that the unit's first token sees
  int t0, tokens;              // its first token among all, and how many it has
  int head, s, keys;           // K/V head; sequence; keys that are looked at
  int c0, c1;                  // chunks to do; c0 < 0: no more units
  int slot;                    // of its part in scratch; -1: the unit is done here
  int pad[2];
};
static_assert(sizeof(TileUnit) == 48, "unit");

template <bool B>
struct Flag {
  static constexpr bool value = B;
};

struct TileSeq {
  int t0, n, keys, tiles, uniform;
  long long first;
  bool bad;
};
__device__ __forceinline__ TileSeq tile_seq_of(const PParams& p, int s) {
  const Seq q = seq_of(p, s);
  TileSeq w;
  w.t0 = q.t0;
  w.n = q.n;
  w.keys = q.keys;
  w.bad = q.bad;
  w.first = q.len - q.n;
  w.tiles = (q.n + p.unit_tokens - 1) / p.unit_tokens;
  w.uniform = !p.causal || w.first < 0 || q.len > q.keys;        // every unit goes over all keys (for the odd lengths, masked)
  return w;
}
template <int G>
__device__ __forceinline__ int tile_chunks(const PParams& p, const TileSeq& q, int tile) {
  long long vis = q.keys;
  if (!q.uniform) vis = min(vis, q.first + (long long)(tile + 1) * p.unit_tokens);
  return vis > G ? (int)((vis + G - 1) / G) : 1;
}
// sum of floor((a t + b) / m), t = 0 .. n-1 (a, b >= 0): whole parts out, then the points below the line counted along the other axis, which
// swaps a and m as Euclid's algorithm does
__device__ __noinline__ long long floor_sum(long long n, long long m, long long a, long long b) {
  long long sum = 0;
  while (n > 0) {
    sum += n * (n - 1) / 2 * (a / m) + n * (b / m);
    a %= m;
    b %= m;
    const long long y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const long long t = m;
    m = a;
    a = t;
  }
  return sum;
}
// chunks of the first k units of a K/V head
template <int G>
__device__ inline long long tile_chunks_before(const PParams& p, const TileSeq& q, int k) {
  if (k <= 0) return 0;
  if (q.uniform) return (long long)k * tile_chunks<G>(p, q, 0);
  const int full = k < q.tiles ? k : q.tiles - 1;
  const long long step = p.unit_tokens;
  return floor_sum(full, G, step, q.first + step + G - 1) + (k == q.tiles ? tile_chunks<G>(p, q, q.tiles - 1) : 0);
}

template <int D>
struct TileCfg {
  // (256 channels: an accumulator of 256 columns, so one tile of rows, and half of the buffers)
  static constexpr bool WIDE = D == 256;
  static constexpr int G = kTileKeys, THREADS = kTileThreads, TILES = WIDE ? 1 : 2, NK = WIDE ? 3 : 5, NV8 = WIDE ? 2 : 4, NV = WIDE ? 2 : 3, NSC = 8, NU = 4;
  static constexpr int PANEL = D < 128 ? D : 128, PANELS = D / PANEL;   // Q, K and the int8 V lie in panels of at most 128 bytes a row
  // start-address offset (16-byte units) of the kk-th 32-byte slice of an operand of so many rows
  __host__ __device__ static constexpr uint32_t slice(int kk, int rows) { return (uint32_t)((kk / 4) * ((rows * PANEL) >> 4) + 2 * (kk % 4)); }
  static constexpr int Q_BYTES = kTileRows * D, K_BYTES = G * D, V_BYTES = G * D * 2;
  static constexpr int SC_FLOATS = 3 * G + 4;
  static constexpr int OFF_Q = 0, OFF_K = OFF_Q + TILES * Q_BYTES, OFF_V8 = OFF_K + NK * K_BYTES, OFF_V = OFF_V8 + NV8 * K_BYTES;
  static constexpr int OFF_ARM = OFF_V + NV * V_BYTES;
  static constexpr int OFF_SC = OFF_ARM + 4096;
  static constexpr int OFF_UNIT = OFF_SC + NSC * SC_FLOATS * 4;
  static constexpr int OFF_PRE = OFF_UNIT + NU * (int)sizeof(TileUnit);
  static constexpr int NBARS = 4 + 2 * NK + 2 * NV8 + 2 * NV + 2 * NSC + 2 * NU + 12;
  static constexpr int OFF_BAR = OFF_PRE + (THREADS + 2) * 8;
  static constexpr int OFF_MISC = OFF_BAR + NBARS * 8;
  static constexpr int OFF_OUT = (OFF_MISC + 32 + 127) / 128 * 128;      // 32 rows x 64 channels of each softmax warp, on their way out
  static constexpr int SMEM = OFF_OUT + 8 * 4096 + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static_assert(OFF_UNIT % 16 == 0 && OFF_SC % 16 == 0 && OFF_PRE % 8 == 0, "alignment");
  static constexpr int COL_S = 0, COL_O = 4 * G;
  static_assert(COL_O + TILES * D <= 512, "TMEM columns");
  static constexpr uint64_t SWZ_QK = PANEL == 128 ? kSwz128 : kSwz64;
  static constexpr uint32_t IDESC_QK = make_idesc(2, 1, 1, 0, 0, kTileRows, G);
  static constexpr uint32_t IDESC_PV = make_idesc(1, 0, 0, 0, 1, kTileRows, D);
  static constexpr uint32_t IDESC_ARM = make_idesc(1, 0, 0, 0, 0, kTileRows, G);
};

enum TileWait { TW_UNIT = 65, TW_UEMPTY, TW_QE, TW_KE, TW_V8E, TW_QF, TW_KF, TW_VF, TW_P, TW_SCE, TW_V8F, TW_VE, TW_SC, TW_S, TW_O };

template <int D>
__global__ void __launch_bounds__(kTileThreads, 1) paged_tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                                                            const __grid_constant__ CUtensorMap tmV, const PParams p) {
  using C = TileCfg<D>;
  constexpr int G = C::G;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t bars = smem_u32(smem + C::OFF_BAR);
  auto BAR = [&](int i) { return bars + 8u * i; };
  constexpr int B_QF = 0, B_QE = 2;                              // [2] TMA: Q tile landed; commit: its last S is done
  constexpr int B_KF = 4, B_KE = B_KF + C::NK;                   // TMA; commit
  constexpr int B_V8F = B_KE + C::NK, B_V8E = B_V8F + C::NV8;    // TMA; converting warps (4)
  constexpr int B_VF = B_V8E + C::NV8, B_VE = B_VF + C::NV;      // converting warps (4); commit
  constexpr int B_SCF = B_VE + C::NV, B_SCE = B_SCF + C::NSC;    // scale loader; softmax warps (8)
  constexpr int B_UF = B_SCE + C::NSC, B_UE = B_UF + C::NU;      // unit published; taken over by TMA, MMA, scale, converting, softmax warps (15)
  constexpr int B_S = B_UE + C::NU, B_P = B_S + 4, B_O = B_P + 4;        // [tile][buffer of the chunk] commit: S; softmax warps of the tile (4): S read, P written; commit: P V
  static_assert(B_O + 4 == C::NBARS, "barriers");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 8);
  TileUnit* units = reinterpret_cast<TileUnit*>(smem + C::OFF_UNIT);
  long long* pre = reinterpret_cast<long long*>(smem + C::OFF_PRE);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(BAR(B_QF + i), 1);
      mbar_init(BAR(B_QE + i), 1);
      mbar_init(BAR(B_S + 2 * i), 1);
      mbar_init(BAR(B_S + 2 * i + 1), 1);
      mbar_init(BAR(B_P + 2 * i), 4);
      mbar_init(BAR(B_P + 2 * i + 1), 4);
      mbar_init(BAR(B_O + 2 * i), 1);
      mbar_init(BAR(B_O + 2 * i + 1), 1);
    }
    for (int i = 0; i < C::NK; ++i) {
      mbar_init(BAR(B_KF + i), 1);
      mbar_init(BAR(B_KE + i), 1);
    }
    for (int i = 0; i < C::NV8; ++i) {
      mbar_init(BAR(B_V8F + i), 1);
      mbar_init(BAR(B_V8E + i), 4);
    }
    for (int i = 0; i < C::NV; ++i) {
      mbar_init(BAR(B_VF + i), 4);
      mbar_init(BAR(B_VE + i), 1);
    }
    for (int i = 0; i < C::NSC; ++i) {
      mbar_init(BAR(B_SCF + i), 1);
      mbar_init(BAR(B_SCE + i), 8);
    }
    for (int i = 0; i < C::NU; ++i) {
      mbar_init(BAR(B_UF + i), 1);
      mbar_init(BAR(B_UE + i), 15);
    }
    abort_flag[0] = 0;
    abort_flag[1] = (int)(1u << 31);
    mbar_init_fence();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  // the constant operand whose product with itself is 1.5*2^23 everywhere: each row's 16 values are (1024, 1024, 2048, 0 ..) twice
  if (threadIdx.x < 256) reinterpret_cast<uint4*>(smem + C::OFF_ARM)[threadIdx.x] = make_uint4(0x64006400u, 0x00006800u, 0u, 0u);
  fence_proxy_async_smem();
  if (warp == 2) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
    tc_fence_before();
  }
  pdl_wait();
  pdl_launch();
  // ---- the row of all chunks: thread i counts the sequences i*seg .. (i+1)*seg - 1
  const int seg = (p.S + C::THREADS - 1) / C::THREADS;
  {
    long long c = 0;
    bool bad = false;
    for (int s = threadIdx.x * seg; s < (threadIdx.x + 1) * seg && s < p.S; ++s) {
      const TileSeq q = tile_seq_of(p, s);
      if (q.n > 0) c += tile_chunks_before<G>(p, q, q.tiles) * p.Hkv;
      bad |= q.bad;
    }
    if (bad && p.status && blockIdx.x == 0) atomicCAS(p.status, 0, kStatusBadIndex);
    pre[threadIdx.x + 1] = c;
    if (threadIdx.x == 0) pre[0] = 0;
  }
  __syncthreads();
  if (warp == 0) {
    long long c0 = 0;
    for (int w = 0; w < C::THREADS / 32; ++w) {
      long long c = pre[w * 32 + lane + 1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c += x;
      }
      pre[w * 32 + lane + 1] = c + c0;
      c0 += __shfl_sync(0xffffffffu, c, 31);
    }
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_uniform(*tmem_slot);
  const long long total = pre[C::THREADS];
  long long share = (total + p.workers - 1) / p.workers;
  if (share < p.least) share = p.least;
  const int code_hi = (int)(blockIdx.x << 8);
  auto wait = [&](int bar, uint32_t parity, int code) { return mbar_wait_warp(BAR(bar), parity, abort_flag, p.status, code_hi | code); };
  uint32_t useq = 0;
  // the next unit, or false
  auto next_unit = [&](TileUnit& u) {
    const uint32_t slot = useq % C::NU;
    if (!wait(B_UF + slot, (useq / C::NU) & 1u, TW_UNIT)) return false;
    ++useq;
    u = units[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(BAR(B_UE + slot));
    u.t0 = warp_uniform(u.t0);
    u.tokens = warp_uniform(u.tokens);
    u.head = warp_uniform(u.head);
    u.s = warp_uniform(u.s);
    u.keys = warp_uniform(u.keys);
    u.c0 = warp_uniform(u.c0);
    u.c1 = warp_uniform(u.c1);
    u.slot = warp_uniform(u.slot);
    return u.c0 >= 0;
  };
  const int page_mask = (1 << p.page_log) - 1;
  auto bad_page = [&](int page) { return page < 0 || page >= p.pages; };

  if (warp < 4) {
    reg_dealloc<kTileService>();
    if (warp == 3) {
      // ------------------------------------------------------------------ units
      const long long begin = (long long)blockIdx.x * share;
      const long long end = begin + share < total ? begin + share : total;
      long long pos = begin;
      int s = 0, head = 0, tile = 0;
      TileSeq q;
      q.n = q.tiles = 0;
      UnitPart part;
      part.open = 0;
      if (pos < end) {
        const int i = find_last(C::THREADS, begin, [&](int j) { return pre[j]; });
        long long off = begin - pre[i];
        for (s = i * seg;; ++s) {
          q = tile_seq_of(p, s);
          const long long c = q.n > 0 ? tile_chunks_before<G>(p, q, q.tiles) * p.Hkv : 0;
          if (off < c || s + 1 >= p.S) break;
          off -= c;
        }
        const long long per_head = tile_chunks_before<G>(p, q, q.tiles);
        head = (int)(off / per_head);
        off -= head * per_head;
        int lo = 0, hi = q.tiles;                              // the last tile whose chunks begin at or before `off`
        while (hi - lo > 1) {
          const int mid = (lo + hi) / 2;
          if (tile_chunks_before<G>(p, q, mid) <= off) lo = mid; else hi = mid;
        }
        tile = lo;
        pos = begin - (off - tile_chunks_before<G>(p, q, tile));  // where the first unit begins
      }
      bool ok = true;
      uint32_t seq = 0;
      const TileUnit none = {0, 0, 0, 0, 0, 0, -1, -1, -1, {0, 0}};
      while (ok) {
        TileUnit u = none;
        if (pos < end) {
          const int n = tile_chunks<G>(p, q, tile), token = tile * p.unit_tokens;
          u.lim0 = p.causal ? q.first + token : (long long)q.keys;
          u.t0 = q.t0 + token;
          u.tokens = min(p.unit_tokens, q.n - token);
          u.head = head;
          u.s = s;
          u.keys = q.keys;
          u.c0 = pos < begin ? (int)(begin - pos) : 0;
          u.c1 = pos + n > end ? (int)(end - pos) : n;
          const bool starts = pos >= begin, ends = pos + n <= end;
          u.slot = starts && ends ? -1 : 2 * (int)blockIdx.x + (starts ? 1 : 0);
          if (starts && !ends) {
            part.open = 1;
            set_parts(part, pos, pos + n, share, total, 1);
            part.token = u.t0;
            part.tokens = u.tokens;
            part.row = 0;
            part.head = head;
          }
          pos += n;
          if (++tile == q.tiles) {
            tile = 0;
            if (++head == p.Hkv) {
              head = 0;
              if (pos < end) {
                do q = tile_seq_of(p, ++s); while (q.n == 0 && s + 1 < p.S);
              }
            }
          }
        }
        const uint32_t slot = seq % C::NU;
        if (seq >= C::NU) ok = wait(B_UE + slot, (seq / C::NU - 1) & 1u, TW_UEMPTY);
        if (!ok) break;
        if (lane == 0) {
          units[slot] = u;
          mbar_arrive(BAR(B_UF + slot));
        }
        ++seq;
        if (u.c0 < 0) break;
      }
      if (lane == 0) p.units[blockIdx.x] = part;
    } else if (warp == 0) {
      // ------------------------------------------------------------------ TMA
      uint32_t kit = 0, vit = 0, uit = 0;                      // chunks of K, of V, units so far
      uint32_t qit1 = 0;                                       // units with a second tile
      const int box_rows = 1 << p.box_log, boxes = G >> p.box_log;
      const uint32_t sQ = smem_u32(smem + C::OFF_Q), sK = smem_u32(smem + C::OFF_K), sV8 = smem_u32(smem + C::OFF_V8);
      const uint32_t q_box = (uint32_t)(p.tile_tokens * p.ratio * D);
      TileUnit u;
      bool ok = true;
      while (ok && next_unit(u)) {
        const int* table = p.table + (long long)u.s * p.table_stride;
        const int two = u.tokens > p.tile_tokens;
        for (int i = 0; i <= two && ok; ++i) {
          const uint32_t n = i ? qit1 : uit;
          ok = wait(B_QE + i, (n & 1u) ^ 1u, TW_QE);
          if (ok && lane == 0) {
            mbar_expect_tx(BAR(B_QF + i), q_box);
            for (int pn = 0; pn < C::PANELS; ++pn)
              tma_load_4d(sQ + i * C::Q_BYTES + pn * (kTileRows * C::PANEL), &tmQ, BAR(B_QF + i), pn * C::PANEL, u.head * p.ratio, u.t0 + i * p.tile_tokens, 0);
          }
          __syncwarp();
          if (ok && i == 0) ++uit;
          if (ok && i == 1) ++qit1;
        }
        // lane j: the page of box j of the next chunk
        auto look_up = [&](int c) {
          const int key = c * G + lane * box_rows;
          return lane < boxes && c < u.c1 && key < u.keys ? table[key >> p.page_log] : 0;
        };
        int next = look_up(u.c0);
        for (int c = u.c0; c < u.c1 && ok; ++c) {
          int page = next;
          next = look_up(c + 1);
          if (bad_page(page)) {
            if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
            page = p.pages;                                    // (one past the last: the copies are zeros, and the scales leave them out)
          }
          const int key0 = c * G, full = max(0, min(boxes, (u.keys - key0 + box_rows - 1) >> p.box_log));
          const int slot = (key0 + lane * box_rows) & page_mask;
          const uint32_t bytes = (uint32_t)full * box_rows * D;
          const uint32_t k = kit % C::NK, v = vit % C::NV8;
          ok = wait(B_KE + k, ((kit / C::NK) & 1u) ^ 1u, TW_KE);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(BAR(B_KF + k), bytes);
          __syncwarp();
          if (lane < full)
            for (int pn = 0; pn < C::PANELS; ++pn)
              tma_load_4d(sK + k * C::K_BYTES + (pn * G + lane * box_rows) * C::PANEL, &tmK, BAR(B_KF + k), pn * C::PANEL, slot, u.head, page);
          __syncwarp();
          ++kit;
          ok = wait(B_V8E + v, ((vit / C::NV8) & 1u) ^ 1u, TW_V8E);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(BAR(B_V8F + v), bytes);
          __syncwarp();
          if (lane < full)
            for (int pn = 0; pn < C::PANELS; ++pn)
              tma_load_4d(sV8 + v * C::K_BYTES + (pn * G + lane * box_rows) * C::PANEL, &tmV, BAR(B_V8F + v), pn * C::PANEL, slot, u.head, page);
          __syncwarp();
          ++vit;
        }
      }
      if (*abort_flag) {                                       // a wait ran out: what was asked for comes before the CTA goes, or not at all
        for (uint32_t i = kit > C::NK ? kit - C::NK : 0; i < kit; ++i) mbar_drain(BAR(B_KF + i % C::NK), (i / C::NK) & 1u);
        for (uint32_t i = vit > C::NV8 ? vit - C::NV8 : 0; i < vit; ++i) mbar_drain(BAR(B_V8F + i % C::NV8), (i / C::NV8) & 1u);
        if (uit > 0) mbar_drain(BAR(B_QF), (uit - 1) & 1u);
        if (qit1 > 0) mbar_drain(BAR(B_QF + 1), (qit1 - 1) & 1u);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA
      const uint32_t sQ = smem_u32(smem + C::OFF_Q), sK = smem_u32(smem + C::OFF_K), sV = smem_u32(smem + C::OFF_V);
      const uint64_t descQ = make_smem_desc(sQ, 16, 8 * C::PANEL, C::SWZ_QK), descK = make_smem_desc(sK, 16, 8 * C::PANEL, C::SWZ_QK);
      const uint64_t descV = make_smem_desc(sV, D > 64 ? G * 128 : 16, 8 * 128, kSwz128);
      const uint64_t descArm = make_smem_desc(smem_u32(smem + C::OFF_ARM), 128, 256, 0);
      uint32_t kit = 0, vit = 0;                               // chunks of K, of V
      uint32_t uit = 0, sit = 0, pit = 0;                      // bit i: units, S tiles of tile i mod 2; bits 2i, 2i + 1: P tiles mod 4
      TileUnit u;
      bool ok = true;
      // S of a chunk of tile i into its buffer `buf`
      auto scores = [&](int i, uint32_t buf, uint32_t k, bool last) {
        const uint32_t tS = tmem + C::COL_S + (2 * i + buf) * G;
        umma_f16(tS, descArm, descArm, C::IDESC_ARM, 0);
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)
          umma_i8(tS, descQ + (uint64_t)(i * (C::Q_BYTES >> 4) + C::slice(kk, kTileRows)), descK + (uint64_t)(k * (C::K_BYTES >> 4) + C::slice(kk, G)), C::IDESC_QK,
                  1);
        umma_commit(BAR(B_S + 2 * i + buf));
        if (last) umma_commit(BAR(B_QE + i));
      };
      while (ok && next_unit(u)) {
        const int n = u.c1 - u.c0, two = u.tokens > p.tile_tokens;
#pragma unroll 1
        for (int j = 0; j < 2 && j < n && ok; ++j) {
          const uint32_t k = kit % C::NK;
          ok = wait(B_KF + k, (kit / C::NK) & 1u, TW_KF);
#pragma unroll 1
          for (int i = 0; i <= two && ok; ++i) {
            if (j == 0) ok = wait(B_QF + i, uit >> i & 1u, TW_QF);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              scores(i, sit >> i & 1u, k, j + 1 == n);
              if (i == two) umma_commit(BAR(B_KE + k));
            }
            __syncwarp();
            sit ^= 1u << i;
          }
          ++kit;
        }
        uit ^= two ? 3u : 1u;
#pragma unroll 1
        for (int j = 0; j < n && ok; ++j) {
          const uint32_t k = kit % C::NK, v = vit % C::NV;
          const bool more = j + 2 < n;
          ok = wait(B_VF + v, (vit / C::NV) & 1u, TW_VF);
          if (ok && more) ok = wait(B_KF + k, (kit / C::NK) & 1u, TW_KF);
#pragma unroll 1
          for (int i = 0; i <= two && ok; ++i) {
            // (a buffer's barrier: warps whose S is there may be a chunk ahead of the others)
            const uint32_t buf = pit >> (2 * i) & 1u;
            ok = wait(B_P + 2 * i + buf, pit >> (2 * i + 1) & 1u, TW_P);
            if (!ok) break;
            pit = (pit & ~(3u << (2 * i))) | (((pit >> (2 * i)) + 1u & 3u) << (2 * i));
            tc_fence_after();
            const uint32_t tP = tmem + C::COL_S + (2 * i + buf) * G, tO = tmem + C::COL_O + i * D;
            if (elect_one()) {
              const uint64_t vd = descV + (uint64_t)(v * (C::V_BYTES >> 4));
#pragma unroll
              for (int kk = 0; kk < G / 16; ++kk)
                umma_f16_ts(tO, tP + kk * 16, vd + (uint64_t)(kk * ((16 * 128) >> 4)), C::IDESC_PV, j > 0 || kk > 0 ? 1u : 0u);
              umma_commit(BAR(B_O + 2 * i + buf));
              // (the tensor core takes them in this order: S of the chunk after the next comes over P when the P V that reads it is done)
              if (more) scores(i, buf, k, j + 3 == n);
              if (i == two) {
                umma_commit(BAR(B_VE + v));
                if (more) umma_commit(BAR(B_KE + k));
              }
            }
            __syncwarp();
            if (more) sit ^= 1u << i;
          }
          ++vit;
          if (more) ++kit;
        }
      }
    } else {
      // ------------------------------------------------------------------ scales
      uint32_t it = 0;
      TileUnit u;
      bool ok = true;
      while (ok && next_unit(u)) {
        const int* table = p.table + (long long)u.s * p.table_stride;
        const float* ks = p.ks + u.head * p.ksH;
        const float* vs = p.vs + u.head * p.vsH;
        constexpr int N = G / 32;
        // pages two chunks ahead, scales one chunk ahead of what is written
        int page[N];
        float a[N], b[N], na[N], nb[N];
        auto look_up = [&](int c) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int key = c * G + i * 32 + lane;
            page[i] = c < u.c1 && key < u.keys ? table[key >> p.page_log] : -1;
          }
        };
        auto fetch = [&](int c) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int key = c * G + i * 32 + lane, blk = (key & page_mask) >> p.block_log;
            na[i] = 0.f;
            nb[i] = 1.f;
            if (c < u.c1 && key < u.keys) {
              nb[i] = -INFINITY;                               // a page outside the cache: the key does not count
              if (!bad_page(page[i])) {
                na[i] = ks[page[i] * p.ksP + blk * p.ksB];
                nb[i] = vs[page[i] * p.vsP + blk * p.vsB];
              }
            }
          }
        };
        look_up(u.c0);
        fetch(u.c0);
        look_up(u.c0 + 1);
        for (int c = u.c0; c < u.c1 && ok; ++c, ++it) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            a[i] = na[i];
            b[i] = nb[i];
          }
          fetch(c + 1);
          look_up(c + 2);
          const uint32_t slot = it % C::NSC;
          float* sc = reinterpret_cast<float*>(smem + C::OFF_SC) + slot * C::SC_FLOATS;
          ok = wait(B_SCE + slot, ((it / C::NSC) & 1u) ^ 1u, TW_SCE);
          if (!ok) break;
          float lo = INFINITY, hi = -INFINITY;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const bool gap = b[i] == -INFINITY;                // logarithm -inf, reciprocal 0: neither w nor p of it
            const float l = gap ? -INFINITY : log2_approx(b[i]);
            sc[i * 32 + lane] = a[i];
            sc[G + i * 32 + lane] = l;
            sc[2 * G + i * 32 + lane] = 1.0f / b[i];
            if (c * G + i * 32 + lane < u.keys && !gap) {
              const bool odd = !(fabsf(l) < 120.f);            // zero, infinite, NaN, next to them (1/b is not normal): the general way
              lo = fminf(lo, odd ? -INFINITY : l);
              hi = fmaxf(hi, odd ? INFINITY : l);
            }
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
          }
          if (lane == 0) {
            sc[3 * G] = lo;
            sc[3 * G + 1] = hi;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(BAR(B_SCF + slot));
        }
      }
    }
    __syncwarp();
  } else if (warp < 8) {
    reg_dealloc<kTileConvert>();
    // -------------------------------------------------------------------- V: int8 -> fp16
    // A warp takes 8 keys x 64 channels at a time: lane = 4 pieces of 16 channels x 2 keys x 4.  The two keys of 8 lanes are k and k ^ 5, which lie
    // in different banks in both tiles, the int8 one (pieces ^ key) and the fp16 one (pieces 2 pc ^ key).
    constexpr int BOXES = D / 64;
    const int key = ((lane >> 3) ^ ((lane >> 2 & 1) * 5)), pc = lane & 3, w0 = warp - 4;
    const uint32_t sV8 = smem_u32(smem + C::OFF_V8), sV = smem_u32(smem + C::OFF_V);
    const uint32_t at0 = key * 128 + (((2 * pc) ^ key) << 4), at1 = key * 128 + (((2 * pc + 1) ^ key) << 4);
    uint32_t it = 0;
    TileUnit u;
    bool ok = true;
    while (ok && next_unit(u)) {
      for (int c = u.c0; c < u.c1 && ok; ++c, ++it) {
        const uint32_t a = it % C::NV8, b = it % C::NV;
        ok = wait(B_V8F + a, (it / C::NV8) & 1u, TW_V8F) && wait(B_VE + b, ((it / C::NV) & 1u) ^ 1u, TW_VE);
        if (!ok) break;
        const uint32_t src = sV8 + a * C::K_BYTES, dst = sV + b * C::V_BYTES;
#pragma unroll 2
        for (int i = w0; i < G / 8 * BOXES; i += 4) {
          const int blk = i / BOXES, box = i % BOXES;
          const int row = blk * 8 + key;
          const uint32_t from = D == 64 ? row * 64 + ((pc ^ ((row >> 1) & 3)) << 4) : (box >> 1) * (G * 128) + row * 128 + ((((box & 1) * 4 + pc) ^ key) << 4);
          const uint4 x = lds16(src + from);
          const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
          uint32_t h[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t r = __byte_perm(w[k / 2], 0x64646464u, k & 1 ? 0x4342 : 0x4140);
            const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&r), __half2half2(__ushort_as_half(0x6480)));
            h[k] = *reinterpret_cast<const uint32_t*>(&y);
          }
          const uint32_t to = dst + box * (G * 128) + blk * 1024;
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + at0), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + at1), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(BAR(B_VF + b));
          mbar_arrive(BAR(B_V8E + a));
        }
      }
    }
    __syncwarp();
  } else {
    reg_alloc<kTileSoftmax>();
    // -------------------------------------------------------------------- softmax, one thread a row
    constexpr int NB = G / 16;                                 // blocks of 16 columns
    const int tile = (warp - 8) >> 2, rr = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;         // (lane 32 * (warp % 4) in bits 16 and up)
    const uint32_t tS0 = tmem + C::COL_S + tile * 2 * G + lanes, tO = tmem + C::COL_O + tile * D + lanes;
    const int tok = tile * p.tile_tokens + rr / p.ratio, hr = rr % p.ratio;
    uint32_t sit = 0, it = 0;                                  // chunks of this tile, of all so far
    // what a row needs of its unit; the scale of its query is asked for here and used a while later
    TileUnit u;
    float qs_raw = 0.f;
    bool mine = false;
    auto take = [&]() {
      if (!next_unit(u)) return false;
      mine = tok < u.tokens && rr < p.tile_tokens * p.ratio;
      qs_raw = 0.f;
      if (mine) qs_raw = p.qs[(long long)(u.t0 + tok) * p.qsn + (u.head * p.ratio + hr) * p.qsh];
      return true;
    };
    bool ok = true, have = take();
    while (have) {
      if (tile > 0 && u.tokens <= p.tile_tokens) {             // no rows in this tile
        for (int c = u.c0; c < u.c1 && ok; ++c, ++it) {
          ok = wait(B_SCF + it % C::NSC, (it / C::NSC) & 1u, TW_SC);
          if (lane == 0) mbar_arrive(BAR(B_SCE + it % C::NSC));
        }
        have = ok && take();
        continue;
      }
      const float qs = qs_raw * p.c;
      const uint64_t qs2 = f2_pack(qs, qs), magic2 = f2_pack(-kMagicF, -kMagicF);
      // the last key that the row sees; the least and the most of the warp
      int lim = u.keys - 1;
      if (p.causal && mine && u.lim0 + tok < lim) lim = u.lim0 + tok < -1 ? -1 : (int)(u.lim0 + tok);
      const int lim_least = __reduce_min_sync(0xffffffffu, lim), lim_most = __reduce_max_sync(0xffffffffu, lim);
      float mref = -INFINITY, ref = -INFINITY, l = 0.f;        // references of p and of w (of the accumulator)
      for (int c = u.c0; c < u.c1; ++c, ++it, ++sit) {
        const uint32_t slot = it % C::NSC;
        ok = mbar_wait2_warp(BAR(B_SCF + slot), (it / C::NSC) & 1u, code_hi | TW_SC, BAR(B_S + 2 * tile + (sit & 1u)), sit >> 1 & 1u, code_hi | TW_S, abort_flag,
                             p.status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tS = tS0 + (sit & 1u) * G;
        const float* sc = reinterpret_cast<const float*>(smem + C::OFF_SC) + slot * C::SC_FLOATS;
        const float lo = sc[3 * G], hi = sc[3 * G + 1];
        const int key0 = c * G, rel = lim - key0;              // (the last column that the row sees)
        const bool whole = lim_least - key0 >= G - 1;
        // exponents of w, x + log2 v_scale - off, of 16 columns, in place of the scores
        auto exponents = [&](int b, uint32_t* r, float off, bool mask) {
          const uint64_t off2 = f2_pack(-off, -off);
          const ulonglong2* ks = reinterpret_cast<const ulonglong2*>(sc + b * 16);
          const ulonglong2* lv = reinterpret_cast<const ulonglong2*>(sc + G + b * 16);
#pragma unroll
          for (int k = 0; k < 16; k += 4) {
            const ulonglong2 a = ks[k / 4], v = lv[k / 4];
            f2_unpacku(f2_fma(f2_add(f2_packu(r[k], r[k + 1]), magic2), f2_mul(a.x, qs2), f2_add(v.x, off2)), r[k], r[k + 1]);
            f2_unpacku(f2_fma(f2_add(f2_packu(r[k + 2], r[k + 3]), magic2), f2_mul(a.y, qs2), f2_add(v.y, off2)), r[k + 2], r[k + 3]);
          }
          if (mask) {
            const int last = rel - b * 16;
#pragma unroll
            for (int k = 0; k < 16; ++k) r[k] = k <= last ? r[k] : __float_as_uint(-INFINITY);
          }
        };
        // The references are taken over as they are, and P is made with them in one go.  The sum of p = w / v_scale bounds every w (w <= sum p
        // times the largest v_scale); where that does not say that all w are below 2^15, or a row has no reference yet, the reference is
        // looked for: in a unit's first chunk in 16 columns, then, if need be, in all.  (A row without one is looked at whatever its sum says: all V
        // scales so far were 0, and relative to nothing w may be too small for fp32.)
        uint64_t sum2, sum3;
        uint32_t pk[8 * NB];
        float total = 0.f;
        int find = c == u.c0 ? 1 : 0;                          // columns to look at: none, 16, all
        const float most = hi < 100.f ? ex2_approx(15.f - hi) : 0.f;
        for (;;) {
          if (find) {
            float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll 1
            for (int b = 0; b * 16 <= lim_most - key0 && b < (find == 1 ? 1 : NB); ++b) {
              uint32_t r[16];
              tmem_ld16(tS + b * 16, r);
              tmem_ld_wait16(r);
              exponents(b, r, 0.f, true);
#pragma unroll
              for (int k = 0; k < 16; k += 4) {
                mx0 = max3(mx0, __uint_as_float(r[k]), __uint_as_float(r[k + 1]));
                mx1 = max3(mx1, __uint_as_float(r[k + 2]), __uint_as_float(r[k + 3]));
              }
            }
            const float top = fmaxf(mx0, mx1);
            const float to = top > ref ? top : ref, f = ref == -INFINITY ? 0.f : ex2_approx(ref - to);
            // (the reference of p as far from the largest p as a middling V scale is from 1; it stays until `easy` does not hold)
            if (to > -INFINITY && mref == -INFINITY && hi - lo < 60.f) mref = to - 0.5f * (lo + hi);
            ref = to;
            if (c > u.c0) {                                    // (the first P V does not look at what is there)
              ok = wait(B_O + 2 * tile + ((sit - 1u) & 1u), (sit - 1u) >> 1 & 1u, TW_O);       // P V of the chunk before is done
              if (!ok) break;
              tc_fence_after();
              const uint64_t f2 = f2_pack(f, f);
#pragma unroll 1
              for (int b = 0; b < D / 16; ++b) {
                uint32_t o[16];
                tmem_ld16(tO + b * 16, o);
                tmem_ld_wait16(o);
#pragma unroll
                for (int k = 0; k < 16; k += 2) f2_unpacku(f2_mul(f2_packu(o[k], o[k + 1]), f2), o[k], o[k + 1]);
                tmem_st16(tO + b * 16, o);
              }
            }
          }
          const float base = safe(ref);
          sum2 = sum3 = 0;
          // (all columns of a chunk at once, in a straight line: there are two such warps a scheduler, and only what is independent within one
          // hides the latencies)
          auto make_p = [&](auto mask) {
            uint32_t r[G];
#pragma unroll
            for (int b = 0; b < G; b += 32) tmem_ld32(tS + b, *reinterpret_cast<uint32_t(*)[32]>(r + b));
#pragma unroll
            for (int b = 0; b < G; b += 32) tmem_ld_wait(*reinterpret_cast<uint32_t(*)[32]>(r + b));
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              exponents(b, r + b * 16, base, decltype(mask)::value);
              const ulonglong2* iv = reinterpret_cast<const ulonglong2*>(sc + 2 * G + b * 16);
#pragma unroll
              for (int k = 0; k < 16; k += 4) {
                const ulonglong2 v = iv[k / 4];
                const uint32_t* x = r + b * 16 + k;
                const float w0 = ex2_approx(__uint_as_float(x[0])), w1 = ex2_approx(__uint_as_float(x[1]));
                const float w2 = ex2_approx(__uint_as_float(x[2])), w3 = ex2_approx(__uint_as_float(x[3]));
                sum2 = f2_fma(f2_pack(w0, w1), v.x, sum2);
                sum3 = f2_fma(f2_pack(w2, w3), v.y, sum3);
                const __half2 y0 = __floats2half2_rn(w0, w1), y1 = __floats2half2_rn(w2, w3);
                pk[b * 8 + k / 2] = *reinterpret_cast<const uint32_t*>(&y0);
                pk[b * 8 + k / 2 + 1] = *reinterpret_cast<const uint32_t*>(&y1);
              }
            }
          };
          if (whole) make_p(Flag<false>());
          else make_p(Flag<true>());
          {
            float s0, s1, s2, s3;
            f2_unpack(sum2, s0, s1);
            f2_unpack(sum3, s2, s3);
            total = (s0 + s1) + (s2 + s3);
          }
          if (find == 2 || !__any_sync(0xffffffffu, !(total < most) || (ref == -INFINITY && rel >= 0 && hi > -INFINITY))) break;
          find = 2;
        }
        if (!ok) break;
        const float d = ref - mref;
        const bool easy = ref == -INFINITY ? mref == -INFINITY && lo > -INFINITY : lo >= d - 60.f && hi <= d + 60.f;
        if (__all_sync(0xffffffffu, easy)) {
          l = ref > -INFINITY ? fmaf(total, ex2_approx(d), l) : l + total;       // (without a reference: 0, or NaN where no score is a number)
        } else {
          // p by itself: the scores once more
          float top = -INFINITY;
#pragma unroll 1
          for (int pass = 0; pass < 2; ++pass) {
            float sum = 0.f;
            const float base = safe(mref);
#pragma unroll 1
            for (int b = 0; b < NB; ++b) {
              uint32_t o[16];
              tmem_ld16(tS + b * 16, o);
              tmem_ld_wait16(o);
              const float4* ks = reinterpret_cast<const float4*>(sc + b * 16);
#pragma unroll
              for (int k = 0; k < 16; k += 4) {
                const float4 a = ks[k / 4];
                const float aa[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float x = (__uint_as_float(o[k + e]) - kMagicF) * (aa[e] * qs);
                  const int at = b * 16 + k + e;
                  if (at > rel || (sc[2 * G + at] == 0.f && sc[G + at] == -INFINITY)) x = -INFINITY;
                  if (pass == 0) top = fmaxf(top, x);
                  else sum += ex2_approx(x - base);
                }
              }
            }
            if (pass == 0) {
              if (top > mref + 8.f || (mref == -INFINITY && top > -INFINITY)) {
                if (mref > -INFINITY) l *= ex2_approx(mref - top);         // (else 0, or NaN)
                mref = top;
              }
            } else {
              l += sum;
            }
          }
        }
        // P over the scores it was made of: 16 keys in the first 8 of their 16 columns
#pragma unroll
        for (int b = 0; b < NB; ++b) tmem_st8(tS + b * 16, reinterpret_cast<const uint32_t(&)[8]>(pk[b * 8]));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(BAR(B_P + 2 * tile + (sit & 1u)));
          mbar_arrive(BAR(B_SCE + slot));
        }
      }
      if (!ok) break;
      // ---- the unit's rows (and the scale of the row's next query on its way)
      const TileUnit done = u;
      const bool write = mine;
      have = take();
      ok = wait(B_O + 2 * tile + ((sit - 1u) & 1u), (sit - 1u) >> 1 & 1u, TW_O);
      if (!ok) break;
      tc_fence_after();
      const float f = done.slot < 0 ? row_factor(mref, ref, l) : 1.f;
      const int h = done.head * p.ratio + hr;
      const long long row = (long long)done.slot * p.rows_tile + tile * kTileRows + rr;
      const long long out_at = write ? (long long)(done.t0 + tok) * p.on + h * p.oh : -1;
      // 64 channels at a time: the warp's 32 rows through shared memory (16-byte pieces ^ row: no bank conflicts), then out as 128-byte lines;
      // a unit's part goes to scratch as it is.
      uint8_t* stage = smem + C::OFF_OUT + (warp - 8) * 4096 + lane * 128;
      const uint8_t* staged = smem + C::OFF_OUT + (warp - 8) * 4096 + (lane >> 3) * 128;
      float* part = p.part + row * D;
#pragma unroll 1
      for (int b = 0; b < D; b += 64) {
        uint32_t o[64];
        tmem_ld32(tO + b, reinterpret_cast<uint32_t(&)[32]>(o[0]));
        tmem_ld32(tO + b + 32, reinterpret_cast<uint32_t(&)[32]>(o[32]));
        tmem_ld_wait(reinterpret_cast<uint32_t(&)[32]>(o[0]));
        tmem_ld_wait(reinterpret_cast<uint32_t(&)[32]>(o[32]));
        if (done.slot >= 0) {
          if (write) {
#pragma unroll
            for (int k = 0; k < 64; k += 4) *reinterpret_cast<uint4*>(part + b + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          }
          __syncwarp();
          continue;
        }
        if (p.o_bf16) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(o[2 * i]) * f, __uint_as_float(o[2 * i + 1]) * f);
            o[i] = *reinterpret_cast<const uint32_t*>(&y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const __half2 y = __floats2half2_rn(__uint_as_float(o[2 * i]) * f, __uint_as_float(o[2 * i + 1]) * f);
            o[i] = *reinterpret_cast<const uint32_t*>(&y);
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          *reinterpret_cast<uint4*>(stage + ((k ^ (lane & 7)) << 4)) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        __syncwarp();
        uint4 y[8];
        long long to[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int from = 4 * i + (lane >> 3);
          y[i] = *reinterpret_cast<const uint4*>(staged + i * 512 + (((lane & 7) ^ (from & 7)) << 4));
          to[i] = __shfl_sync(0xffffffffu, out_at, from);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (to[i] >= 0) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o) + to[i] + b + (lane & 7) * 8) = y[i];
        __syncwarp();
      }
      if (write) {
        if (done.slot >= 0) *reinterpret_cast<float4*>(p.part_ml + row * 4) = make_float4(mref, ref, l, 0.f);
        else if (p.lse) p.lse[(long long)(done.t0 + tok) * p.H + h] = mref + log2f(l);
      }
      tc_fence_before();
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}
