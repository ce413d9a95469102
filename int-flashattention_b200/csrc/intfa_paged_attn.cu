// Attention of packed int8 query rows over a paged int8 K/V cache: decode, and the few rows of a draft or a chunk.
//
//   s = dot(q8, k8) * (q_scale * sm_scale * log2 e) * k_scale[block],   p = exp2(s - max),   o = sum p v_scale[block] v8 / sum p
//
// Reads K and V once (64 sequences of up to 8192 keys, 8 heads x 128: 703 MB, 109 us at the measured copy rate, 118 to 133 here): bound by HBM.  One
// sequence of 131 072 keys 41.6 and 57: ten microseconds are the start, the end and the combination.  Short calls are all that, 6.4 in clusters.
// 16 rows a K/V head at 64 channels (91 MB) 14.1 and 34.0: the latency of two warps a scheduler, whose exp2 are per row and key.
//
// Work.  A unit is (sequence, K/V head, tile of RT = 8 NT rows); the rows of all query heads that share the K/V head are packed into it, so
// that K and V are read once for all of them.  Its keys are cut into chunks of G = 32, 64 at head dim 64.  The chunks of all units in a row are
// dealt out to the warps of the GPU in equal contiguous shares, whatever the sequences' lengths are: the lengths are read on the device, so
// nothing waits for the host and a captured graph takes other lengths at its next replay.  A warp keeps the softmax state and the output of the unit it is in
// in registers.  A unit that lies within one warp's share is written at once; the parts of the others go to scratch and combine_kernel adds
// them up, in the order of the keys.  Few units of few keys: a unit is the work of a cluster of CTAs, whose parts are added up through their shared
// memory, with no second launch.
//
// Loads.  Each warp has a ring of NS chunks of its own, filled by TMA (pages of any size and order, 8 to G rows a copy) and by cp.async (scales,
// query rows), so no warp waits for another and NS - 1 chunks a warp (64 to 128 KB an SM) are in flight.  A chunk's rows are swizzled by the
// TMA such that the 16-byte reads below are free of bank conflicts.
//
// Arithmetic.  m16n8 warp-level MMAs straight from that ring: 8 or 16 rows are far below the smallest tcgen05 tile.  Q K^T is an int8
// product, exact in int32; the order of the k index is free, so lane t of a quad takes 16-byte piece 2t of each row and calls it its
// fragment.  For P V the int8 V becomes fp16 (exact: the byte is put behind fp16's 1024 and 1152 is taken off), two keys of a channel in a word.
// The V scale of a key multiplies its p ahead of the rounding to fp16.  Since the scales of a cache may differ by any factor, the products
// w = p * v_scale have a running maximum of their own (of s + log2 v_scale), so the largest w is 1 whatever the scales are and the rounding
// (2^-11 of each w, or 2^-25 of the largest) costs no more than with equal scales; sums and both maxima are fp32.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "intfa_internal.h"
#include "intfa_ptx.cuh"
#include "intfa_rows.cuh"

namespace intfa {
namespace {

constexpr float kMagicF = 12582912.0f;            // 1.5*2^23: added to an int32 below 2^22 as a bit pattern, it reads as fp32 1.5*2^23 + value
constexpr int kMagicI = 0x4B400000;

// A unit as combine_kernel sees it (one load tells it all): where the parts are and which query rows it has.
struct __align__(16) UnitPart {
  int open;                                       // 1: its parts are in scratch
  int first;                                      // warp that began it
  int n0, n1, n2;                                 // parts of single warps first, first+1 ..; of whole CTAs; of single warps again
  int cta;                                        // the first of those CTAs
  int token, tokens;                              // its first token among all, its tokens
  int row, head;                                  // row of that token that it begins with; K/V head
  int pad[2];
};
static_assert(sizeof(UnitPart) == 48, "unit");
// the parts of chunks chunk0 .. chunk1-1 in shares of `share`: CTAs that lie in the unit as a whole leave one part each, in their first warp's slot
__device__ inline void set_parts(UnitPart& u, long long chunk0, long long chunk1, long long share, long long total, int cta_warps) {
  const long long cs = share * cta_warps, a = chunk0 / share, b = (chunk1 - 1) / share;
  const long long ka = (chunk0 + cs - 1) / cs, kb = chunk1 == total ? (total - 1) / cs : chunk1 / cs - 1;
  u.first = (int)a;
  u.cta = (int)ka;
  u.n0 = (int)(ka <= kb ? ka * cta_warps - a : b - a + 1);
  u.n1 = (int)(ka <= kb ? kb - ka + 1 : 0);
  u.n2 = (int)(ka <= kb && b >= (kb + 1) * cta_warps ? b - (kb + 1) * cta_warps + 1 : 0);
}

struct PParams {
  const int8_t* q; const float* qs; void* o; float* lse;
  long long qn, qh, qsn, qsh, on, oh;
  const float* ks; const float* vs;
  long long ksP, ksH, ksB, vsP, vsH, vsB;
  const int* table; long long table_stride; int width;
  const int* lens; const int* cu;
  int S, H, Hkv, ratio, pages, page_log, block_log, box_log, chunk_log;
  long long T;
  int causal, o_bf16;
  float c;                                        // sm_scale * log2(e)
  int workers, least;                             // warps of the grid; fewest chunks a warp takes
  int rows_tile;                                  // rows of a unit: RT, or those of one or two 128-row tiles
  int tile_tokens, unit_tokens;                   // 128-row tiles: whole tokens in one, in a unit; 0: packed RT rows
  float* part; float* part_ml;                    // [2*workers][RT][D]; [2*workers][RT]{m, mw, l, -}
  UnitPart* units; long long max_units;           // [max_units]
  int* head;                                      // {units}; packed rows only
  int* status;
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t lds_u64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float lds_f(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// what a sequence asks for
struct Seq {
  int t0, n;                 // its query rows: tokens t0 .. t0 + n - 1
  int keys;                  // that are looked at
  long long len;
  int tiles, chunks;         // row tiles and chunks of each K/V head
  bool bad;                  // its rows or its tokens are not where they can be
};
__device__ __forceinline__ Seq seq_of(const PParams& p, int s) {
  Seq q;
  const long long t0 = p.cu ? p.cu[s] : s, t1 = p.cu ? p.cu[s + 1] : s + 1;
  q.t0 = (int)t0;
  q.n = t0 >= 0 && t1 > t0 && t1 <= p.T ? (int)(t1 - t0) : 0;
  q.len = p.lens[s];
  const long long most = (long long)p.width << p.page_log;
  q.keys = (int)(q.len < 0 ? 0 : q.len < most ? q.len : most);
  q.bad = t0 < 0 || t1 < t0 || t1 > p.T || (q.n > 0 && q.len != q.keys);
  q.tiles = (int)(((long long)q.n * p.ratio + p.rows_tile - 1) / p.rows_tile);
  q.chunks = q.keys > 0 ? ((q.keys - 1) >> p.chunk_log) + 1 : 1;        // (a row without keys is written, too)
  return q;
}

// a place in the row of all chunks
struct Cursor {
  Seq q;
  int s, head, tile, chunk;  // sequence; unit in it: K/V head and tile; chunk in that
  __device__ __forceinline__ void next(const PParams& p) {
    if (++chunk < q.chunks) return;
    chunk = 0;
    if (++tile < q.tiles) return;
    tile = 0;
    if (++head < p.Hkv) return;
    head = 0;
    next_seq(p);
  }
  // to the next sequence with query rows, if there is one
  __device__ __forceinline__ void next_seq(const PParams& p) {
    q.n = 0;
    while (++s < p.S) {
      q = seq_of(p, s);
      if (q.n > 0) break;
    }
  }
};

// G: keys of a chunk
template <int D, int NT, int WARPS, int NS, int G>
struct DecodeCfg {
  static constexpr int RT = 8 * NT, KV = G * D;                         // rows of a tile; bytes of K or V of a chunk
  static constexpr int PANEL = D < 128 ? D : 128, PANELS = D / PANEL;   // a row lies in panels of at most 128 bytes
  static constexpr int EXTRA = 2 * G * 4 + RT * D + RT * 4;             // scales, query rows and their scales
  static constexpr int OFF_EXTRA = WARPS * NS * 2 * KV;
  static constexpr int OFF_BAR = OFF_EXTRA + WARPS * NS * EXTRA;
  static constexpr int OFF_PRE = OFF_BAR + WARPS * NS * 8;              // [threads + 1] chunks (long long) and units (int) before a thread's sequences
  static constexpr int OFF_MISC = OFF_PRE + ((32 * WARPS + 1) * 12 + 15) / 16 * 16;
  static constexpr int OFF_SUMS = OFF_EXTRA;                            // [warps] chunks and units (long long) of a warp's sequences, ahead of the first load
  static_assert(OFF_SUMS >= WARPS * NS * 2 * KV, "the sums lie outside the ring: the async proxy's copies into it know nothing of plain stores");
  static constexpr int SMEM = OFF_MISC + 32 + 1024;
  static constexpr int MERGE = (WARPS + 1) * RT * ((D + 4) + 4) * 4;    // (over the ring, when it is done with)
  static_assert(MERGE <= OFF_EXTRA, "merge");
  static_assert(EXTRA % 16 == 0, "alignment");
  static_assert(WARPS * 16 <= WARPS * NS * EXTRA, "sums");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// state of the rows of a unit in one warp: rows n*8 + lane/4 (maxima, l: of this lane's keys only until reduced), channels as `acc`
template <int D, int NT>
struct RowState {
  static constexpr int PANELS = D < 128 ? 1 : D / 128, W = D < 128 ? D / 32 : 4, MT = PANELS * W * 2;
  float m[NT], mw[NT], l[NT];
  float acc[NT][MT][4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = mw[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
    }
  }
  __device__ __forceinline__ void reduce_l() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
    }
  }
};
// channel of entry (i, 0/1) of a lane; entries 2, 3: the next channel
template <int D>
__device__ __forceinline__ int channel_of(int i, int g) {
  constexpr int W = D < 128 ? D / 32 : 4;
  return i / (2 * W) * 128 + g * (4 * W) + i % (2 * W) * 2;
}

__device__ __forceinline__ float safe(float m) { return m == -INFINITY ? 0.f : m; }

// what the sum of a row is multiplied by: 2^(mw - m) / l.  A row that sees nothing has l = 0, one whose values are all zero mw = -inf.
// (The power in two halves: V scales below 2^-126 leave one that exp2 would flush to zero.)
__device__ __forceinline__ float row_factor(float m, float mw, float l) {
  const float half = ex2_approx(0.5f * (mw - safe(m)));
  return l == 0.f ? 0.f : mw == -INFINITY ? l * 0.f : half / l * half;
}

template <int D, int NT>
__device__ __forceinline__ void write_rows(const PParams& p, const Seq& q, int head, int tile, const RowState<D, NT>& st) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  constexpr int MT = RowState<D, NT>::MT, W = RowState<D, NT>::W, PANELS = RowState<D, NT>::PANELS;
  const int R = q.n * p.ratio;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float f = row_factor(st.m[n], st.mw[n], st.l[n]);
    const int rg = tile * (8 * NT) + n * 8 + g;
    if (p.lse && t == 0 && rg < R) p.lse[(q.t0 + rg / p.ratio) * (long long)p.H + head * p.ratio + rg % p.ratio] = st.m[n] + log2f(st.l[n]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float fe = __shfl_sync(0xffffffffu, f, (2 * t + e) * 4);
      const int r = tile * (8 * NT) + n * 8 + 2 * t + e;
      if (r >= R) continue;
      uint16_t* o = static_cast<uint16_t*>(p.o) + (q.t0 + r / p.ratio) * p.on + (head * p.ratio + r % p.ratio) * p.oh;
#pragma unroll
      for (int pn = 0; pn < PANELS; ++pn) {
        uint32_t w[2 * W];
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
          const float a = st.acc[n][pn * 2 * W + i][e] * fe, b = st.acc[n][pn * 2 * W + i][2 + e] * fe;
          if (p.o_bf16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
          } else {
            const __half2 h = __floats2half2_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        uint4* d = reinterpret_cast<uint4*>(o + channel_of<D>(pn * 2 * W, g));
#pragma unroll
        for (int i = 0; i < 2 * W; i += 4) d[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      }
    }
  }
  static_assert(MT == PANELS * 2 * W, "tiles");
}

// 4 channels of a row, added up part by part
struct Sum {
  float m, mw, l;
  float4 a;
  __device__ __forceinline__ void clear() {
    m = mw = -INFINITY;
    l = 0.f;
    a = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void add(const float4& ml, const float4& x) {
    const float m1 = fmaxf(m, ml.x), w1 = fmaxf(mw, ml.y);
    l = l * ex2_approx(m - safe(m1)) + ml.z * ex2_approx(ml.x - safe(m1));
    const float f = ex2_approx(mw - safe(w1)), h = ex2_approx(ml.y - safe(w1));
    a.x = a.x * f + x.x * h; a.y = a.y * f + x.y * h; a.z = a.z * f + x.z * h; a.w = a.w * f + x.w * h;
    m = m1;
    mw = w1;
  }
};
// ... and written: query row n, head h
__device__ __forceinline__ void write_sum(const PParams& p, long long n, int h, int ch, const Sum& x) {
  const float f = row_factor(x.m, x.mw, x.l);
  uint2 w;
  if (p.o_bf16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.a.x * f, x.a.y * f), b = __floats2bfloat162_rn(x.a.z * f, x.a.w * f);
    w.x = *reinterpret_cast<const uint32_t*>(&a);
    w.y = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    const __half2 a = __floats2half2_rn(x.a.x * f, x.a.y * f), b = __floats2half2_rn(x.a.z * f, x.a.w * f);
    w.x = *reinterpret_cast<const uint32_t*>(&a);
    w.y = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.o) + n * p.on + h * p.oh + ch) = w;
  if (p.lse && ch == 0) p.lse[n * p.H + h] = x.m + log2f(x.l);
}

template <int D, int NT>
__device__ __forceinline__ void write_part(float* part, float* ml, int stride, const RowState<D, NT>& st) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  constexpr int MT = RowState<D, NT>::MT;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (t == 0) *reinterpret_cast<float4*>(ml + (n * 8 + g) * 4) = make_float4(st.m[n], st.mw[n], st.l[n], 0.f);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* d = part + (n * 8 + 2 * t + e) * stride;
#pragma unroll
      for (int i = 0; i < MT; i += 2)
        *reinterpret_cast<float4*>(d + channel_of<D>(i, g)) = make_float4(st.acc[n][i][e], st.acc[n][i][2 + e], st.acc[n][i + 1][e], st.acc[n][i + 1][2 + e]);
    }
  }
}

constexpr float kNoKey = -INFINITY;               // in place of the K scale: no key, its page lies outside the cache (the V scale is 0)
__device__ const float no_key = kNoKey;

// One chunk.  sK, sV: its rows in shared memory; sS: its K scales, then the logarithms of its V scales; last[n]: the last key of the chunk that row n*8 + g sees.
// MASKED: not all rows see all keys, or the K scales say kNoKey.
template <int D, int NT, int G, bool MASKED>
__device__ __forceinline__ void chunk_step(RowState<D, NT>& st, const uint32_t (&q)[D / 64][NT][4], const float (&qs)[NT], const int (&last)[NT],
                                           uint32_t sK, uint32_t sV, uint32_t sS) {
  const int magic[4] = {kMagicI, kMagicI, kMagicI, kMagicI};
  const uint64_t less = f2_pack(-kMagicF, -kMagicF);
  constexpr int CH = D / 64, AT = (NT + 1) / 2, W = RowState<D, NT>::W, PANELS = RowState<D, NT>::PANELS, PANEL = D < 128 ? D : 128;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  constexpr int KT = G / 8;
  uint64_t x[NT][KT], lv[KT];                     // keys 2t, 2t + 1 of each tile of 8
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    int d[AT][4];
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      // row kt*8 + g; piece 2t + (ch & 1) of a 128-byte panel, or t of a 64-byte one
      const int row = kt * 8 + g;
      uint32_t a;
      if constexpr (PANEL == 128) a = sK + (ch / 2) * (G * 128) + row * 128 + (((2 * t + (ch & 1)) ^ g) << 4);
      else a = sK + row * 64 + ((t ^ ((g >> 1) & 3)) << 4);
      const uint4 kw = lds16(a);
#pragma unroll
      for (int i = 0; i < AT; ++i) {
        const bool two = 2 * i + 1 < NT;
        const uint32_t(&lo)[4] = q[ch][2 * i];
        const uint32_t(&hi)[4] = q[ch][two ? 2 * i + 1 : 2 * i];
        if (ch == 0) mma_s8(d[i], lo[0], two ? hi[0] : 0u, lo[1], two ? hi[1] : 0u, kw.x, kw.y, magic);
        else mma_s8(d[i], lo[0], two ? hi[0] : 0u, lo[1], two ? hi[1] : 0u, kw.x, kw.y, d[i]);
        mma_s8(d[i], lo[2], two ? hi[2] : 0u, lo[3], two ? hi[3] : 0u, kw.z, kw.w, d[i]);
      }
    }
    const uint64_t ks = lds_u64(sS + (kt * 8 + 2 * t) * 4);
    lv[kt] = lds_u64(sS + (G + kt * 8 + 2 * t) * 4);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      x[n][kt] = f2_mul(f2_add(f2_packu(d[n / 2][(n & 1) * 2], d[n / 2][(n & 1) * 2 + 1]), less), f2_mul(ks, f2_pack(qs[n], qs[n])));
      if (MASKED) {
        float x0, x1, k0, k1;
        f2_unpack(x[n][kt], x0, x1);
        f2_unpack(ks, k0, k1);
        x[n][kt] = f2_pack(k0 == kNoKey ? -INFINITY : x0, k1 == kNoKey ? -INFINITY : x1);
      }
    }
  }
  uint32_t b[NT][KT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    uint64_t w[KT];
    float mx = -INFINITY, mw = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      w[kt] = f2_add(x[n][kt], lv[kt]);
      float x0, x1, w0, w1;
      f2_unpack(x[n][kt], x0, x1);
      f2_unpack(w[kt], w0, w1);
      // (chosen, not added: what lies in a place that is not looked at may be anything)
      if (MASKED) {
        if (kt * 8 + 2 * t > last[n]) x0 = w0 = -INFINITY;
        if (kt * 8 + 2 * t + 1 > last[n]) x1 = w1 = -INFINITY;
        x[n][kt] = f2_pack(x0, x1);
        w[kt] = f2_pack(w0, w1);
      }
      mx = max3(mx, x0, x1);
      mw = max3(mw, w0, w1);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, o));
    }
    mx = fmaxf(mx, st.m[n]);
    mw = fmaxf(mw, st.mw[n]);
    const float ms = safe(mx), mws = safe(mw);
    st.l[n] *= ex2_approx(st.m[n] - ms);
    const bool moved = mw != st.mw[n];
    const float f = ex2_approx(st.mw[n] - mws);
    st.m[n] = mx;
    st.mw[n] = mw;
    uint64_t sum = 0;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      float x0, x1, w0, w1;
      f2_unpack(f2_add(x[n][kt], f2_pack(-ms, -ms)), x0, x1);
      f2_unpack(f2_add(w[kt], f2_pack(-mws, -mws)), w0, w1);
      sum = f2_add(sum, f2_pack(ex2_approx(x0), ex2_approx(x1)));
      const __half2 h = __floats2half2_rn(ex2_approx(w0), ex2_approx(w1));
      b[n][kt] = *reinterpret_cast<const uint32_t*>(&h);
    }
    float s0, s1;
    f2_unpack(sum, s0, s1);
    st.l[n] += s0 + s1;
    if (__any_sync(0xffffffffu, moved)) {
      const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
      for (int i = 0; i < RowState<D, NT>::MT; ++i) {
        st.acc[n][i][0] *= f0;
        st.acc[n][i][1] *= f1;
        st.acc[n][i][2] *= f0;
        st.acc[n][i][3] *= f1;
      }
    }
  }
  // O^T (channels x rows) += V^T P^T, 16 keys at a time: two 8-key tiles, of which the lane holds keys 2t and 2t + 1
#pragma unroll
  for (int h = 0; h < G / 16; ++h) {
#pragma unroll
    for (int pn = 0; pn < PANELS; ++pn) {
      uint32_t v[4][W];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = h * 16 + (i >> 1) * 8 + 2 * t + (i & 1);
        if constexpr (W == 4) {
          const uint4 y = lds16(sV + pn * (G * 128) + row * 128 + ((g ^ (row & 7)) << 4));
          v[i][0] = y.x; v[i][1] = y.y; v[i][2] = y.z; v[i][3] = y.w;
        } else {
          const uint2 y = lds8(sV + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8);
          v[i][0] = y.x; v[i][1] = y.y;
        }
      }
#pragma unroll
      for (int j = 0; j < W; ++j) {
        uint32_t a[4][2];                        // [channel of four][8-key tile]
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t lo = __byte_perm(v[2 * k][j], v[2 * k + 1][j], 0x5140) ^ 0x80808080u;
          const uint32_t hi = __byte_perm(v[2 * k][j], v[2 * k + 1][j], 0x7362) ^ 0x80808080u;
          const uint32_t r[4] = {__byte_perm(lo, 0x64646464u, 0x4140), __byte_perm(lo, 0x64646464u, 0x4342),
                                 __byte_perm(hi, 0x64646464u, 0x4140), __byte_perm(hi, 0x64646464u, 0x4342)};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&r[i]), __half2half2(__ushort_as_half(0x6480)));
            a[i][k] = *reinterpret_cast<const uint32_t*>(&y);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16(st.acc[n][(pn * W + j) * 2], a[0][0], a[1][0], a[0][1], a[1][1], b[n][2 * h], b[n][2 * h + 1]);
          mma_f16(st.acc[n][(pn * W + j) * 2 + 1], a[2][0], a[3][0], a[2][1], a[3][1], b[n][2 * h], b[n][2 * h + 1]);
        }
      }
    }
  }
}

enum { kWaitChunk = 64 };

// CL: a unit is the work of a cluster of CTAs, whose warps share its chunks; the parts are added up through their shared memory
template <int D, int NT, int WARPS, int NS, int G, bool CL>
__global__ void __launch_bounds__(32 * WARPS, 1) paged_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PParams p) {
  using C = DecodeCfg<D, NT, WARPS, NS, G>;
  constexpr int RT = C::RT, THREADS = 32 * WARPS, M = G / 32;            // keys a lane
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t bar0 = smem_u32(smem + C::OFF_BAR) + warp * NS * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC);
  long long* pre_c = reinterpret_cast<long long*>(smem + C::OFF_PRE);
  int* pre_u = reinterpret_cast<int*>(pre_c + THREADS + 1);
  int* whole = reinterpret_cast<int*>(smem + C::OFF_MISC + 8);           // of the unit that all warps' shares lie in
  if (lane == 0)
    for (int i = 0; i < NS; ++i) mbar_init(bar0 + 8 * i, 1);
  if (threadIdx.x == 0) {
    abort_flag[0] = 0;
    abort_flag[1] = (int)(1u << 31);              // (2^31 cycles, about a second)
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  mbar_init_fence();
  pdl_wait();
  pdl_launch();
  Cursor at;
  long long total, share, begin, unit_id = 0;                // chunks, of a warp, before this warp; the unit among all
  if constexpr (CL) {
    const int size = (int)cluster_size(), rank = (int)cluster_rank(), unit = blockIdx.x / size, per_seq = (gridDim.x / size) / p.S;
    at.s = unit / per_seq;
    at.q = seq_of(p, at.s);
    at.head = (unit - at.s * per_seq) / at.q.tiles;
    at.tile = (unit - at.s * per_seq) - at.head * at.q.tiles;
    if (at.q.bad && p.status && threadIdx.x == 0 && rank == 0) atomicCAS(p.status, 0, kStatusBadIndex);
    total = at.q.chunks;
    share = (total + size * WARPS - 1) / (size * WARPS);
    begin = (warp * size + rank) * share;                    // (few chunks: on as many SMs as there are)
    at.chunk = (int)begin;
    __syncthreads();
  } else {
    // ---- the row of all chunks: thread i counts the sequences i*seg .. (i+1)*seg - 1
    const int seg = (p.S + THREADS - 1) / THREADS;
    {
      long long c = 0, u = 0;
      bool bad = false;
      for (int s = threadIdx.x * seg; s < (threadIdx.x + 1) * seg && s < p.S; ++s) {
        const Seq q = seq_of(p, s);
        const long long units = (long long)q.tiles * p.Hkv;
        c += units * q.chunks;
        u += units;
        bad |= q.bad;
      }
      if (bad && p.status && blockIdx.x == 0) atomicCAS(p.status, 0, kStatusBadIndex);
      // sums up to and with each thread: within the warps, then on top of the warps before
      const long long most = p.max_units;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, c, o), y = __shfl_up_sync(0xffffffffu, u, o);
        if (lane >= o) {
          c += x;
          u += y;
        }
      }
      long long* sums = reinterpret_cast<long long*>(smem + C::OFF_SUMS);
      if (lane == 31) {
        sums[2 * warp] = c;
        sums[2 * warp + 1] = u;
      }
      __syncthreads();
      for (int w = 0; w < warp; ++w) {
        c += sums[2 * w];
        u += sums[2 * w + 1];
      }
      pre_c[threadIdx.x + 1] = c;
      pre_u[threadIdx.x + 1] = (int)(u < most ? u : most);       // (more of them only where cu_seqlens overlap)
      if (threadIdx.x == 0) {
        pre_c[0] = 0;
        pre_u[0] = 0;
      }
    }
    __syncthreads();
    total = pre_c[THREADS];
    share = (total + p.workers - 1) / p.workers;
    if (share < p.least) share = p.least;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      p.head[0] = pre_u[THREADS];
    }
    begin = (long long)(blockIdx.x * WARPS + warp) * share;
    if (begin < total) {
      const int i = find_last(THREADS, begin, [&](int j) { return pre_c[j]; });
      long long off = begin - pre_c[i];
      unit_id = pre_u[i];
      at.s = i * seg - 1;
      do {
        at.next_seq(p);
        const long long units = (long long)at.q.tiles * p.Hkv, c = units * at.q.chunks;
        if (off < c) break;
        off -= c;
        unit_id += units;
      } while (at.s < p.S);
      const int unit = (int)(off / at.q.chunks);
      at.chunk = (int)(off - (long long)unit * at.q.chunks);
      at.head = unit / at.q.tiles;
      at.tile = unit - at.head * at.q.tiles;
      unit_id += unit;
    }
  }
  const int worker = blockIdx.x * WARPS + warp;
  const long long left0 = total - begin < share ? total - begin : share;
  long long left = left0 < 0 ? 0 : left0;                    // chunks to do
  auto advance = [&](Cursor& c) {
    if constexpr (CL) ++c.chunk;
    else c.next(p);
  };
  // ---- loads
  const uint32_t sKV = smem_u32(smem) + warp * NS * 2 * C::KV;
  const uint32_t sX = smem_u32(smem + C::OFF_EXTRA) + warp * NS * C::EXTRA;
  Cursor ahead = at;
  long long to_load = left;
  bool fresh = true;                                         // the next chunk to load needs its query rows, too
  int page[M];                                               // of keys `lane`, `lane` + 32 .. of the next chunk to load
  auto look_up = [&]() {
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int key = ahead.chunk * G + i * 32 + lane;
      page[i] = 0;
      if (to_load > 0 && key < ahead.q.keys) page[i] = p.table[ahead.s * p.table_stride + (key >> p.page_log)];
    }
  };
  const int rows_box = 1 << p.box_log, boxes = G >> p.box_log;
  auto load = [&](int stage) {
    if (to_load > 0) {
      const int key0 = ahead.chunk * G, head = ahead.head, tile = ahead.tile;
      // the rows of a copy lie in one page; lane j issues copy j
      int first_page = 0;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        if (page[i] < 0 || page[i] >= p.pages) {
          if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
          page[i] = p.pages;                                 // (one past the last: the copies are zeros)
        }
        const int pg = __shfl_sync(0xffffffffu, page[i], (lane << p.box_log) & 31);
        if (M == 1 || (lane << p.box_log) >> 5 == i) first_page = pg;
      }
      const uint32_t bar = bar0 + 8 * stage, dst = sKV + stage * 2 * C::KV, x = sX + stage * C::EXTRA;
      const int full = min(boxes, (ahead.q.keys - key0 + rows_box - 1) >> p.box_log);
      if (lane == 0) mbar_expect_tx(bar, full > 0 ? full * rows_box * 2 * D : 0);
      __syncwarp();
      if (lane < full) {
        const int slot = (key0 + (lane << p.box_log)) & ((1 << p.page_log) - 1);
#pragma unroll
        for (int pn = 0; pn < C::PANELS; ++pn) {
          const uint32_t d = dst + pn * (G * C::PANEL) + (lane << p.box_log) * C::PANEL;
          tma_load_4d(d, &tmK, bar, pn * C::PANEL, slot, head, first_page);
          tma_load_4d(d + C::KV, &tmV, bar, pn * C::PANEL, slot, head, first_page);
        }
      }
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const int key = key0 + i * 32 + lane;
        const bool gap = page[i] == p.pages, in = key < ahead.q.keys && !gap;
        const long long blk = (key & ((1 << p.page_log) - 1)) >> p.block_log;
        const float* ks = p.ks + (in ? page[i] * p.ksP + head * p.ksH + blk * p.ksB : 0);
        cp_async4(x + (i * 32 + lane) * 4, gap ? &no_key : ks, in || gap);
        cp_async4(x + (G + i * 32 + lane) * 4, p.vs + (in ? page[i] * p.vsP + head * p.vsH + blk * p.vsB : 0), in);
      }
      if (fresh) {
        const uint32_t xq = x + 2 * G * 4;
        const int R = ahead.q.n * p.ratio;
#pragma unroll
        for (int i = lane; i < RT * (D / 16); i += 32) {
          const int r = tile * RT + i / (D / 16);
          const bool ok = r < R;
          const int n = ok ? r / p.ratio : 0, h = head * p.ratio + (ok ? r - n * p.ratio : 0);
          cp_async16(xq + i * 16, p.q + (ahead.q.t0 + n) * p.qn + h * p.qh + i % (D / 16) * 16, ok);
        }
        if (lane < RT) {
          const int r = tile * RT + lane;
          const bool ok = r < R;
          const int n = ok ? r / p.ratio : 0, h = head * p.ratio + (ok ? r - n * p.ratio : 0);
          cp_async4(xq + RT * D + lane * 4, p.qs + (ahead.q.t0 + n) * p.qsn + h * p.qsh, ok);
        }
      }
      --to_load;
      advance(ahead);
      fresh = ahead.chunk == 0;
      look_up();
    }
    cp_async_commit();
  };
  look_up();
#pragma unroll 1
  for (int i = 0; i < NS; ++i) load(i);

  // Where the shares of all warps of the CTA lie in one unit, their parts are added up here before they go to scratch.
  const long long cta0 = (long long)blockIdx.x * WARPS * share, cta1 = cta0 + WARPS * share < total ? cta0 + WARPS * share : total;
  bool merge = false;
  RowState<D, NT> st;
  st.clear();
  uint32_t q[D / 64][NT][4];
  float qs[NT];
  int last[NT], full_keys = 0;
  int stage = 0, parity = 0;
  bool open = false, ok = true;
  long long unit0 = 0, unit1 = 0;                            // the unit's chunks among all
  long long pos = begin;
#pragma unroll 1
  while (left > 0) {
    cp_async_wait<NS - 1>();
    __syncwarp();
    ok = mbar_wait_warp(bar0 + 8 * stage, parity, abort_flag, p.status, (int)(blockIdx.x << 8) | kWaitChunk);
    if (!ok) break;
    const uint32_t kv = sKV + stage * 2 * C::KV, x = sX + stage * C::EXTRA;
    // the logarithms of the V scales, once for all rows
    bool zero = false;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const uint32_t at_v = x + (G + i * 32 + lane) * 4;
      const float v = lds_f(at_v);
      zero |= v == 0.f;
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(at_v), "f"(log2_approx(v)) : "memory");
    }
    zero = __any_sync(0xffffffffu, zero);                    // (among them may be keys that are not there)
    __syncwarp();
    if (!open) {
      open = true;
      unit0 = pos - at.chunk;
      unit1 = unit0 + at.q.chunks;
      st.clear();
      const int tile = at.tile, R = at.q.n * p.ratio;
      const uint32_t xq = x + 2 * G * 4;
      full_keys = at.q.keys;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int ch = 0; ch < D / 64; ++ch) {
          // (the pieces of K's rows that chunk_step() takes)
          const int piece = C::PANEL == 128 ? (ch / 2) * 8 + 2 * t + (ch & 1) : t;
          const uint4 w = lds16(xq + (n * 8 + g) * D + piece * 16);
          q[ch][n][0] = w.x; q[ch][n][1] = w.y; q[ch][n][2] = w.z; q[ch][n][3] = w.w;
        }
        qs[n] = lds_f(xq + RT * D + (n * 8 + g) * 4) * p.c;
        const int r = tile * RT + n * 8 + g;
        last[n] = at.q.keys - 1;
        if (p.causal && r < R) {
          const long long lim = at.q.len - at.q.n + r / p.ratio;
          if (lim < last[n]) last[n] = lim < 0 ? -1 : (int)lim;
        }
        full_keys = min(full_keys, last[n] + 1);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) full_keys = min(full_keys, __shfl_xor_sync(0xffffffffu, full_keys, o));
    }
    const int key0 = at.chunk * G;
    if (key0 + G <= full_keys && !zero) {
      chunk_step<D, NT, G, false>(st, q, qs, last, kv, kv + C::KV, x);
    } else {
      int rel[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) rel[n] = last[n] - key0;
      chunk_step<D, NT, G, true>(st, q, qs, rel, kv, kv + C::KV, x);
    }
    __syncwarp();
    load(stage);
    if (++stage == NS) {
      stage = 0;
      parity ^= 1;
    }
    --left;
    ++pos;
    if constexpr (CL) {
      if (left == 0) st.reduce_l();
    } else if (at.chunk + 1 == at.q.chunks || left == 0) {
      st.reduce_l();
      const int head = at.head, tile = at.tile;
      const bool starts = unit0 >= begin, ends = unit1 <= pos;
      if (unit_id >= p.max_units) {
        if (p.status && lane == 0) atomicCAS(p.status, 0, kStatusBadIndex);            // (cu_seqlens that overlap)
      } else if (starts && lane == 0) {
        UnitPart u;
        u.open = !(ends || (cta0 == unit0 && cta1 == unit1));
        if (u.open) set_parts(u, unit0, unit1, share, total, WARPS);
        u.token = at.q.t0 + tile * RT / p.ratio;
        u.tokens = at.q.t0 + at.q.n - u.token;
        u.row = tile * RT % p.ratio;
        u.head = head;
        p.units[unit_id] = u;
      }
      if (starts && ends) {
        write_rows(p, at.q, head, tile, st);
      } else if (cta0 >= unit0 && cta1 <= unit1) {
        merge = true;
        if (lane == 0) {
          whole[0] = cta0 == unit0 && cta1 == unit1;
          whole[1] = cta0 == unit0;
          whole[2] = at.q.t0;
          whole[3] = at.q.n * p.ratio - tile * RT;
          whole[4] = head;
          whole[5] = tile;
        }
      } else {
        const long long slot = 2LL * worker + (starts ? 1 : 0);
        write_part<D, NT>(p.part + slot * RT * D, p.part_ml + slot * RT * 4, D, st);
      }
      open = false;
      ++unit_id;
    }
    advance(at);
  }
  if (!ok) {
    // A wait ran out.  The units that this share begins and that were not reached are no parts for combine_kernel; what this warp asked for comes
    // before it goes, or does not come at all.
    for (long long i = left - to_load; i > 0; --i) {
      mbar_drain(bar0 + 8 * stage, parity);
      if (++stage == NS) {
        stage = 0;
        parity ^= 1;
      }
    }
    for (bool begins = open ? unit0 >= begin : at.chunk == 0; !CL && left > 0; --left) {
      if (begins && lane == 0 && unit_id < p.max_units) p.units[unit_id].open = 0;
      if (at.chunk + 1 == at.q.chunks) ++unit_id;
      at.next(p);
      begins = at.chunk == 0;
    }
  }
  if (!__syncthreads_or(merge || CL)) return;
  // (every warp is done with its ring: what it asked for has come)
  float* red = reinterpret_cast<float*>(smem);
  float* red_ml = red + WARPS * RT * (D + 4);
  write_part<D, NT>(red + warp * RT * (D + 4), red_ml + warp * RT * 4, D + 4, st);
  __syncthreads();
  float* mine = red_ml + WARPS * RT * 4;                     // (CL) the CTA's sums, then their m, mw, l
  float* mine_ml = mine + RT * (D + 4);
  const long long slot = CL ? 0 : 2LL * blockIdx.x * WARPS + whole[1];
  for (int i = threadIdx.x; i < RT * (D / 4); i += THREADS) {
    const int r = i / (D / 4), ch = i % (D / 4) * 4;
    Sum x;
    x.clear();
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
      x.add(*reinterpret_cast<const float4*>(red_ml + (w * RT + r) * 4), *reinterpret_cast<const float4*>(red + (w * RT + r) * (D + 4) + ch));
    if constexpr (CL) {
      *reinterpret_cast<float4*>(mine + r * (D + 4) + ch) = x.a;
      if (ch == 0) *reinterpret_cast<float4*>(mine_ml + r * 4) = make_float4(x.m, x.mw, x.l, 0.f);
    } else if (!whole[0]) {
      *reinterpret_cast<float4*>(p.part + (slot * RT + r) * D + ch) = x.a;
      if (ch == 0) *reinterpret_cast<float4*>(p.part_ml + (slot * RT + r) * 4) = make_float4(x.m, x.mw, x.l, 0.f);
    } else if (r < whole[3]) {
      const int row = whole[5] * RT + r;
      write_sum(p, whole[2] + row / p.ratio, whole[4] * p.ratio + row % p.ratio, ch, x);
    }
  }
  if constexpr (CL) {
    const int size = (int)cluster_size(), rank = (int)cluster_rank();
    cluster_arrive();
    cluster_wait();
    for (int i = rank + size * threadIdx.x; i < RT * (D / 4); i += size * THREADS) {
      const int r = i / (D / 4), ch = i % (D / 4) * 4, row = at.tile * RT + r;
      if (row >= at.q.n * p.ratio) continue;
      Sum x;
      x.clear();
#pragma unroll 8
      for (int c = 0; c < size; ++c) x.add(ld_peer4(mine_ml + r * 4, c), ld_peer4(mine + r * (D + 4) + ch, c));
      write_sum(p, at.q.t0 + row / p.ratio, at.head * p.ratio + row % p.ratio, ch, x);
    }
    cluster_arrive();                                        // (no CTA ends while a peer reads from it)
    cluster_wait();
  }
}

// row r of a unit: query row (token n among the unit's, head h of the K/V head's), or false
__device__ __forceinline__ bool row_of(const PParams& p, const UnitPart& up, int r, int& n, int& h) {
  const int rr = p.tile_tokens ? r & 127 : up.row + r;
  n = rr / p.ratio;
  h = rr - n * p.ratio;
  if (p.tile_tokens && n >= p.tile_tokens) return false;
  if (p.tile_tokens) n += (r >> 7) * p.tile_tokens;
  return n < up.tokens;
}
// the i-th part's place in scratch
__device__ __forceinline__ long long slot_of(const UnitPart& up, int i, int cta_warps) {
  const int w = i < up.n0 ? up.first + i : i < up.n0 + up.n1 ? (up.cta + (i - up.n0)) * cta_warps : (up.cta + up.n1) * cta_warps + (i - up.n0 - up.n1);
  return 2LL * w + (w == up.first ? 1 : 0);
}

// Sum of the parts of the units that lie in several warps' shares.  GROUPS groups of D/4 threads a row take the parts in turn; the groups'
// sums are added in order, so a call repeats itself bit for bit.  A chain of L2 latencies: with few units, and so many parts each, one
// row a CTA and all groups on it; else one unit a CTA.
template <int D, int GROUPS>
__global__ void __launch_bounds__(GROUPS * (D / 4)) combine_kernel(const PParams p, int cta_warps, int rows_cta) {
  constexpr int C4 = D / 4;
  __shared__ float4 red[GROUPS][C4 + 1];
  __shared__ float4 red_ml[GROUPS];
  const int per_unit = p.rows_tile / rows_cta;
  const long long u = blockIdx.x / per_unit;
  const int grp = threadIdx.x / C4, ch = threadIdx.x % C4 * 4;
  pdl_wait();
  pdl_launch();
  const int units = p.head[0];
  const UnitPart up = p.units[u];                 // (the two loads do not wait for one another)
  if (u >= units || !up.open) return;
  const int parts = up.n0 + up.n1 + up.n2;
  const int first_row = (int)(blockIdx.x % per_unit) * rows_cta;
  const int row_step = rows_cta == 1 ? 1 : GROUPS, part_step = rows_cta == 1 ? GROUPS : 1;
  for (int r = first_row + (rows_cta == 1 ? 0 : grp); r < first_row + rows_cta; r += row_step) {
    int n, h;
    if (!row_of(p, up, r, n, h)) continue;
    Sum x;
    x.clear();
#pragma unroll 4
    for (int i = rows_cta == 1 ? grp : 0; i < parts; i += part_step) {
      const long long s = slot_of(up, i, cta_warps) * p.rows_tile + r;
      x.add(*reinterpret_cast<const float4*>(p.part_ml + s * 4), *reinterpret_cast<const float4*>(p.part + s * D + ch));
    }
    if (rows_cta == 1) {
      red[grp][ch / 4] = x.a;
      if (ch == 0) red_ml[grp] = make_float4(x.m, x.mw, x.l, 0.f);
      __syncthreads();
      if (grp > 0) return;
      for (int i = 1; i < GROUPS; ++i) x.add(red_ml[i], red[i][ch / 4]);
    }
    write_sum(p, up.token + n, up.head * p.ratio + h, ch, x);
  }
}

// The same for the 128-row tiles: at most one unit a CTA is open, and which are is known on the device alone.  Every CTA lists them; their
// rows are dealt out to all groups of D/4 threads of the grid.
template <int D>
__global__ void __launch_bounds__(256) combine_tiles_kernel(const PParams p, int entries) {
  constexpr int C4 = D / 4, GROUPS = 256 / C4;
  extern __shared__ int list[];
  __shared__ int counts[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = threadIdx.x / C4, ch = threadIdx.x % C4 * 4;
  pdl_wait();
  pdl_launch();
  int open_units = 0;
  for (int e0 = 0; e0 < entries; e0 += 256) {
    const int e = e0 + threadIdx.x;
    const bool open = e < entries && p.units[e].open;
    const unsigned votes = __ballot_sync(0xffffffffu, open);
    if (lane == 0) counts[warp] = __popc(votes);
    __syncthreads();
    int at = open_units;
    for (int w = 0; w < 8; ++w) {
      if (w < warp) at += counts[w];
      open_units += counts[w];
    }
    if (open) list[at + __popc(votes & ((1u << lane) - 1u))] = e;
    __syncthreads();
  }
  for (int i = blockIdx.x * GROUPS + grp; i < open_units * p.rows_tile; i += gridDim.x * GROUPS) {
    const UnitPart up = p.units[list[i / p.rows_tile]];
    const int r = i % p.rows_tile, parts = up.n0 + up.n1 + up.n2;
    int n, h;
    if (!row_of(p, up, r, n, h)) continue;
    Sum x;
    x.clear();
#pragma unroll 4
    for (int k = 0; k < parts; ++k) {
      const long long s = slot_of(up, k, 1) * p.rows_tile + r;
      x.add(*reinterpret_cast<const float4*>(p.part_ml + s * 4), *reinterpret_cast<const float4*>(p.part + s * D + ch));
    }
    write_sum(p, up.token + n, up.head * p.ratio + h, ch, x);
  }
}

#include "intfa_paged_tile.cuh"

// ---------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------
struct Plan {
  bool tiles = false;                   // 128-row tiles
  int NT = 1, ctas = 0, warps = 8;
  long long max_units = 0;
  size_t off_ml = 0, off_units = 0, off_head = 0, bytes = 0;
};
// 128-row tiles, or packed rows of 8 or 16?  A tile costs the same however many of its rows there are, and a unit on tiles takes longer to
// begin, to end and to be put together.  The lengths of the sequences are not known here; timed on both with up to 600 and 4000 keys, packed /
// on tiles, in us.  16 sequences of 8 K/V heads: at 64 channels 64 rows a head 18.5 / 26.6 and 38.9 / 57.6, 128 rows 25.3 / 30.6 and
// 63.1 / 56.3, 256 rows 39.0 / 33.9 and 125 / 77.5; at 128 channels 64 rows 25.6 / 31.0 and 58.5 / 62.9, 128 rows 35.2 / 35.8 and 100 / 63.1; at 256
// channels 32 rows 39.1 / 36.4 and 96.9 / 71.3.  Few rows in all do not fill the GPU with tiles: one sequence of 8 heads, at 64 channels 256 rows
// 20.4 / 21.7 and 31.3 / 25.8, four of one head and 512 rows 16.0 / 23.1 and 24.9 / 32.0; at 128 channels 128 rows 16.5 / 18.0 and 25.4 / 29.6, 256
// rows 21.9 / 28.8 and 42.8 / 29.0; at 256 channels 64 rows 17.5 / 18.5 and 31.5 / 31.3, 128 rows 25.8 / 21.7 and 52.7 / 37.3.
// The rule goes by the rows of an average sequence alone.  So it is off where few sequences have many keys (256 rows at 64 channels above: packed) and where
// a call mixes row counts, which all take one path (32 / 8 heads x 128: 63 single rows with up to 8192 keys and 512 rows with 4608 in one call 349 / 441,
// as two calls 117 and 79).
bool takes_tiles(const IntfaPagedParams* a) {
  if (a->debug_path) return a->debug_path == 2;
  const double rows = (double)a->tokens * (a->H / a->cache.H_kv) / a->cache.S;          // of an average sequence and K/V head
  const int D = a->cache.D;
  return a->H / a->cache.H_kv <= kTileRows && rows >= (D == 64 ? 128 : D == 128 ? 96 : 32) &&
         rows * a->cache.S * a->cache.H_kv >= (D == 64 ? 4096 : D == 128 ? 2048 : 1024);
}
Plan make_plan(const IntfaPagedParams* a, int sms) {
  Plan pl;
  const IntfaPagedCache& c = a->cache;
  const int ratio = a->H / c.H_kv;
  pl.ctas = sms;
  auto take = [&](size_t bytes) {
    const size_t r = pl.bytes;
    pl.bytes += (bytes + 255) / 256 * 256;
    return r;
  };
  pl.tiles = takes_tiles(a);
  if (pl.tiles) {
    pl.warps = 1;
    pl.max_units = pl.ctas;
    const int rows = c.D == 256 ? kTileRows : 2 * kTileRows;
    take((size_t)2 * pl.ctas * rows * c.D * 4);
    pl.off_ml = take((size_t)2 * pl.ctas * rows * 16);
    pl.off_units = take((size_t)pl.max_units * sizeof(UnitPart));
    return pl;
  }
  // Rows a tile: 16 where an average sequence has more than 8 rows a K/V head (up to 8 of them cost half in tiles of 8, more twice the bytes)
  pl.NT = (double)a->tokens * ratio > 8.0 * c.S ? 2 : 1;
  pl.warps = c.D == 256 ? 4 : 8;
  pl.max_units = (a->tokens * ratio / (8 * pl.NT) + c.S) * c.H_kv;
  if (pl.max_units > 0x7fffffffLL) return Plan();
  const int RT = 8 * pl.NT;
  const long long slots = 2LL * pl.ctas * pl.warps;
  take((size_t)slots * RT * c.D * 4);
  pl.off_ml = take((size_t)slots * RT * 16);
  pl.off_units = take((size_t)pl.max_units * sizeof(UnitPart));
  pl.off_head = take(32);
  return pl;
}

// Clusters of 2^n CTAs (up to 16) of paged_kernel that the current device holds at once, one CTA an SM; 0: none, or it cannot be asked.
template <int D, int NT, int WARPS, int NS, int G>
int cluster_places(int n) {
  static std::atomic<int> cache[64][5];                       // number + 1; 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::atomic<int>& known = cache[dev][n];
  if (const int k = known.load(std::memory_order_acquire)) return k - 1;
  auto kern = paged_kernel<D, NT, WARPS, NS, G, true>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1 << n);
  cfg.blockDim = dim3(32 * WARPS);
  cfg.dynamicSmemBytes = DecodeCfg<D, NT, WARPS, NS, G>::SMEM;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1u << n;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes) != cudaSuccess ||
      cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    clusters = 0;
  }
  known.store(clusters + 1, std::memory_order_release);
  return clusters;
}

template <int D, int NT, int WARPS, int NS, int G = 32>
int run(const IntfaPagedParams* a, const Plan& pl, PParams p, cudaStream_t stream) {
  using C = DecodeCfg<D, NT, WARPS, NS, G>;
  const IntfaPagedCache& c = a->cache;
  p.chunk_log = G == 64 ? 6 : 5;
  p.box_log = c.page_size < G ? p.page_log : p.chunk_log;
  CUtensorMap tmK, tmV;
  const CUtensorMapSwizzle swz = C::PANEL == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  int rc;
  if ((rc = make_tmap(&tmK, c.k, 1, c.k_stride, c.pages, c.H_kv, c.page_size, D, C::PANEL, 1 << p.box_log, swz))) return rc;
  if ((rc = make_tmap(&tmV, c.v, 1, c.v_stride, c.pages, c.H_kv, c.page_size, D, C::PANEL, 1 << p.box_log, swz))) return rc;
  // Units whose number is known here (one row a sequence) and which are there all at once, a cluster each: one launch and no scratch, but each
  // unit takes as long as its own keys.  Where the table has room for so few that a CTA reads 400 KB at most: measured against the shares, 32 / 8
  // heads x 128, up to 513 keys 6.4 against 9.9 us (8 sequences 7.1 / 10.6), 2048 6.7 / 9.8 (10.3 / 14.3), 8192 in clusters of 8 (270 KB) 10.7 / 11.8,
  // of 4 (540 KB) 16.0 / 15.6, 32768 26.1 / 20.1; at 64 channels 32768 (557 KB) 17.1 / 15.0, at 256 8192 (532 KB) 17.3 / 16.4.
  const long long units = (long long)c.S * c.H_kv * ((p.ratio + C::RT - 1) / C::RT);
  if (!a->cu_seqlens && units <= pl.ctas) {
    int n = 4;
    while (n >= 0 && units > cluster_places<D, NT, WARPS, NS, G>(n)) --n;
    const int size = n < 0 ? 0 : 1 << n;
    if ((long long)c.table_width * c.page_size * (2 * D + 8) <= 400000LL * size)
      return launch_clusters("paged attention", paged_kernel<D, NT, WARPS, NS, G, true>, (unsigned)(units * size), size, 32 * WARPS, C::SMEM, stream, tmK, tmV, p);
  }
  auto kern = paged_kernel<D, NT, WARPS, NS, G, false>;
  static std::atomic<bool> attr_done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return set_error(INTFA_ERR_CUDA, "cannot query the current device");
  if (!attr_done[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return set_error(INTFA_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    attr_done[dev].store(true, std::memory_order_release);
  }
  if ((rc = launch_kernel("paged attention", kern, pl.ctas, 32 * WARPS, C::SMEM, stream, tmK, tmV, p))) return rc;
  constexpr int GROUPS = 1024 / D;
  const int rows_cta = pl.max_units * p.rows_tile <= 16LL * pl.ctas ? 1 : p.rows_tile;
  const long long grid = pl.max_units * (p.rows_tile / rows_cta);
  if (grid > 0x7fffffffLL) return set_error(INTFA_ERR_TOO_LARGE, "too many query rows");
  return launch_kernel("paged combine", combine_kernel<D, GROUPS>, (unsigned)grid, GROUPS * (D / 4), 0, stream, p, WARPS, rows_cta);
}

template <int D>
int run_tiles(const IntfaPagedParams* a, const Plan& pl, PParams p, cudaStream_t stream) {
  using C = TileCfg<D>;
  const IntfaPagedCache& c = a->cache;
  CUtensorMap tmQ, tmK, tmV;
  const CUtensorMapSwizzle swz = C::PANEL == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  const int64_t qst[3] = {(int64_t)p.T * p.qn, p.qn, p.qh};
  int rc;
  if ((rc = make_tmap(&tmQ, a->q, 1, qst, 1, (int)p.T, a->H, D, C::PANEL, p.ratio, swz, p.tile_tokens))) return rc;
  if ((rc = make_tmap(&tmK, c.k, 1, c.k_stride, c.pages, c.H_kv, c.page_size, D, C::PANEL, 1 << p.box_log, swz))) return rc;
  if ((rc = make_tmap(&tmV, c.v, 1, c.v_stride, c.pages, c.H_kv, c.page_size, D, C::PANEL, 1 << p.box_log, swz))) return rc;
  auto kern = paged_tile_kernel<D>;
  static std::atomic<bool> attr_done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return set_error(INTFA_ERR_CUDA, "cannot query the current device");
  if (!attr_done[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return set_error(INTFA_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    attr_done[dev].store(true, std::memory_order_release);
  }
  if ((rc = launch_kernel("paged attention", kern, pl.ctas, C::THREADS, C::SMEM, stream, tmQ, tmK, tmV, p))) return rc;
  return launch_kernel("paged combine", combine_tiles_kernel<D>, 4 * pl.ctas, 256, pl.ctas * sizeof(int), stream, p, pl.ctas);
}

int log2_of(long long n) {
  int i = 0;
  while ((1LL << i) < n) ++i;
  return i;
}

}  // namespace

size_t paged_workspace_bytes(const IntfaPagedParams* a) {
  const int sms = sm_count_cached();
  return make_plan(a, sms > 0 ? sms : 148).bytes;
}

int paged_attention(const IntfaPagedParams* a, cudaStream_t stream) {
  const int sms = sm_count_cached();
  if (sms <= 0) return set_error(INTFA_ERR_CUDA, "cannot query SM count");
  const Plan pl = make_plan(a, sms);
  if (pl.bytes == 0) return set_error(INTFA_ERR_TOO_LARGE, "too many query rows or sequences");
  if (!a->workspace || a->workspace_bytes < pl.bytes) return set_error(INTFA_ERR_INVALID_ARG, "workspace missing or smaller than intfa_paged_workspace_bytes()");
  const IntfaPagedCache& c = a->cache;
  PParams p;
  p.q = static_cast<const int8_t*>(a->q);
  p.qs = a->q_scale;
  p.o = a->o;
  p.lse = a->lse_out;
  p.qn = a->q_stride[0]; p.qh = a->q_stride[1];
  p.qsn = a->qs_stride[0]; p.qsh = a->qs_stride[1];
  p.on = a->o_stride[0]; p.oh = a->o_stride[1];
  p.ks = c.k_scale; p.vs = c.v_scale;
  p.ksP = c.ks_stride[0]; p.ksH = c.ks_stride[1]; p.ksB = c.ks_stride[2];
  p.vsP = c.vs_stride[0]; p.vsH = c.vs_stride[1]; p.vsB = c.vs_stride[2];
  p.table = c.block_table;
  p.table_stride = c.table_stride;
  p.width = c.table_width;
  p.lens = c.seq_lens;
  p.cu = a->cu_seqlens;
  p.S = c.S; p.H = a->H; p.Hkv = c.H_kv; p.ratio = a->H / c.H_kv; p.pages = c.pages;
  p.page_log = log2_of(c.page_size);
  p.block_log = log2_of(c.block);
  p.T = a->tokens;
  p.causal = a->causal ? 1 : 0;
  p.o_bf16 = a->o_dtype == INTFA_OUT_BF16;
  p.c = a->sm_scale * 1.44269504f;
  p.workers = pl.ctas * pl.warps;
  p.least = 1;
  p.rows_tile = 8 * pl.NT;
  char* ws = static_cast<char*>(a->workspace);
  p.part = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + pl.off_ml);
  p.units = reinterpret_cast<UnitPart*>(ws + pl.off_units);
  p.max_units = pl.max_units;
  p.head = pl.tiles ? nullptr : reinterpret_cast<int*>(ws + pl.off_head);
  p.status = a->status;
  p.tile_tokens = 0;
  p.chunk_log = p.box_log = 5;
  if (pl.tiles) {
    p.rows_tile = c.D == 256 ? kTileRows : 2 * kTileRows;
    p.tile_tokens = kTileRows / p.ratio;
    p.unit_tokens = p.tile_tokens * (p.rows_tile / kTileRows);
    p.box_log = c.page_size < kTileKeys ? p.page_log : log2_of(kTileKeys);
    p.least = 2;
    return c.D == 64 ? run_tiles<64>(a, pl, p, stream) : c.D == 128 ? run_tiles<128>(a, pl, p, stream) : run_tiles<256>(a, pl, p, stream);
  }
  // Warps and chunks a ring, as timed with 64 sequences of one row and up to 8192 keys (NT 1), 32 of 4 rows, 4 query heads a K/V head, and
  // up to 4097 (NT 2), in us.  64 channels: 71.3 (12 warps with 2 chunks 73.1; chunks of 32 keys, 8 with 5: 92.8), NT 2 33.5 (7 with 3 37.8, 6 with 3
  // 39.4, 9 with 2 42; chunks of 32 keys, 8 with 4: 38.6).  128 channels: 118 (chunks of 64 keys, 6 with 2: 124, 4 with 3: 125), NT 2 49.8 (6 with 3
  // 57.8, 4 with 5 63.7).  256 channels: what fits shared memory (32 of one row 75, 55 at the copy rate; 32 of 4 rows 79 and 27: 372 bytes of its
  // accumulators spill, 78 in the cluster form).
  switch (c.D) {
    case 64: return pl.NT == 2 ? run<64, 2, 8, 2, 64>(a, pl, p, stream) : run<64, 1, 8, 3, 64>(a, pl, p, stream);
    case 128: return pl.NT == 2 ? run<128, 2, 8, 2>(a, pl, p, stream) : run<128, 1, 8, 3>(a, pl, p, stream);
    default: return pl.NT == 2 ? run<256, 2, 4, 2>(a, pl, p, stream) : run<256, 1, 4, 3>(a, pl, p, stream);
  }
}

}  // namespace intfa
