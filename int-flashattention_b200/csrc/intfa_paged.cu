// New tokens into a paged int8 cache: keys rotated by their positions, keys and values quantised with one scale for each block of
// `block` tokens and head, queries of the same tokens rotated and quantised per token, all in one launch.
//
// Reads 2 bytes a value, writes 1 (18 048 tokens of 32 + 8 + 8 heads x 128: 345 MB, 53 us at the measured copy rate): 85 us, bound by the issue of
// instructions (72 % of the slots: 300 for a warp's 16 values a lane; 126 with the rotation, of which its products and sums, each rounded by
// itself, are 48, and 80 with the proof that the codes are those of a division).  Three CTAs an SM leave 80 registers a thread, and 32 bytes
// spill (40 where pairs are neighbours).  The few tokens of a decode step: launch and latency, 5.4 us in a graph.
//   block = 1   a row (one head of one token) is quantised by the lanes that loaded it; a CTA takes one token, or a few of few heads
//   block > 1   a warp (short blocks: 12 us for 40 sequences of up to 200 tokens, where CTAs took 19) or a CTA takes what a sequence adds to one
//               block, for some heads: the largest magnitudes first, then the codes.  A block that
//               began in an earlier call keeps the larger of its old scale and the new tokens'; where that grew its older codes become
//               rint(code * (old / new)).  So a block's codes depend on how its tokens were handed over, as its scale must.
#include "intfa_rows.cuh"

namespace intfa {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 32;           // tokens of a CTA

struct AppendJob {
  const void* x[3];                      // q, k, v: packed [tokens, heads, D]
  long long xn[3], xh[3];
  int heads[3];
  int8_t* q8; float* qs;                 // contiguous
  int8_t* cache[2]; float* scale[2];     // k, v
  long long cp[2], ch[2], cn[2], sp[2], sh[2], sb[2];
  const int* table; long long table_stride; int width;
  const int* lens; const int* cu;
  int S, pages, page_log, block_log;
  long long tokens;
  const float* rot_table; long long rot_rows; int rot;
  int* status;
};

__device__ __forceinline__ int cu_at(const AppendJob& p, int s) { return p.cu ? p.cu[s] : s; }
__device__ __forceinline__ void report(const AppendJob& p) {
  if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
}

// Where a token goes.  page < 0: nowhere (it is behind the last sequence, or of one without tokens, or an index lies outside the cache).
// Called by a warp.
struct Place {
  long long pos;
  int page, slot;
  int own;                               // belongs to a sequence
};
__device__ __forceinline__ Place place_of(const AppendJob& p, long long t) {
  Place r;
  r.pos = 0;
  r.page = -1;
  r.slot = r.own = 0;
  if (t >= p.tokens) return r;
  int s = 0;
  if (p.cu) {
    const int first = p.cu[0], last = p.cu[p.S];
    if (last > p.tokens) report(p);
    if (t < first || t >= last) return r;
    s = find_last(p.S, t, [&](int i) { return (long long)p.cu[i]; });
  } else {
    s = (int)t;
  }
  const int end = cu_at(p, s + 1), len = p.lens[s];
  if (len == 0) return r;                // (padding)
  const long long pos = (long long)len - (end - t);
  r.own = 1;
  r.pos = pos;
  const long long col = pos >> p.page_log;
  if (t < end && pos >= 0 && col < p.width) {
    const int page = p.table[s * p.table_stride + col];
    if (page >= 0 && page < p.pages) {
      r.page = page;
      r.slot = (int)(pos & ((1 << p.page_log) - 1));
    }
  }
  if (r.page < 0) report(p);
  return r;
}

// Rows that each have a scale of their own, tokens_cta tokens a CTA: q's, and with KV those of K and V.  A slot (the lanes of a row) goes
// through the rows of one token in pairs, two of q or one of K and V.  Two pairs are on their way meanwhile, through shared memory, where they take
// no registers (no thread reads another's, so nothing waits for the CTA); the first are asked for ahead of where the token goes.  What a slot
// needs of the rotary table stays in registers for all rows.
struct RowRing {
  uint4 at[2][4][kThreads];              // [pair][row, piece][thread]
};
template <typename T, int D, int SPIN, bool KV>
__device__ __forceinline__ void token_rows(const AppendJob& p, long long cta, int tokens_cta, int per_token, Place* place, RowRing& ring) {
  constexpr int LPR = D / 16;
  const int slot = threadIdx.x / LPR, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mine = slot / per_token, row0 = slot % per_token;
  const long long token = cta * tokens_cta + mine;
  const bool in = token < p.tokens && mine < tokens_cta;
  const int hq = p.heads[0], hk = p.heads[1];
  const int pairs_q = (hq + 2 * per_token - 1) / (2 * per_token), pairs = pairs_q + (KV ? (hk + per_token - 1) / per_token : 0);
  Pieces at;
  at.place<SPIN>(threadIdx.x % LPR, p.rot);
  auto row_of = [&](int w) { return static_cast<const T*>(p.x[w]) + (in ? token : 0) * p.xn[w] + row0 * p.xh[w]; };
  const long long sq = per_token * p.xh[0];
  const uint32_t mem = smem_u32(&ring.at[0][0][threadIdx.x]);
  const T *la = hq > 0 ? row_of(0) : row_of(1), *lb = hq > 0 ? la + sq : row_of(2);          // the next pair to ask for
  auto load = [&](int g) {
    if (g < pairs) {
      const bool q = g < pairs_q;
      const int h = row0 + (q ? 2 * g : g - pairs_q) * per_token;
      const uint32_t to = mem + (g & 1) * (4 * kThreads * 16);
      if (in && h < (q ? hq : hk)) {
        cp_async16(to, la + at.a);
        cp_async16(to + kThreads * 16, la + at.b);
      }
      if (in && (q ? h + per_token < hq : h < hk)) {
        cp_async16(to + 2 * kThreads * 16, lb + at.a);
        cp_async16(to + 3 * kThreads * 16, lb + at.b);
      }
      if (q && g + 1 == pairs_q) {
        if (KV) {
          la = row_of(1);
          lb = row_of(2);
        }
      } else {
        la += q ? 2 * sq : per_token * p.xh[1];
        lb += q ? 2 * sq : per_token * p.xh[2];
      }
    }
    cp_async_commit();
  };
  load(0);
  load(1);
  for (int i = warp; i < tokens_cta; i += kThreads / 32) {
    const Place x = place_of(p, cta * tokens_cta + i);
    if (lane == 0) place[i] = x;
  }
  __syncthreads();
  const Place to = place[in ? mine : 0];
  Turn<SPIN> turn;
  bool goes = in && to.page >= 0;
  if constexpr (SPIN != kNone) {
    const bool pos_ok = to.pos >= 0 && to.pos < p.rot_rows;
    turn.load(p.rot_table, pos_ok ? to.pos : 0, p.rot, false, at);
    if (!pos_ok && in && to.own && threadIdx.x % LPR == 0 && row0 == 0) report(p);
    goes = goes && pos_ok;
  }
  auto take = [&](int g, Row16<T>& a, Row16<T>& b) {
    cp_async_wait<1>();
    Raw<T>* const r[4] = {&a.a, &a.b, &b.a, &b.b};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = ring.at[g & 1][i][threadIdx.x];
      r[i]->w[0] = v.x; r[i]->w[1] = v.y; r[i]->w[2] = v.z; r[i]->w[3] = v.w;
    }
    load(g + 2);
  };
  auto row = [&](const Row16<T>& raw, const T* src, bool ok, bool spin, int8_t* out, float* scale) {
    float x[16];
    widen16(raw, x);
    if (spin && ok) turn.apply(x, src, p.rot, at);
    const float s = scale_of(row_max<LPR>(absmax16(x)));
    uint32_t c[4];
    codes(x, s, c);
    if (ok) {
      *reinterpret_cast<uint2*>(out + at.a) = make_uint2(c[0], c[1]);
      *reinterpret_cast<uint2*>(out + at.b) = make_uint2(c[2], c[3]);
      if (threadIdx.x % LPR == 0) *scale = s;
    }
  };
  // (every lane of a warp makes every round, for the shuffles)
  Row16<T> r0, r1;
  int g = 0, h = row0;
  if (pairs_q > 0) {
    const T* xq = row_of(0);
    int8_t* q8 = p.q8 + (token * hq + row0) * D;
    float* qs = p.qs + token * hq + row0;
    if (in && to.own && !goes) {           // refused: zeros
      for (int i = 0; row0 + i < hq; i += per_token) {
        *reinterpret_cast<uint2*>(q8 + i * D + at.a) = *reinterpret_cast<uint2*>(q8 + i * D + at.b) = make_uint2(0u, 0u);
        if (threadIdx.x % LPR == 0) qs[i] = 0.f;
      }
    }
#pragma unroll 1
    for (; g < pairs_q; ++g) {
      take(g, r0, r1);
      row(r0, xq, goes && h < hq, true, q8, qs);
      row(r1, xq + sq, goes && h + per_token < hq, true, q8 + per_token * D, qs + per_token);
      h += 2 * per_token;
      xq += 2 * sq;
      q8 += 2 * per_token * D;
      qs += 2 * per_token;
    }
  }
  if constexpr (KV) {
    const T *xk = row_of(1), *xv = row_of(2);
    const long long page = goes ? to.page : 0;
    int8_t *ck = p.cache[0] + page * p.cp[0] + to.slot * p.cn[0] + row0 * p.ch[0], *cv = p.cache[1] + page * p.cp[1] + to.slot * p.cn[1] + row0 * p.ch[1];
    float *ak = p.scale[0] + page * p.sp[0] + to.slot * p.sb[0] + row0 * p.sh[0], *av = p.scale[1] + page * p.sp[1] + to.slot * p.sb[1] + row0 * p.sh[1];
    h = row0;
#pragma unroll 1
    for (; g < pairs; ++g) {
      take(g, r0, r1);
      row(r0, xk, goes && h < hk, true, ck, ak);
      row(r1, xv, goes && h < hk, false, cv, av);
      h += per_token;
      xk += per_token * p.xh[1];
      xv += per_token * p.xh[2];
      ck += per_token * p.ch[0];
      cv += per_token * p.ch[1];
      ak += per_token * p.sh[0];
      av += per_token * p.sh[1];
    }
  }
}

// block = 1
template <typename T, int D, int SPIN>
__global__ void __launch_bounds__(kThreads, SPIN == kAny ? 2 : 3) append_tokens_kernel(const AppendJob p, int tokens_cta, int per_token) {
  __shared__ Place place[kMaxTokens];
  __shared__ RowRing ring;
  pdl_wait();
  pdl_launch();
  token_rows<T, D, SPIN, true>(p, blockIdx.x, tokens_cta, per_token, place, ring);
}

// What one sequence adds to one block.  Unit u of sequence s: u = cu[s] / block + 2 s + i for the i-th block that the sequence touches (it
// touches at most n / block + 2).  Called by a warp.
struct BlockRun {
  long long first, b0, n0, n1;           // the sequence's first new token; the block's first token; its new ones (positions)
  int t0, page, slot0;                   // row of the sequence's first new token; page; slot of b0 in it
};
__device__ __forceinline__ bool block_run(const AppendJob& p, int u, bool report_bad, BlockRun& r) {
  const int s = p.cu ? find_last(p.S, u, [&](int i) { return (long long)(p.cu[i] >> p.block_log) + 2 * i; })
                     : find_last(p.S, u, [&](int i) { return (long long)(i >> p.block_log) + 2 * i; });
  const int t1 = cu_at(p, s + 1), block = 1 << p.block_log;
  r.t0 = cu_at(p, s);
  const long long len = p.lens[s];
  r.first = len - (t1 - r.t0);
  if (r.t0 < 0 || t1 < r.t0) {
    if (report_bad) report(p);
    return false;
  }
  if (t1 == r.t0 || len == 0) return false;
  const long long bi = (r.first >> p.block_log) + (u - ((r.t0 >> p.block_log) + 2 * s));
  r.b0 = bi << p.block_log;
  r.n0 = r.b0 > r.first ? r.b0 : r.first;
  r.n1 = r.b0 + block < len ? r.b0 + block : len;
  const long long col = r.b0 >> p.page_log;
  const bool bad = r.first < 0 || t1 > p.tokens;
  if (!bad && r.n0 >= r.n1) return false;
  r.page = !bad && col < p.width ? p.table[s * p.table_stride + col] : -1;
  if (r.page < 0 || r.page >= p.pages || (p.rot_table && r.n1 > p.rot_rows)) {
    if (report_bad) report(p);
    return false;
  }
  r.slot0 = (int)(r.b0 & ((1 << p.page_log) - 1));
  return true;
}
// 16 codes of an older token under a scale that grew
__device__ __forceinline__ void follow(int8_t* at, float was, float now) {
  const uint4 c = *reinterpret_cast<const uint4*>(at);
  const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
  const float ratio = now > 0.f && now <= 3.402823466e38f ? __fdiv_rn(was, now) : 0.f;
  uint32_t b[16], o[4];
#pragma unroll
  for (int j = 0; j < 16; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn((float)(int8_t)(cw[j / 4] >> (8 * (j & 3))), ratio), 12582912.0f));
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = __byte_perm(__byte_perm(b[4 * j], b[4 * j + 1], 0x0040), __byte_perm(b[4 * j + 2], b[4 * j + 3], 0x0040), 0x5410);
  *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
}

// Short blocks: a warp takes what a sequence adds to one block, `pairs` of the (head, K or V) one after the other, and keeps the values of one in
// registers from the maximum to the codes: nothing but shuffles between them.  CTAs from `ctas` on: q.
constexpr int kRounds = 4;               // rows a slot holds: blocks of up to 4 * 32 / (D/16) tokens
template <typename T, int D, int SPIN>
__global__ void __launch_bounds__(kThreads, 2) append_runs_kernel(const AppendJob p, int units, int groups, int pairs, int ctas, int tokens_cta, int per_token) {
  constexpr int LPR = D / 16, SLOTS = 32 / LPR;
  __shared__ Place place[kMaxTokens];
  __shared__ RowRing ring;
  pdl_wait();
  pdl_launch();
  if ((int)blockIdx.x >= ctas) {
    token_rows<T, D, SPIN, false>(p, (int)blockIdx.x - ctas, tokens_cta, per_token, place, ring);
    return;
  }
  const int lane = threadIdx.x & 31, id = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), u = id / groups, g = id - u * groups;
  BlockRun r;
  if (u >= units || !block_run(p, u, lane == 0, r)) return;
  const int slot = lane / LPR, nt = (int)(r.n1 - r.n0), older = (int)(r.n0 - r.b0), blk = r.slot0 >> p.block_log;
  Pieces at;
  at.place<SPIN>(lane % LPR, p.rot);
  const int end = min((g + 1) * pairs, 2 * p.heads[1]);
#pragma unroll 1
  for (int pair = g * pairs; pair < end; ++pair) {
    const int w = pair & 1, h = pair >> 1;
    const T* row = static_cast<const T*>(p.x[1 + w]) + (r.t0 + (r.n0 - r.first) + slot) * p.xn[1 + w] + h * p.xh[1 + w];
    float* sc = p.scale[w] + r.page * p.sp[w] + h * p.sh[w] + blk * p.sb[w];
    int8_t* out = p.cache[w] + r.page * p.cp[w] + h * p.ch[w] + r.slot0 * p.cn[w];
    Row16<T> raw[kRounds];
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      raw[k].zero();
      if (k * SLOTS + slot < nt) raw[k].load(row + k * SLOTS * p.xn[1 + w], at);
    }
    const float was = older > 0 ? *sc : 0.f;
    float x[kRounds][16], m = 0.f;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      if (k * SLOTS >= nt) break;
      widen16(raw[k], x[k]);
      if (SPIN != kNone && w == 0 && k * SLOTS + slot < nt) {
        Turn<SPIN> turn;
        turn.load(p.rot_table, r.n0 + k * SLOTS + slot, p.rot, false, at);
        turn.apply(x[k], row + k * SLOTS * p.xn[1 + w], p.rot, at);
      }
      m = max_nan(m, absmax16(x[k]));
    }
    const float now = max_nan(was, scale_of(row_max<32>(m)));
    __syncwarp();                          // (all lanes have read the old scale)
    if (lane == 0) *sc = now;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      if (k * SLOTS >= nt) break;
      uint32_t c[4];
      codes(x[k], now, c);
      if (k * SLOTS + slot < nt) {
        int8_t* o = out + (older + k * SLOTS + slot) * p.cn[w];
        *reinterpret_cast<uint2*>(o + at.a) = make_uint2(c[0], c[1]);
        *reinterpret_cast<uint2*>(o + at.b) = make_uint2(c[2], c[3]);
      }
    }
    if (__float_as_uint(was) != __float_as_uint(now))
      for (int i = slot; i < older; i += SLOTS) follow(out + i * p.cn[w] + lane % LPR * 16, was, now);
  }
}

// Longer blocks: a CTA takes them, some heads at a time; maxima first, then the rows once more for the codes.  CTAs from units * groups on: q.
// 40 sequences of up to 200 tokens, 32 + 8 + 8 heads x 128, blocks of 64: 50 us (short blocks of 16: 34; 97 MB, 15 us): rows are read and rotated twice.
template <typename T, int D, int SPIN>
__global__ void __launch_bounds__(kThreads, 2) append_blocks_kernel(const AppendJob p, int units, int groups, int heads_cta, int tokens_cta, int per_token) {
  constexpr int LPR = D / 16, SLOTS = kThreads / LPR;
  __shared__ Place place[kMaxTokens];
  __shared__ RowRing ring;
  __shared__ unsigned int most[2 * kThreads];        // [K, V][heads_cta]
  __shared__ float s_old[2 * kThreads], s_new[2 * kThreads];
  pdl_wait();
  pdl_launch();
  if ((long long)blockIdx.x >= (long long)units * groups) {
    token_rows<T, D, SPIN, false>(p, (long long)blockIdx.x - (long long)units * groups, tokens_cta, per_token, place, ring);
    return;
  }
  const int u = blockIdx.x / groups, head0 = (blockIdx.x - u * groups) * heads_cta, nh = min(heads_cta, p.heads[1] - head0);
  BlockRun run;
  if (!block_run(p, u, threadIdx.x == 0, run)) return;
  const int slot0 = run.slot0, blk = slot0 >> p.block_log, page = run.page, older = (int)(run.n0 - run.b0);
  const int slot = threadIdx.x / LPR;
  Pieces at;
  at.place<SPIN>(threadIdx.x % LPR, p.rot);
  for (int i = threadIdx.x; i < 2 * nh; i += kThreads) most[i] = 0u;
  __syncthreads();
  const int nt = (int)(run.n1 - run.n0), rows = nt * nh * 2, rounds = (rows + SLOTS - 1) / SLOTS;
  // row r: token r / (2 nh), then K's heads and V's
  float x[16];
  auto fetch = [&](int k, int& token, int& wh) {
    const int r = k * SLOTS + slot;
    const bool ok = r < rows;
    token = ok ? r / (2 * nh) : 0;
    wh = ok ? r - token * 2 * nh : 0;
    const int w = wh >= nh ? 1 : 0, h = head0 + wh - (w ? nh : 0);
    const T* row = static_cast<const T*>(p.x[1 + w]) + (run.t0 + (run.n0 - run.first) + token) * p.xn[1 + w] + h * p.xh[1 + w];
    Row16<T> raw;
    raw.zero();
    if (ok) raw.load(row, at);
    widen16(raw, x);
    if (SPIN != kNone && ok && w == 0) {
      Turn<SPIN> turn;
      turn.load(p.rot_table, run.n0 + token, p.rot, false, at);
      turn.apply(x, row, p.rot, at);
    }
    return ok;
  };
  int token = 0, wh = 0;
  bool ok = false;
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    ok = fetch(k, token, wh);
    const float m = row_max<LPR>(absmax16(x));
    if (ok && threadIdx.x % LPR == 0) atomicMax(&most[wh], __float_as_uint(m));       // (not negative, a NaN above all: they compare as whole numbers)
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * nh; i += kThreads) {
    const int w = i >= nh ? 1 : 0, h = head0 + i - (w ? nh : 0);
    float* sc = p.scale[w] + page * p.sp[w] + h * p.sh[w] + blk * p.sb[w];
    const float old = older > 0 ? *sc : 0.f, now = max_nan(old, scale_of(__uint_as_float(most[i])));
    s_old[i] = old;
    s_new[i] = now;
    *sc = now;
  }
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    if (rounds > 1) ok = fetch(k, token, wh);
    if (!ok) continue;
    const int w = wh >= nh ? 1 : 0, h = head0 + wh - (w ? nh : 0);
    uint32_t c[4];
    codes(x, s_new[wh], c);
    int8_t* out = p.cache[w] + page * p.cp[w] + h * p.ch[w] + (slot0 + older + token) * p.cn[w];
    *reinterpret_cast<uint2*>(out + at.a) = make_uint2(c[0], c[1]);
    *reinterpret_cast<uint2*>(out + at.b) = make_uint2(c[2], c[3]);
  }
#pragma unroll 1
  for (int r = slot; r < older * nh * 2; r += SLOTS) {
    const int tk = r / (2 * nh), i = r - tk * 2 * nh, w = i >= nh ? 1 : 0, h = head0 + i - (w ? nh : 0);
    if (__float_as_uint(s_old[i]) == __float_as_uint(s_new[i])) continue;
    follow(p.cache[w] + page * p.cp[w] + h * p.ch[w] + (slot0 + tk) * p.cn[w] + threadIdx.x % LPR * 16, s_old[i], s_new[i]);
  }
}

template <typename T, int D, int SPIN>
int run(const AppendJob& p, cudaStream_t stream) {
  constexpr int SLOTS = kThreads / (D / 16);
  // Slots a token: one for about 12 rows, but as many as there are rows where that leaves SMs without work (a decode step)
  auto slots_of = [&](int heads) {
    int n = 1;
    while (n * 12 < heads || (n < heads && p.tokens * n < 3LL * SLOTS * sm_count_cached())) n *= 2;
    if (n < SLOTS / kMaxTokens) n = SLOTS / kMaxTokens;
    return n < SLOTS ? n : SLOTS;
  };
  if (p.block_log == 0) {
    const int per = slots_of(p.heads[0] > 0 ? p.heads[0] + 2 * p.heads[1] : 2 * p.heads[1]), n = SLOTS / per;
    const long long grid = (p.tokens + n - 1) / n;
    if (grid > 0x7fffffffLL) return set_error(INTFA_ERR_TOO_LARGE, "too many tokens");
    return launch_kernel("append", append_tokens_kernel<T, D, SPIN>, (unsigned)grid, kThreads, 0, stream, p, n, per);
  }
  const int per = p.q8 ? slots_of(p.heads[0]) : SLOTS, n = SLOTS / per;
  const long long units = (p.tokens >> p.block_log) + 2LL * p.S, q_ctas = p.q8 ? (p.tokens + n - 1) / n : 0;
  if constexpr (SPIN != kAny) {           // (whose element-wise way has no registers for it)
    if ((1 << p.block_log) <= kRounds * 32 / (D / 16)) {
      // (head, K or V) pairs a warp: so many that all warps are there at once, eight at most
      long long pairs = units * 2 * p.heads[1] / (16LL * sm_count_cached());
      pairs = pairs < 1 ? 1 : pairs > 8 ? 8 : pairs;
      const long long groups = (2 * p.heads[1] + pairs - 1) / pairs, ctas = (units * groups + kThreads / 32 - 1) / (kThreads / 32);
      if (units * groups > 0x7fffffffLL || ctas + q_ctas > 0x7fffffffLL) return set_error(INTFA_ERR_TOO_LARGE, "too many tokens");
      return launch_kernel("append", append_runs_kernel<T, D, SPIN>, (unsigned)(ctas + q_ctas), kThreads, 0, stream, p, (int)units, (int)groups, (int)pairs, (int)ctas, n,
                           per);
    }
  }
  // Heads a CTA: one or two rounds of rows
  int heads_cta = 2 * SLOTS / (2 << p.block_log);
  if (heads_cta < 1) heads_cta = 1;
  if (heads_cta > p.heads[1]) heads_cta = p.heads[1];
  if (heads_cta > kThreads) heads_cta = kThreads;
  const int groups = (p.heads[1] + heads_cta - 1) / heads_cta;
  if (units * groups + q_ctas > 0x7fffffffLL) return set_error(INTFA_ERR_TOO_LARGE, "too many tokens");
  return launch_kernel("append", append_blocks_kernel<T, D, SPIN>, (unsigned)(units * groups + q_ctas), kThreads, 0, stream, p, (int)units, groups, heads_cta, n, per);
}
template <typename T, int D>
int run_spin(const AppendJob& p, bool interleaved, cudaStream_t stream) {
  if (!p.rot_table) return run<T, D, kNone>(p, stream);
  if (interleaved) return run<T, D, kPairs>(p, stream);
  return p.rot % 16 == 0 ? run<T, D, kHalf>(p, stream) : run<T, D, kAny>(p, stream);
}

int log2_of(long long n) {
  int i = 0;
  while ((1LL << i) < n) ++i;
  return i;
}

}  // namespace

int paged_append(const IntfaAppendParams* a, cudaStream_t stream) {
  AppendJob p;
  const void* x[3] = {a->q, a->k, a->v};
  const int64_t* xs[3] = {a->q_stride, a->k_stride, a->v_stride};
  for (int i = 0; i < 3; ++i) {
    p.x[i] = x[i];
    p.xn[i] = xs[i][0];
    p.xh[i] = xs[i][1];
  }
  p.heads[0] = a->q ? a->H : 0;
  p.heads[1] = p.heads[2] = a->cache.H_kv;
  p.q8 = a->q ? static_cast<int8_t*>(a->q8) : nullptr;
  p.qs = a->q_scale;
  const IntfaPagedCache& c = a->cache;
  p.cache[0] = static_cast<int8_t*>(c.k);
  p.cache[1] = static_cast<int8_t*>(c.v);
  p.scale[0] = c.k_scale;
  p.scale[1] = c.v_scale;
  const int64_t *cs[2] = {c.k_stride, c.v_stride}, *ss[2] = {c.ks_stride, c.vs_stride};
  for (int i = 0; i < 2; ++i) {
    p.cp[i] = cs[i][0]; p.ch[i] = cs[i][1]; p.cn[i] = cs[i][2];
    p.sp[i] = ss[i][0]; p.sh[i] = ss[i][1]; p.sb[i] = ss[i][2];
  }
  p.table = c.block_table;
  p.table_stride = c.table_stride;
  p.width = c.table_width;
  p.lens = c.seq_lens;
  p.cu = a->cu_seqlens;
  p.S = c.S;
  p.pages = c.pages;
  p.page_log = log2_of(c.page_size);
  p.block_log = log2_of(c.block);
  p.tokens = a->tokens;
  p.rot_table = a->table;
  p.rot_rows = a->table_rows;
  p.rot = a->rot_dim;
  p.status = a->status;
  const bool f16 = a->dtype == INTFA_TYPE_FP16, pairs = a->interleaved != 0;
  switch (c.D) {
    case 64: return f16 ? run_spin<__half, 64>(p, pairs, stream) : run_spin<__nv_bfloat16, 64>(p, pairs, stream);
    case 128: return f16 ? run_spin<__half, 128>(p, pairs, stream) : run_spin<__nv_bfloat16, 128>(p, pairs, stream);
    default: return f16 ? run_spin<__half, 256>(p, pairs, stream) : run_spin<__nv_bfloat16, 256>(p, pairs, stream);
  }
}

}  // namespace intfa
