// Rotary positions of one or two tensors (q, and k with it) in one launch; the gradient of a rotation is the rotation back.
//
// Moves each value once in and once out (2 * 84 million bf16 values: 340 MB, 52.6 us at the measured copy rate, 62.7 here; 148 MB of fp32, half of
// the channels rotated, 22.9 and 32.2): bound by HBM, and for a few tokens by the launch (2.4 us in a graph).  All heads of
// a token share the (cos, sin) of its position: a slot (the lanes that hold a row) reads what it needs of the table once, keeps it in
// registers and goes through several heads of one token, a few rows in flight.  The first rows are asked for ahead of the table, so
// that the way from the position to its (cos, sin) overlaps them.
#include "intfa_rows.cuh"

namespace intfa {
namespace {

constexpr int kThreads = 256;

struct RotaryJob {
  const void* x[2]; void* y[2];
  long long xb[2], xh[2], xn[2], yb[2], yh[2], yn[2];
  int heads0, heads;                    // of the first tensor, of both
  long long tokens;
  int N, rot, inverse, pos64;
  const float* table; long long rows;
  const void* pos; long long pos_b;
  int lpr_log;                          // lanes of a row, D/16
  int per_token;                        // slots that share a token
  int* status;
};

// PART: rot is no multiple of 8, so that a piece is rotated in part (2 % of the time of large calls, so not for the others)
template <typename T, int SPIN, bool PART>
__global__ void __launch_bounds__(kThreads, SPIN == kAny ? 2 : 3) rotary_kernel(const RotaryJob p) {
  constexpr int U = sizeof(T) == 4 ? 1 : 2;                  // rows in flight
  const int slot = threadIdx.x >> p.lpr_log, slots = kThreads >> p.lpr_log;
  const int row0 = slot % p.per_token;
  const long long token = (long long)blockIdx.x * (slots / p.per_token) + slot / p.per_token;
  pdl_wait();
  pdl_launch();
  if (token >= p.tokens || slot / p.per_token >= slots / p.per_token) return;
  const int b = (int)(token / p.N), n = (int)(token - (long long)b * p.N);
  Pieces at;
  at.place<SPIN>(threadIdx.x & ((1 << p.lpr_log) - 1), p.rot);
  // rows of one tensor at a time, so that a row's address is one addition
  const T* x = nullptr;
  T* y = nullptr;
  long long xs = 0, ys = 0;
  int left = 0;                                              // heads from this slot's next row on
  auto tensor = [&](int w) {
    const int heads = w ? p.heads - p.heads0 : p.heads0;
    x = static_cast<const T*>(p.x[w]) + b * p.xb[w] + n * p.xn[w] + row0 * p.xh[w];
    y = static_cast<T*>(p.y[w]) + b * p.yb[w] + n * p.yn[w] + row0 * p.yh[w];
    xs = p.per_token * p.xh[w];
    ys = p.per_token * p.yh[w];
    left = heads - row0;
  };
  Row16<T> in[U];
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u * p.per_token < left) in[u].load(x + u * xs, at);
  };
  tensor(0);
  load();
  const long long pi = b * p.pos_b + n;
  const long long pos = p.pos64 ? static_cast<const long long*>(p.pos)[pi] : static_cast<const int*>(p.pos)[pi];
  const bool ok = pos >= 0 && pos < p.rows;
  if (!ok && p.status) atomicCAS(p.status, 0, kStatusBadIndex);
  Turn<SPIN> turn;
  turn.load(p.table, ok ? pos : 0, p.rot, p.inverse, at);
#pragma unroll 1
  for (int w = 0; w < 2; ++w) {
    if (w == 1) {
      if (p.heads == p.heads0) return;
      tensor(1);
      load();
    }
#pragma unroll 1
    while (left > 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u * p.per_token >= left) break;
        float v[16];
        widen16(in[u], v);
        turn.apply(v, x + u * xs, p.rot, at);
        Raw<T> a, c;
        narrow(reinterpret_cast<const float(&)[8]>(v[0]), a);
        narrow(reinterpret_cast<const float(&)[8]>(v[8]), c);
        // (what is not rotated as it is, a NaN's bits too)
        if (at.a >= p.rot) a = in[u].a;
        if (at.b >= p.rot) c = in[u].b;
        if constexpr (PART) {
          constexpr int W = Raw<T>::W;
#pragma unroll
          for (int i = 0; i < W; ++i) {
            if (at.a + i * (8 / W) >= p.rot) a.w[i] = in[u].a.w[i];
            if (at.b + i * (8 / W) >= p.rot) c.w[i] = in[u].b.w[i];
          }
        }
        if (!ok) {
          a.zero();
          c.zero();
        }
        a.store(y + u * ys + at.a);
        c.store(y + u * ys + at.b);
      }
      x += U * xs;
      y += U * ys;
      left -= U * p.per_token;
      load();
    }
  }
}

template <typename T>
int run(const RotaryJob& job, int D, bool interleaved, cudaStream_t stream) {
  RotaryJob p = job;
  p.lpr_log = 0;
  while ((16 << p.lpr_log) < D) ++p.lpr_log;
  const int slots = kThreads >> p.lpr_log;
  // Slots a token: one for about 16 heads, so that the table and the position are paid for by 16 rows, but as many as there are
  // heads where that leaves SMs without work (a decode step)
  p.per_token = (p.heads + 15) / 16;
  while (p.per_token < p.heads && p.per_token < slots && p.tokens * p.per_token < 4LL * slots * sm_count_cached()) ++p.per_token;
  if (p.per_token > slots) p.per_token = slots;
  const int tokens_cta = slots / p.per_token;
  const long long grid = (p.tokens + tokens_cta - 1) / tokens_cta;
  if (grid > 0x7fffffffLL) return set_error(INTFA_ERR_TOO_LARGE, "too many tokens");
  auto go = [&](auto kernel) { return launch_kernel("rotary", kernel, (unsigned)grid, kThreads, 0, stream, p); };
  if (interleaved) return p.rot % 8 ? go(rotary_kernel<T, kPairs, true>) : go(rotary_kernel<T, kPairs, false>);
  return p.rot % 16 == 0 ? go(rotary_kernel<T, kHalf, false>) : go(rotary_kernel<T, kAny, true>);
}

}  // namespace

int rotary(const IntfaRotaryParams* a, cudaStream_t stream) {
  RotaryJob p;
  const void* x[2] = {a->q, a->k};
  void* y[2] = {a->q_out, a->k_out};
  const int64_t *xs[2] = {a->q_stride, a->k_stride}, *ys[2] = {a->q_out_stride, a->k_out_stride};
  for (int i = 0; i < 2; ++i) {
    p.x[i] = x[i];
    p.y[i] = y[i];
    p.xb[i] = xs[i][0]; p.xh[i] = xs[i][1]; p.xn[i] = xs[i][2];
    p.yb[i] = ys[i][0]; p.yh[i] = ys[i][1]; p.yn[i] = ys[i][2];
  }
  p.heads0 = a->H;
  p.heads = a->H + (a->k ? a->H_kv : 0);
  p.N = a->N;
  p.tokens = (long long)a->B * a->N;
  p.rot = a->rot_dim;
  p.inverse = a->inverse;
  p.pos64 = a->positions_i64;
  p.table = a->table;
  p.rows = a->table_rows;
  p.pos = a->positions;
  p.pos_b = a->positions_stride;
  p.status = a->status;
  return a->dtype == INTFA_TYPE_FP16 ? run<__half>(p, a->D, a->interleaved, stream)
         : a->dtype == INTFA_TYPE_BF16 ? run<__nv_bfloat16>(p, a->D, a->interleaved, stream) : run<float>(p, a->D, a->interleaved, stream);
}

}  // namespace intfa
