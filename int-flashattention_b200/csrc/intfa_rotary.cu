// Rotary positions of one or two tensors (q, and k with it) in one launch; the gradient of a rotation is the rotation back.
//
// Moves each value once in and once out (2 * 84 million bf16 values in 52.6 us at the measured copy rate): bound by HBM.  A CTA takes
// one token, or a few where a token has few heads: all its heads share the (cos, sin) of the position, which each lane reads once for
// its 8 channels and keeps in registers; the other half of a pair is in another lane of the row and comes by shuffles.  The next rows
// are loaded ahead of the table, so that the way from the position to its (cos, sin) overlaps them.
#include "intfa_rows.cuh"

namespace intfa {
namespace {

constexpr int kThreads = 256;

struct RotaryJob {
  const void* x[2]; void* y[2];
  long long xb[2], xh[2], xn[2], yb[2], yh[2], yn[2];
  int heads0, heads;                    // of the first tensor, of both
  long long tokens;
  int N, rot, interleaved, inverse, pos64;
  const float* table; long long rows;
  const void* pos; long long pos_b;
  int tokens_cta;                       // a power of two
  int* status;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryJob p) {
  constexpr int LPR = D / 8, SLOTS = kThreads / LPR, U = sizeof(T) == 4 ? 2 : 4;      // U: rows in flight
  const int lane_e = threadIdx.x % LPR * 8, slot = threadIdx.x / LPR;
  const int per_token = SLOTS / p.tokens_cta;
  const long long token = (long long)blockIdx.x * p.tokens_cta + slot / per_token;
  const int row0 = slot % per_token;
  pdl_wait();
  pdl_launch();
  const bool token_ok = token < p.tokens;
  const long long tok = token_ok ? token : 0;
  const int b = (int)(tok / p.N), n = (int)(tok - (long long)b * p.N);
  Raw<T> in[U];
  auto src = [&](int r) {
    const int w = r >= p.heads0, h = w ? r - p.heads0 : r;
    return static_cast<const T*>(p.x[w]) + b * p.xb[w] + h * p.xh[w] + n * p.xn[w];
  };
  auto dst = [&](int r) {
    const int w = r >= p.heads0, h = w ? r - p.heads0 : r;
    return static_cast<T*>(p.y[w]) + b * p.yb[w] + h * p.yh[w] + n * p.yn[w];
  };
  auto load = [&](int r) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      in[u].zero();
      if (token_ok && r + u * per_token < p.heads) in[u].load(src(r + u * per_token) + lane_e);
    }
  };
  load(row0);
  const long long pi = b * p.pos_b + n;
  const long long at = p.pos64 ? static_cast<const long long*>(p.pos)[pi] : static_cast<const int*>(p.pos)[pi];
  const bool ok = at >= 0 && at < p.rows;
  if (!ok && token_ok && p.status && lane_e == 0 && row0 == 0) atomicCAS(p.status, 0, kStatusBadIndex);
  Turn turn;
  turn.load(p.table, ok ? at : 0, p.rot, p.interleaved, p.inverse, lane_e);
  // (every lane of a warp makes every round, for the shuffles)
  const int rounds = (p.heads + per_token * U - 1) / (per_token * U);
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    const int r = row0 + k * per_token * U;
    if (k > 0) load(r);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = r + u * per_token;
      const bool row_ok = token_ok && row < p.heads;
      float x[8];
      widen(in[u], x);
      turn.apply(x, in[u], src(row_ok ? row : 0), row_ok, p.rot, p.interleaved, lane_e);
      if (row_ok) {
        Raw<T> out;
        narrow(x, out);
        if (lane_e >= p.rot) out = in[u];        // (as it is, a NaN's bits too)
        if (!ok) out.zero();
        out.store(dst(row) + lane_e);
      }
    }
  }
}

template <typename T>
int run(const RotaryJob& job, int D, cudaStream_t stream) {
  RotaryJob p = job;
  const int slots = kThreads / (D / 8);
  p.tokens_cta = 1;
  while (p.tokens_cta * 2 * p.heads <= slots) p.tokens_cta *= 2;
  const long long grid = (p.tokens + p.tokens_cta - 1) / p.tokens_cta;
  if (grid > 0x7fffffffLL) return set_error(INTFA_ERR_TOO_LARGE, "too many tokens");
  switch (D) {
    case 16: return launch_kernel("rotary", rotary_kernel<T, 16>, (unsigned)grid, kThreads, 0, stream, p);
    case 32: return launch_kernel("rotary", rotary_kernel<T, 32>, (unsigned)grid, kThreads, 0, stream, p);
    case 64: return launch_kernel("rotary", rotary_kernel<T, 64>, (unsigned)grid, kThreads, 0, stream, p);
    case 128: return launch_kernel("rotary", rotary_kernel<T, 128>, (unsigned)grid, kThreads, 0, stream, p);
    default: return launch_kernel("rotary", rotary_kernel<T, 256>, (unsigned)grid, kThreads, 0, stream, p);
  }
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
  p.interleaved = a->interleaved;
  p.inverse = a->inverse;
  p.pos64 = a->positions_i64;
  p.table = a->table;
  p.rows = a->table_rows;
  p.pos = a->positions;
  p.pos_b = a->positions_stride;
  p.status = a->status;
  return a->dtype == INTFA_TYPE_FP16 ? run<__half>(p, a->D, stream)
         : a->dtype == INTFA_TYPE_BF16 ? run<__nv_bfloat16>(p, a->D, stream) : run<float>(p, a->D, stream);
}

}  // namespace intfa
