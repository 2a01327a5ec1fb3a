// softmax_ce.hip — softmax cross entropy of queries against embedding rows, and its gradient. The
// logits are made tile by tile in registers (seq_dev.h) and never stored: the forward keeps one
// running maximum and sum per query, the backward makes the logits again from the same tiles.
#include <algorithm>

#include "mono_common.h"
#include "seq_dev.h"

namespace mono {
namespace {
using namespace seq;

struct Args {
  const void *q, *w;
  int64_t qs, ws;
  const int64_t* labels;
  const float *bias, *grad;
  float *lse, *loss;
  void *dq, *dw;
  float* db;
  float *part, *part2;  // forward: maximum and sum of every split; backward: partial gradients
  int n, v, D, nsplit;
  float scale, scale2;
  int vec_q, vec_w, vec_o;
};

template <typename T, int DP>
struct Tile {
  static constexpr int BN = DP * sizeof(T) <= 256 ? 64 : 32, NR = BN / 32;
};

// what the products of a candidate start from: its bias in units of scale
__device__ inline float start_of(const float* bias, int v, float inv_scale) {
  return bias ? bias[v] * inv_scale : 0.f;
}
__device__ inline void range_of(int n, int nsplit, int split, int BN, int* beg, int* end) {
  const int chunk = ((n + nsplit - 1) / nsplit + BN - 1) / BN * BN;
  *beg = (int)min((int64_t)n, (int64_t)split * chunk);
  *end = (int)min((int64_t)n, (int64_t)*beg + chunk);
}

// ---- forward: running maximum and sum of a tile of queries over one piece of the vocabulary ----
template <typename T, int DP, int NC>
__global__ __launch_bounds__(256, DP <= 128 || sizeof(T) == 2 ? 2 : 1) void k_ce_fwd(Args a) {
  constexpr int BM = NC * 128, BN = Tile<T, DP>::BN, NR = Tile<T, DP>::NR;
  typedef Stage<T, DP, BN, 256> St;
  typedef Mma<T, DP, St::PLANE> M;
  __shared__ __align__(16) bf16 lw[St::LDS];
  __shared__ __align__(16) float lb[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int col[NC];
  typename M::Frag qf[NC][M::KF];
  float m[NC], l[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = blockIdx.x * BM + (wave * NC + c) * 32 + (lane & 31);
    const bool ok = col[c] < a.n;
    M::load_cols(qf[c], (const T*)a.q + (int64_t)(ok ? col[c] : 0) * a.qs, ok, a.D, a.vec_q, lane);
    m[c] = neg_inf();
    l[c] = 0.f;
  }
  int vbeg, vend;
  range_of(a.v, a.nsplit, blockIdx.y, BN, &vbeg, &vend);
  St st;
  float eb = 0.f;
  const float inv_scale = 1.f / a.scale;
  const Rows<T> wr = {(const T*)a.w, a.ws, a.D, a.vec_w != 0};
  auto fetch = [&](int y0) {
    st.load(wr, y0, vend, tid, a.bias, [&](int row) { return a.bias[row] != neg_inf(); });
    if (tid < BN) eb = y0 + tid < vend ? start_of(a.bias, y0 + tid, inv_scale) : neg_inf();
  };
  if (vbeg < vend) fetch(vbeg);
  for (int y0 = vbeg; y0 < vend; y0 += BN) {
    __syncthreads();
    st.store(lw, tid, a.bias);
    if (tid < BN) lb[tid] = eb;
    __syncthreads();
    if (y0 + BN < vend) fetch(y0 + BN);
    f16v s[NR][NC];
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) {
      f16v from = all_of(0.f);
      if (a.bias || y0 + BN > vend) from = by_rows(lb + 32 * rt, lane);
      M::template scores<NC>(lw, rt, qf, s[rt], from, lane);
    }
    // every lane keeps the maximum and sum of the candidates that it holds itself; the two lanes
    // of a query are joined once, behind the loop. m is in units of scale (scale > 0).
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float mx = m[c];
#pragma unroll
      for (int rt = 0; rt < NR; ++rt)
#pragma unroll
        for (int r = 0; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[rt][c][r]), s[rt][c][r + 1]);
      const float base = mx == neg_inf() ? 0.f : mx * a.scale2;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int rt = 0; rt < NR; ++rt)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r & 1] += exp2_hw(fmaf(s[rt][c][r], a.scale2, -base));
      l[c] = fmaf(l[c], exp2_hw(fmaf(m[c], a.scale2, -base)), sum[0] + sum[1]);
      m[c] = mx;
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float mx = col_max(m[c]) * a.scale2, base = mx == neg_inf() ? 0.f : mx;
    const float sum = col_sum(l[c] * exp2_hw(fmaf(m[c], a.scale2, -base)));
    if (lane < 32 && col[c] < a.n) {
      a.part[(int64_t)blockIdx.y * a.n + col[c]] = mx;
      a.part2[(int64_t)blockIdx.y * a.n + col[c]] = sum;
    }
  }
}

// One wave per query: joins the pieces of the vocabulary and takes the label's own logit off.
template <typename T>
__global__ __launch_bounds__(256) void k_ce_loss(Args a) {
  const int lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= a.n) return;
  float m = neg_inf();
  for (int s = lane; s < a.nsplit; s += 64) m = fmaxf(m, a.part[(int64_t)s * a.n + i]);
#pragma unroll
  for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  const float base = m == neg_inf() ? 0.f : m;
  float z = 0.f;
  for (int s = lane; s < a.nsplit; s += 64)
    z += a.part2[(int64_t)s * a.n + i] * exp2_hw(a.part[(int64_t)s * a.n + i] - base);
  const int64_t label = a.labels[i];
  const bool known = label >= 0 && label < a.v;
  float hit = 0.f;
  if (known)
    for (int d = lane; d < a.D; d += 64)
      hit = fmaf((float)((const T*)a.q)[(int64_t)i * a.qs + d], (float)((const T*)a.w)[label * a.ws + d], hit);
#pragma unroll
  for (int x = 32; x; x >>= 1) {
    z += __shfl_xor(z, x);
    hit += __shfl_xor(hit, x);
  }
  if (lane) return;
  const float b = known && a.bias ? a.bias[label] : 0.f;
  const bool out = b == neg_inf();
  const float lse = m + __log2f(z);
  float loss = fmaf(lse, kLn2, -fmaf(hit, a.scale, b));
  if (out) loss = __builtin_inff();
  if (!known) loss = label == -1 ? 0.f : __builtin_nanf("");
  a.loss[i] = loss;
  a.lse[i] = known && !out ? lse : __builtin_inff();
}

// ---- backward ------------------------------------------------------------------------------
// dquery_i = scale g_i (sum_v p_iv w_v - w_label): g and the label's row are taken in behind the
// loop, in 32 bits, so that the products see nothing but the probabilities.
template <typename T>
__device__ inline f4 minus_label(const Args& a, int i, int d0, f4 t) {
  const float lse = a.lse[i];
  if (lse == __builtin_inff()) return f4{0.f, 0.f, 0.f, 0.f};
  const float g = a.grad[i] * a.scale;
  const T* w = (const T*)a.w + a.labels[i] * a.ws;
#pragma unroll
  for (int r = 0; r < 4; ++r) t[r] = d0 + r < a.D ? g * (t[r] - (float)w[d0 + r]) : 0.f;
  return t;
}

template <typename T, int DP, int NC>
__global__ __launch_bounds__(256, DP * sizeof(T) <= 256 ? 2 : 1) void k_ce_dq(Args a) {
  constexpr int BM = NC * 128, BN = Tile<T, DP>::BN, NR = Tile<T, DP>::NR;
  typedef Stage<T, DP, BN, 256> St;
  typedef Mma<T, DP, St::PLANE> M;
  __shared__ __align__(16) bf16 lw[St::LDS];
  __shared__ __align__(16) float lb[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int col[NC];
  typename M::Frag qf[NC][M::KF];
  float lse[NC];
  f16v acc[M::NDT][NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = blockIdx.x * BM + (wave * NC + c) * 32 + (lane & 31);
    const bool ok = col[c] < a.n;
    M::load_cols(qf[c], (const T*)a.q + (int64_t)(ok ? col[c] : 0) * a.qs, ok, a.D, a.vec_q, lane);
    lse[c] = ok ? a.lse[col[c]] : __builtin_inff();
#pragma unroll
    for (int d = 0; d < M::NDT; ++d) acc[d][c] = all_of(0.f);
  }
  int vbeg, vend;
  range_of(a.v, a.nsplit, blockIdx.y, BN, &vbeg, &vend);
  St st;
  float eb = 0.f;
  const float inv_scale = 1.f / a.scale;
  const Rows<T> wr = {(const T*)a.w, a.ws, a.D, a.vec_w != 0};
  auto fetch = [&](int y0) {
    st.load(wr, y0, vend, tid, a.bias, [&](int row) { return a.bias[row] != neg_inf(); });
    if (tid < BN) eb = y0 + tid < vend ? start_of(a.bias, y0 + tid, inv_scale) : neg_inf();
  };
  if (vbeg < vend) fetch(vbeg);
  for (int y0 = vbeg; y0 < vend; y0 += BN) {
    __syncthreads();
    st.store(lw, tid, a.bias);
    if (tid < BN) lb[tid] = eb;
    __syncthreads();
    if (y0 + BN < vend) fetch(y0 + BN);
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) {
      f16v s[NC], from = all_of(0.f);
      if (a.bias || y0 + BN > vend) from = by_rows(lb + 32 * rt, lane);
      M::template scores<NC>(lw, rt, qf, s, from, lane);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[c][r] = exp2_hw(fmaf(s[c][r], a.scale2, -lse[c]));
      M::template accumulate<NC>(lw, rt, s, acc, lane);
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (col[c] >= a.n) continue;
    if (a.part) {
      store_col(a.part + ((int64_t)blockIdx.y * a.n + col[c]) * a.D, a.D, acc, c, 1.f, a.vec_o, lane);
      continue;
    }
#pragma unroll
    for (int d = 0; d < M::NDT; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d0 = 32 * d + 8 * q + 4 * (lane >> 5);
        const f4 t = {acc[d][c][4 * q], acc[d][c][4 * q + 1], acc[d][c][4 * q + 2], acc[d][c][4 * q + 3]};
        if (d0 < a.D)
          store4((T*)a.dq + (int64_t)col[c] * a.D, d0, a.D, minus_label<T>(a, col[c], d0, t), a.vec_o);
      }
  }
}

// dquery from the splits' partial sums, four elements of a row per thread
template <typename T>
__global__ __launch_bounds__(256) void k_ce_dq_join(Args a) {
  const int per = (a.D + 3) / 4;
  const int64_t total = (int64_t)a.n * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int row = (int)(i / per), d0 = (int)(i % per) * 4;
    f4 t = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.nsplit; ++s) {
      const float* p = a.part + ((int64_t)s * a.n + row) * a.D;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (d0 + r < a.D) t[r] += p[d0 + r];
    }
    store4((T*)a.dq + (int64_t)row * a.D, d0, a.D, minus_label<T>(a, row, d0, t), a.vec_o);
  }
}

// drows_v = scale sum_i g_i (p_iv - [v = label_i]) query_i, dbias_v the same without scale and query:
// a tile of candidates keeps its sums while all queries stream by. The label's share is rare: one
// ballot per tile of queries says whether any label falls into the candidates of the workgroup.
template <typename T, int DP, int NC>
__global__ __launch_bounds__(256, DP * sizeof(T) <= 256 ? 2 : 1) void k_ce_dw(Args a) {
  constexpr int BM = NC * 128, BN = Tile<T, DP>::BN, NR = Tile<T, DP>::NR;
  typedef Stage<T, DP, BN, 256> St;
  typedef Mma<T, DP, St::PLANE> M;
  __shared__ __align__(16) bf16 lq[St::LDS];
  __shared__ __align__(16) float ll[BN], lg[BN];
  __shared__ __align__(16) int lab[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int v0 = blockIdx.x * BM;
  int col[NC];
  typename M::Frag wf[NC][M::KF];
  float b2[NC], sb[NC];
  f16v acc[M::NDT][NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = v0 + (wave * NC + c) * 32 + (lane & 31);
    const bool ok = col[c] < a.v;
    b2[c] = !ok ? neg_inf() : a.bias ? a.bias[col[c]] * kLog2e : 0.f;
    M::load_cols(wf[c], (const T*)a.w + (int64_t)(ok ? col[c] : 0) * a.ws, b2[c] != neg_inf(), a.D, a.vec_w, lane);
    sb[c] = 0.f;
#pragma unroll
    for (int d = 0; d < M::NDT; ++d) acc[d][c] = all_of(0.f);
  }
  int nbeg, nend;
  range_of(a.n, a.nsplit, blockIdx.y, BN, &nbeg, &nend);
  St st;
  const Rows<T> qr = {(const T*)a.q, a.qs, a.D, a.vec_q != 0};
  const float inv_scale2 = 1.f / a.scale2;
  float el = 0.f, eg = 0.f;
  int lb = -1;
  auto fetch = [&](int y0) {
    st.load(qr, y0, nend, tid, true, [&](int row) { return a.lse[row] != __builtin_inff(); });
    if (tid < BN) {
      el = __builtin_inff();
      eg = 0.f;
      lb = -1;
      if (y0 + tid < nend) {
        el = a.lse[y0 + tid];
        if (el != __builtin_inff()) {
          eg = a.grad[y0 + tid];
          lb = (int)a.labels[y0 + tid];
        }
      }
    }
  };
  if (nbeg < nend) fetch(nbeg);
  for (int y0 = nbeg; y0 < nend; y0 += BN) {
    __syncthreads();
    st.store(lq, tid, true);
    if (tid < BN) {
      ll[tid] = -el * inv_scale2;
      lg[tid] = eg;
      lab[tid] = lb;
    }
    __syncthreads();
    if (y0 + BN < nend) fetch(y0 + BN);
    const int mine = lab[lane & (BN - 1)];
    const bool hits = __any(mine >= v0 && mine < v0 + BM);
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) {
      f16v s[NC];
      M::template scores<NC>(lq, rt, wf, s, by_rows(ll + 32 * rt, lane), lane);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[c][r] = exp2_hw(fmaf(s[c][r], a.scale2, b2[c]));
      if (hits) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int label = lab[32 * rt + tile_row(r, lane)];
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (label == col[c]) s[c][r] -= 1.f;
        }
      }
      const f16v g = by_rows(lg + 32 * rt, lane);
#pragma unroll
      for (int c = 0; c < NC; ++c) s[c] *= g;
      if (a.db) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int r = 0; r < 16; ++r) sb[c] += s[c][r];
      }
      M::template accumulate<NC>(lq, rt, s, acc, lane);
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float b = col_sum(sb[c]);
    if (col[c] >= a.v) continue;
    const int64_t row = (a.nsplit > 1 ? (int64_t)blockIdx.y * a.v : 0) + col[c];
    if (a.db && lane < 32) (a.nsplit > 1 ? a.part2 : a.db)[row] = b;
    if (!a.dw) continue;
    if (a.nsplit > 1) store_col(a.part + row * a.D, a.D, acc, c, a.scale, a.vec_o, lane);
    else store_col((T*)a.dw + row * a.D, a.D, acc, c, a.scale, a.vec_o, lane);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_ce_sum(const float* part, int n_part, int64_t total, T* out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    float t = 0.f;
    for (int s = 0; s < n_part; ++s) t += part[(int64_t)s * total + i];
    out[i] = (T)t;
  }
}

// ---- host ----------------------------------------------------------------------------------
int cols_of(const mono_softmax_ce_args* p) {
  return p->dtype == MONO_ROW_BF16 && p->dim <= 64 ? 2 : 1;
}
// tiles of `kept` rows, and pieces of the streamed rows that fill the card when there are few tiles
int64_t tiles_of(const mono_softmax_ce_args* p, int64_t kept) {
  const int bm = 128 * cols_of(p);
  return (kept + bm - 1) / bm;
}
int pieces_of(const mono_softmax_ce_args* p, int64_t kept, int64_t streamed) {
  const int64_t tiles = tiles_of(p, kept), want = 256 * 4;
  if (tiles >= want) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(want / std::max<int64_t>(1, tiles), streamed / 64));
}

int check(const mono_softmax_ce_args* p, const char* who) {
  MONO_REQUIRE(p != nullptr, "%s: args is NULL", who);
  MONO_REQUIRE(p->dtype == MONO_ROW_FP32 || p->dtype == MONO_ROW_BF16, "%s: unknown row type %d", who, p->dtype);
  MONO_REQUIRE(p->dim >= 1 && p->dim <= 256, "%s: dim must be in [1, 256], got %d", who, p->dim);
  MONO_REQUIRE(p->scale > 0.f && p->scale < __builtin_inff(), "%s: scale must be positive and finite", who);
  MONO_REQUIRE(p->n >= 0 && p->vocab >= 1 && p->n < (1LL << 31) - 65536 && p->vocab < (1LL << 31) - 65536,
               "%s: %lld queries and %lld rows are out of range", who, (long long)p->n, (long long)p->vocab);
  return 0;
}
Args base_args(const mono_softmax_ce_args* p) {
  Args a{};
  const int e = p->dtype == MONO_ROW_BF16 ? 8 : 4;
  a.q = p->query, a.qs = p->query_stride, a.w = p->rows, a.ws = p->rows_stride;
  a.labels = p->labels, a.bias = p->bias, a.grad = p->grad_loss, a.lse = p->lse, a.loss = p->loss;
  a.dq = p->grad_query, a.dw = p->grad_rows, a.db = p->grad_bias;
  a.n = (int)p->n, a.v = (int)p->vocab, a.D = p->dim, a.nsplit = 1;
  a.scale = p->scale, a.scale2 = p->scale * kLog2e;
  a.vec_q = p->dim % e == 0 && p->query_stride % e == 0 && ((uintptr_t)p->query & 15) == 0;
  a.vec_w = p->dim % e == 0 && p->rows_stride % e == 0 && ((uintptr_t)p->rows & 15) == 0;
  a.vec_o = p->dim % e == 0 && (((uintptr_t)p->grad_query | (uintptr_t)p->grad_rows) & 15) == 0;
  return a;
}

enum Which { kFwd, kDq, kDw };
template <int W, typename T, int DP, int NC>
int launch1(const Args& a, int64_t tiles, hipStream_t st) {
  const dim3 grid((unsigned)tiles, (unsigned)a.nsplit);
  if (W == kFwd) k_ce_fwd<T, DP, NC><<<grid, 256, 0, st>>>(a);
  else if (W == kDq) k_ce_dq<T, DP, NC><<<grid, 256, 0, st>>>(a);
  else k_ce_dw<T, DP, NC><<<grid, 256, 0, st>>>(a);
  MONO_HIP(hipGetLastError());
  return 0;
}
template <int W>
int launch(int dtype, const Args& a, int64_t tiles, hipStream_t st) {
  if (dtype == MONO_ROW_BF16) {
    if (a.D <= 16) return launch1<W, bf16, 16, 2>(a, tiles, st);
    if (a.D <= 32) return launch1<W, bf16, 32, 2>(a, tiles, st);
    if (a.D <= 64) return launch1<W, bf16, 64, 2>(a, tiles, st);
    if (a.D <= 128) return launch1<W, bf16, 128, 1>(a, tiles, st);
    return launch1<W, bf16, 256, 1>(a, tiles, st);
  }
  if (a.D <= 16) return launch1<W, float, 16, 1>(a, tiles, st);
  if (a.D <= 32) return launch1<W, float, 32, 1>(a, tiles, st);
  if (a.D <= 64) return launch1<W, float, 64, 1>(a, tiles, st);
  if (a.D <= 128) return launch1<W, float, 128, 1>(a, tiles, st);
  return launch1<W, float, 256, 1>(a, tiles, st);
}
int64_t round16(int64_t b) { return (b + 15) & ~(int64_t)15; }
template <typename T>
int sum_parts(const float* part, int n_part, int64_t total, T* out, hipStream_t st) {
  k_ce_sum<T><<<grid_for(total, 256), 256, 0, st>>>(part, n_part, total, out);
  MONO_HIP(hipGetLastError());
  return 0;
}
}  // namespace
}  // namespace mono

extern "C" {
using namespace mono;

int64_t mono_softmax_cross_entropy_workspace(const mono_softmax_ce_args* p) {
  if (check(p, "mono_softmax_cross_entropy_workspace")) return -1;
  return 2 * round16((int64_t)pieces_of(p, p->n, p->vocab) * p->n * 4);
}

int mono_softmax_cross_entropy(const mono_softmax_ce_args* p, void* stream) {
  MONO_TRY(check(p, "mono_softmax_cross_entropy"));
  if (p->n == 0) return 0;
  MONO_REQUIRE(p->workspace_bytes >= mono_softmax_cross_entropy_workspace(p),
               "mono_softmax_cross_entropy: workspace of %lld bytes is too small", (long long)p->workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  Args a = base_args(p);
  a.nsplit = pieces_of(p, p->n, p->vocab);
  a.part = (float*)p->workspace;
  a.part2 = (float*)((char*)p->workspace + round16((int64_t)a.nsplit * p->n * 4));
  MONO_TRY(launch<kFwd>(p->dtype, a, tiles_of(p, p->n), st));
  const unsigned grid = (unsigned)((p->n + 3) / 4);
  if (p->dtype == MONO_ROW_BF16) k_ce_loss<bf16><<<grid, 256, 0, st>>>(a);
  else k_ce_loss<float><<<grid, 256, 0, st>>>(a);
  MONO_HIP(hipGetLastError());
  return 0;
}

int64_t mono_softmax_cross_entropy_gradient_workspace(const mono_softmax_ce_args* p) {
  if (check(p, "mono_softmax_cross_entropy_gradient_workspace")) return -1;
  const int64_t sq = pieces_of(p, p->n, p->vocab), sw = pieces_of(p, p->vocab, p->n);
  return std::max(sq <= 1 ? 0 : round16(sq * p->n * p->dim * 4),
                  sw <= 1 ? 0 : round16(sw * p->vocab * p->dim * 4) + round16(sw * p->vocab * 4));
}

int mono_softmax_cross_entropy_gradient(const mono_softmax_ce_args* p, void* stream) {
  MONO_TRY(check(p, "mono_softmax_cross_entropy_gradient"));
  MONO_REQUIRE(p->workspace_bytes >= mono_softmax_cross_entropy_gradient_workspace(p),
               "mono_softmax_cross_entropy_gradient: workspace of %lld bytes is too small",
               (long long)p->workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  const bool half = p->dtype == MONO_ROW_BF16;
  Args a = base_args(p);
  if (p->grad_query && p->n) {
    a.nsplit = pieces_of(p, p->n, p->vocab);
    a.part = a.nsplit > 1 ? (float*)p->workspace : nullptr;
    MONO_TRY(launch<kDq>(p->dtype, a, tiles_of(p, p->n), st));
    if (a.part) {
      const int grid = grid_for(p->n * ((p->dim + 3) / 4), 256);
      if (half) k_ce_dq_join<bf16><<<grid, 256, 0, st>>>(a);
      else k_ce_dq_join<float><<<grid, 256, 0, st>>>(a);
      MONO_HIP(hipGetLastError());
    }
  }
  if (p->grad_rows || p->grad_bias) {
    a.nsplit = pieces_of(p, p->vocab, p->n);
    const int64_t total = p->vocab * p->dim;
    a.part = (float*)p->workspace;
    a.part2 = (float*)((char*)p->workspace + round16((int64_t)a.nsplit * total * 4));
    MONO_TRY(launch<kDw>(p->dtype, a, tiles_of(p, p->vocab), st));
    if (a.nsplit > 1) {
      if (p->grad_rows && half) MONO_TRY(sum_parts(a.part, a.nsplit, total, (bf16*)p->grad_rows, st));
      if (p->grad_rows && !half) MONO_TRY(sum_parts(a.part, a.nsplit, total, (float*)p->grad_rows, st));
      if (p->grad_bias) MONO_TRY(sum_parts(a.part2, a.nsplit, p->vocab, p->grad_bias, st));
    }
  }
  return 0;
}
}
