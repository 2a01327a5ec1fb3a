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
  float *part, *part2;         // forward: maximum and sum of every piece
  float *q_part, *w_part, *b_part;  // backward: partial gradients of every piece
  int n, v, D;
  int nsplit, q_split, w_split;     // pieces of the streamed rows: forward, and the gradient's two halves
  int q_tiles, w_tiles;
  float scale, scale2;
  int vec_q, vec_w, vec_o;
};

template <typename T, int DP>
struct Tile {
  static constexpr int BN = DP * sizeof(T) <= 256 ? 64 : 32, NR = BN / 32;
};

// A finite bias below kFloor counts as kFloor beside other candidates: its weight is 0 either way, but on a tile of
// nothing else the exponent's base, the rounded product of maximum and scale, would be off by more than an
// exponential holds, and infinite for the type's lowest value.
constexpr float kFloor = -1e7f;
__device__ inline float floored(float bias) { return bias < kFloor && bias != neg_inf() ? kFloor : bias; }

constexpr uint32_t kMinusInf = 0xff800000u, kPlusInf = 0x7f800000u;
__device__ inline void range_of(int n, int nsplit, int split, int BN, int* beg, int* end) {
  const int chunk = ((n + nsplit - 1) / nsplit + BN - 1) / BN * BN;
  *beg = (int)min((int64_t)n, (int64_t)split * chunk);
  *end = (int)min((int64_t)n, (int64_t)*beg + chunk);
}

// ---- forward: running maximum and sum of a tile of queries over one piece of the vocabulary ----
// loss_i = log(1 + x_i), x_i = sum over v other than the label of exp(l_iv - l_i,label), and 1 - p_label =
// x / (1 + x): the label is left out of the sum where its tile comes by, so that loss and gradient of a likely label
// are made from the others' small sum and not as the difference of two numbers near each other. (1000 candidates of
// 64 elements, p_label 0.984: dquery rows 1.6e-3 off in the median for bf16 and 4.5e-7 for fp32, the loss 4e-7; with
// p - 1 from the stored log-sum and the label's row taken off a sum of rounded weights 5e-2, 4e-5 and 6e-5.)
// A tile of 128 or (bf16 rows of 64 elements or less: two column
// tiles a wave, half the LDS reads of a product) 256 queries stays in registers, the candidates stream.
// Bound by the vector unit: an exponential, a multiply-add, a sum and half a maximum for each logit.
// 4096 queries against 1000003 rows of 64 bf16: 770 us, 5.3e12 logits a second, the vector unit at work 85% of the
// time; 8192 against 16385 rows of 64 floats: 111 us.
template <typename T, int DP, int NC>
__global__ __launch_bounds__(256, DP <= 128 || sizeof(T) == 2 ? 2 : 1) void k_ce_fwd(Args a) {
  constexpr int BM = NC * 128, BN = Tile<T, DP>::BN, NR = Tile<T, DP>::NR;
  typedef Stage<T, DP, BN, 256> St;
  typedef Mma<T, DP, St::PLANE> M;
  __shared__ __align__(16) bf16 lw[St::LDS];
  __shared__ __align__(16) float lb[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int col[NC], label[NC];
  typename M::Frag qf[NC][M::KF];
  float m[NC], l[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = blockIdx.x * BM + (wave * NC + c) * 32 + (lane & 31);
    const bool ok = col[c] < a.n;
    M::load_cols(qf[c], (const T*)a.q + (int64_t)(ok ? col[c] : 0) * a.qs, ok, a.D, a.vec_q, lane);
    m[c] = neg_inf();
    l[c] = 0.f;
    const int64_t known = ok ? a.labels[col[c]] : -1;
    label[c] = known >= 0 && known < a.v ? (int)known : -1;
  }
  int vbeg, vend;
  range_of(a.v, a.nsplit, blockIdx.y, BN, &vbeg, &vend);
  St st;
  float eb = 0.f;
  const float inv_scale = 1.f / a.scale;
  const Rows<T> wr = {(const T*)a.w, a.ws, a.D, a.vec_w != 0};
  auto fetch = [&](int y0) {
    st.load(wr, y0, vend, tid, a.bias, [&](int row) { return __float_as_uint(a.bias[row]); });
    if (tid < BN) {
      eb = y0 + tid < vend ? 0.f : neg_inf();
      if (a.bias && y0 + tid < vend) eb = a.bias[y0 + tid];
    }
  };
  if (vbeg < vend) fetch(vbeg);
  for (int y0 = vbeg; y0 < vend; y0 += BN) {
    __syncthreads();
    st.store(lw, tid, a.bias, kMinusInf);
    if (tid < BN) lb[tid] = floored(eb) * inv_scale;  // what a candidate's products start from, in units of scale
    __syncthreads();
    if (y0 + BN < vend) fetch(y0 + BN);
    uint32_t near = ~0u;  // (a label in front of the tile, or none, is far behind it as an unsigned number)
#pragma unroll
    for (int c = 0; c < NC; ++c) near = min(near, (uint32_t)(label[c] - y0));
    const bool hits = __any(near < BN);
    f16v s[NR][NC];
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) {
      if (a.bias || y0 + BN > vend) M::template scores<NC>(lw, rt, qf, s[rt], by_rows(lb + 32 * rt, lane), lane);
      else M::template scores<NC>(lw, rt, qf, s[rt], all_of(0.f), lane);
      if (hits) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int at = label[c] - y0 - 32 * rt - 4 * (lane >> 5);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (at == 8 * (r >> 2) + (r & 3)) s[rt][c][r] = neg_inf();
        }
      }
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

// One wave per query: joins the pieces of the vocabulary and the label, whose logit it makes. In units of log 2
// the others' sum is base + log2 z and the label's logit base + d.
template <typename T>
__global__ __launch_bounds__(256) void k_ce_loss(Args a) {
  const int lane = threadIdx.x & 63;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < a.n; i += (int64_t)gridDim.x * 4) {
    float m = neg_inf();
    for (int s = lane; s < a.nsplit; s += 64) m = fmaxf(m, a.part[(int64_t)s * a.n + i]);
#pragma unroll
    for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    float base = m == neg_inf() ? 0.f : m;
    float z = 0.f;
    for (int s = lane; s < a.nsplit; s += 64)
      z += a.part2[(int64_t)s * a.n + i] * exp2_hw(a.part[(int64_t)s * a.n + i] - base);
#pragma unroll
    for (int x = 32; x; x >>= 1) z += __shfl_xor(z, x);
    const int64_t label = a.labels[i];
    const bool known = label >= 0 && label < a.v;
    float hit = 0.f;
    if (known)
      for (int d = lane; d < a.D; d += 64)
        hit = fmaf((float)((const T*)a.q)[i * a.qs + d], (float)((const T*)a.w)[label * a.ws + d], hit);
#pragma unroll
    for (int x = 32; x; x >>= 1) hit += __shfl_xor(hit, x);
    if (lane == 0) {
      const float b = known && a.bias ? a.bias[label] : 0.f;
      float loss = label == -1 ? 0.f : __builtin_nanf(""), lse = __builtin_inff(), miss = 0.f;
      if (b == neg_inf()) {
        loss = __builtin_inff();
      } else if (known) {
        hit = fmaf(hit, a.scale2, floored(b) * kLog2e);
        if (m == neg_inf()) base = hit;  // (there are no others)
        const float d = hit - base, x = z * exp2_hw(-d);
        if (d > -64.f) {
          loss = log1pf(x);
          miss = x / (1.f + x);
        } else {  // (the 1 is less than a rounding of x, which may be beyond the largest number)
          loss = (__log2f(z) - d) * kLn2 + (floored(b) - b);
          miss = x == x ? 1.f : x;
        }
        lse = d > 0.f ? hit + __log2f(1.f + x) : base + __log2f(z + exp2_hw(d));
      }
      a.loss[i] = loss;
      a.lse[i] = lse;
      a.lse[a.n + i] = miss;
    }
  }
}

// ---- backward ------------------------------------------------------------------------------
// dquery_i = scale g_i (sum over v other than the label of p_iv w_v - (1 - p_label) w_label): g and the label's row
// are taken in behind the loop, in 32 bits, so that the products see nothing but the others' probabilities.
template <typename T>
__device__ inline f4 minus_label(const Args& a, int i, int d0, f4 t) {
  const float lse = a.lse[i];
  if (lse == __builtin_inff()) return f4{0.f, 0.f, 0.f, 0.f};
  const float g = a.grad[i] * a.scale, miss = a.lse[a.n + (int64_t)i];
  const T* w = (const T*)a.w + a.labels[i] * a.ws;
#pragma unroll
  for (int r = 0; r < 4; ++r) t[r] = d0 + r < a.D ? g * (t[r] - miss * (float)w[d0 + r]) : 0.f;
  return t;
}

template <typename T, int DP, int NC>
__device__ inline void query_half(const Args& a, int tile, int piece, bf16* lw, float* lb) {
  constexpr int BM = NC * 128, BN = Tile<T, DP>::BN, NR = Tile<T, DP>::NR;
  typedef Stage<T, DP, BN, 256> St;
  typedef Mma<T, DP, St::PLANE> M;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int col[NC];
  typename M::Frag qf[NC][M::KF];
  float lse[NC];
  int label[NC];
  f16v acc[M::NDT][NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = tile * BM + (wave * NC + c) * 32 + (lane & 31);
    const bool ok = col[c] < a.n;
    M::load_cols(qf[c], (const T*)a.q + (int64_t)(ok ? col[c] : 0) * a.qs, ok, a.D, a.vec_q, lane);
    lse[c] = ok ? a.lse[col[c]] : __builtin_inff();
    label[c] = lse[c] == __builtin_inff() ? -1 : (int)a.labels[col[c]];
#pragma unroll
    for (int d = 0; d < M::NDT; ++d) acc[d][c] = all_of(0.f);
  }
  int vbeg, vend;
  range_of(a.v, a.q_split, piece, BN, &vbeg, &vend);
  St st;
  float eb = 0.f;
  const float inv_scale = 1.f / a.scale;
  const Rows<T> wr = {(const T*)a.w, a.ws, a.D, a.vec_w != 0};
  auto fetch = [&](int y0) {
    st.load(wr, y0, vend, tid, a.bias, [&](int row) { return __float_as_uint(a.bias[row]); });
    if (tid < BN) {
      eb = y0 + tid < vend ? 0.f : neg_inf();
      if (a.bias && y0 + tid < vend) eb = a.bias[y0 + tid];
    }
  };
  if (vbeg < vend) fetch(vbeg);
  for (int y0 = vbeg; y0 < vend; y0 += BN) {
    __syncthreads();
    st.store(lw, tid, a.bias, kMinusInf);
    if (tid < BN) lb[tid] = floored(eb) * inv_scale;  // what a candidate's products start from, in units of scale
    __syncthreads();
    if (y0 + BN < vend) fetch(y0 + BN);
    uint32_t near = ~0u;  // (a label in front of the tile, or none, is far behind it as an unsigned number)
#pragma unroll
    for (int c = 0; c < NC; ++c) near = min(near, (uint32_t)(label[c] - y0));
    const bool hits = __any(near < BN);
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) {
      f16v s[NC];
      if (a.bias || y0 + BN > vend) M::template scores<NC>(lw, rt, qf, s, by_rows(lb + 32 * rt, lane), lane);
      else M::template scores<NC>(lw, rt, qf, s, all_of(0.f), lane);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[c][r] = exp2_hw(fmaf(s[c][r], a.scale2, -lse[c]));
      if (hits) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int at = label[c] - y0 - 32 * rt - 4 * (lane >> 5);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (at == 8 * (r >> 2) + (r & 3)) s[c][r] = 0.f;
        }
      }
      M::template accumulate<NC>(lw, rt, s, acc, lane);
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (col[c] >= a.n) continue;
    if (a.q_split > 1) {
      store_col(a.q_part + ((int64_t)piece * a.n + col[c]) * a.D, a.D, acc, c, 1.f, a.vec_o, lane);
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

// drows_v = scale sum_i g_i (p_iv - [v = label_i]) query_i, dbias_v the same without scale and query:
// a tile of candidates keeps its sums while all queries stream by. The label's weight is the forward's
// 1 - p, and rare: one ballot per tile of queries says whether any label falls into the candidates of the workgroup.
template <typename T, int DP, int NC>
__device__ inline void rows_half(const Args& a, int tile, int piece, bf16* lq, float* ll, float* lg, float* lm, int* lab) {
  constexpr int BM = NC * 128, BN = Tile<T, DP>::BN, NR = Tile<T, DP>::NR;
  typedef Stage<T, DP, BN, 256> St;
  typedef Mma<T, DP, St::PLANE> M;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int v0 = tile * BM;
  int col[NC];
  typename M::Frag wf[NC][M::KF];
  float b2[NC], sb[NC];
  f16v acc[M::NDT][NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = v0 + (wave * NC + c) * 32 + (lane & 31);
    const bool ok = col[c] < a.v;
    b2[c] = !ok ? neg_inf() : a.bias ? floored(a.bias[col[c]]) * kLog2e : 0.f;
    M::load_cols(wf[c], (const T*)a.w + (int64_t)(ok ? col[c] : 0) * a.ws, b2[c] != neg_inf(), a.D, a.vec_w, lane);
    sb[c] = 0.f;
#pragma unroll
    for (int d = 0; d < M::NDT; ++d) acc[d][c] = all_of(0.f);
  }
  int nbeg, nend;
  range_of(a.n, a.w_split, piece, BN, &nbeg, &nend);
  St st;
  const Rows<T> qr = {(const T*)a.q, a.qs, a.D, a.vec_q != 0};
  const float inv_scale2 = 1.f / a.scale2;
  float el = 0.f, eg = 0.f, em = 0.f;
  int lb = -1;
  auto fetch = [&](int y0) {
    st.load(qr, y0, nend, tid, true, [&](int row) { return __float_as_uint(a.lse[row]); });
    if (tid < BN) {
      el = __builtin_inff();
      if (y0 + tid < nend) {
        el = a.lse[y0 + tid];
        em = a.lse[a.n + (int64_t)(y0 + tid)];
        eg = a.grad[y0 + tid];
        lb = (int)a.labels[y0 + tid];
      }
    }
  };
  if (nbeg < nend) fetch(nbeg);
  for (int y0 = nbeg; y0 < nend; y0 += BN) {
    __syncthreads();
    st.store(lq, tid, true, kPlusInf);
    if (tid < BN) {
      const bool live = el != __builtin_inff();
      ll[tid] = -el * inv_scale2;
      lg[tid] = live ? eg : 0.f;
      lm[tid] = -em;
      lab[tid] = live ? lb : -1;
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
          const int row = 32 * rt + tile_row(r, lane), label = lab[row];
          const float weight = lm[row];
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (label == col[c]) s[c][r] = weight;
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
    const int64_t row = (a.w_split > 1 ? (int64_t)piece * a.v : 0) + col[c];
    if (a.db && lane < 32) (a.w_split > 1 ? a.b_part : a.db)[row] = b;
    if (!a.dw) continue;
    if (a.w_split > 1) store_col(a.w_part + row * a.D, a.D, acc, c, a.scale, a.vec_o, lane);
    else store_col((T*)a.dw + row * a.D, a.D, acc, c, a.scale, a.vec_o, lane);
  }
}

// Both halves of the gradient in one launch: they share nothing, the queries' half first. 2.15 ms for 4096
// queries against 1000003 rows of 64 bf16, 0.98 PFLOP/s of executed products where a library matrix product
// of 8192 reaches 1.13: with operands that are not random but zeros the same loop takes half the time, and the clock
// falls to 1.75 GHz, so it is the card's power that bounds it. 410 us for 8192 against 16385 rows of 64 floats.
// (Rows of 32 elements or less: three waves a SIMD, for which pieces_of cuts; 169 registers without the bound.)
template <typename T, int DP, int NC>
__global__ __launch_bounds__(256, DP <= 32 ? 3 : DP * sizeof(T) <= 256 ? 2 : 1) void k_ce_bwd(Args a) {
  constexpr int BN = Tile<T, DP>::BN;
  __shared__ __align__(16) bf16 rows[Stage<T, DP, BN, 256>::LDS];
  __shared__ __align__(16) float first[BN], second[BN], third[BN];
  __shared__ __align__(16) int labels[BN];
  const int of_queries = a.q_tiles * a.q_split, i = blockIdx.x - of_queries;
  if (i < 0) query_half<T, DP, NC>(a, blockIdx.x % a.q_tiles, blockIdx.x / a.q_tiles, rows, first);
  else rows_half<T, DP, NC>(a, i % a.w_tiles, i / a.w_tiles, rows, first, second, third, labels);
}

// four elements from `at` on of the pieces' partial sums, first to last; several pieces' loads in flight
__device__ inline f4 sum_parts(const float* part, int n_part, int64_t total, int64_t at, int n, bool vec) {
  f4 t = {0.f, 0.f, 0.f, 0.f};
  if (vec) {
#pragma unroll 8
    for (int s = 0; s < n_part; ++s) t += *(const f4*)(part + (int64_t)s * total + at);
  } else {
    for (int s = 0; s < n_part; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < n) t[r] += part[(int64_t)s * total + at + r];
  }
  return t;
}
// what of the gradient came in pieces: dquery and drows by four elements of a row, dbias by candidates
template <typename T>
__global__ __launch_bounds__(256) void k_ce_join(Args a) {
  const int per = (a.D + 3) / 4;
  const bool vec = a.D % 4 == 0;
  const int64_t nq = a.dq && a.q_split > 1 ? (int64_t)a.n * per : 0;
  const int64_t nw = a.dw && a.w_split > 1 ? (int64_t)a.v * per : 0;
  const int64_t nb = a.db && a.w_split > 1 ? a.v : 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nq + nw + nb; i += (int64_t)gridDim.x * 256) {
    if (i < nq) {
      const int row = (int)(i / per), d0 = (int)(i % per) * 4;
      const f4 t = sum_parts(a.q_part, a.q_split, (int64_t)a.n * a.D, (int64_t)row * a.D + d0, a.D - d0, vec);
      store4((T*)a.dq + (int64_t)row * a.D, d0, a.D, minus_label<T>(a, row, d0, t), a.vec_o);
    } else if (i < nq + nw) {
      const int row = (int)((i - nq) / per), d0 = (int)((i - nq) % per) * 4;
      const f4 t = sum_parts(a.w_part, a.w_split, (int64_t)a.v * a.D, (int64_t)row * a.D + d0, a.D - d0, vec);
      store4((T*)a.dw + (int64_t)row * a.D, d0, a.D, t, a.vec_o);
    } else {
      a.db[i - nq - nw] = sum_parts(a.b_part, a.w_split, a.v, i - nq - nw, 1, false)[0];
    }
  }
}

// ---- host ----------------------------------------------------------------------------------
int cols_of(const mono_softmax_ce_args* p) {
  return p->dtype == MONO_ROW_BF16 && p->dim <= 64 ? 2 : 1;
}
int64_t tiles_of(const mono_softmax_ce_args* p, int64_t kept) {
  const int bm = 128 * cols_of(p);
  return (kept + bm - 1) / bm;
}
// Few tiles of kept rows: the streamed rows are cut into pieces of 64 or more, as many as make `rounds`
// rounds of the workgroups that the card holds at once (with 1024 workgroups where it holds 768 the last
// 256 run alone: 138 us instead of 124 for 8192 queries against 16385 rows of 64 floats). The forward's
// partial results are two numbers a query, so it takes several rounds; the backward's are whole rows, so
// each of its halves takes one.
int pieces_of(const mono_softmax_ce_args* p, int64_t kept, int64_t streamed, int rounds) {
  const int row = p->dim * (p->dtype == MONO_ROW_BF16 ? 2 : 4);
  const int64_t want = 256 * rounds * (row > 256 ? 1 : cols_of(p) == 2 && p->dim > 32 ? 2 : 3);
  const int64_t tiles = std::max<int64_t>(1, tiles_of(p, kept));
  return (int)std::max<int64_t>(1, std::min<int64_t>(want / tiles, streamed / 64));
}
int fwd_pieces(const mono_softmax_ce_args* p) { return pieces_of(p, p->n, p->vocab, 4); }
int query_pieces(const mono_softmax_ce_args* p) { return pieces_of(p, p->n, p->vocab, 1); }
int rows_pieces(const mono_softmax_ce_args* p) { return pieces_of(p, p->vocab, p->n, 1); }

int check(const mono_softmax_ce_args* p, const char* who) {
  MONO_REQUIRE(p != nullptr, "%s: args is NULL", who);
  MONO_REQUIRE(p->dtype == MONO_ROW_FP32 || p->dtype == MONO_ROW_BF16, "%s: unknown row type %d", who, p->dtype);
  MONO_REQUIRE(p->dim >= 1 && p->dim <= 256, "%s: dim must be in [1, 256], got %d", who, p->dim);
  MONO_REQUIRE(p->scale >= 1e-20f && p->scale <= 1e20f, "%s: scale must be in [1e-20, 1e20], got %g", who,
               (double)p->scale);
  MONO_REQUIRE(p->n >= 0 && p->vocab >= 1 && p->n < (1LL << 26) && p->vocab < (1LL << 31) - 65536,
               "%s: %lld queries and %lld rows are out of range", who, (long long)p->n, (long long)p->vocab);
  MONO_REQUIRE(((uintptr_t)p->workspace & 15) == 0, "%s: workspace must be 16-byte aligned", who);
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

// a gradient's launch has a workgroup for every 128 candidates or fewer beside the queries' ones, of 256 threads each:
// fewer than 2^32 threads
int check_grad(const mono_softmax_ce_args* p, const char* who) {
  MONO_TRY(check(p, who));
  MONO_REQUIRE((!p->grad_rows && !p->grad_bias) || p->vocab < (1LL << 31) - (1LL << 27),
               "%s: the gradient of %lld rows is out of range", who, (long long)p->vocab);
  return 0;
}

enum Which { kFwd, kBwd };
template <int W, typename T, int DP, int NC>
int launch1(const Args& a, hipStream_t st) {
  if (W == kFwd) {
    k_ce_fwd<T, DP, NC><<<dim3((unsigned)a.q_tiles, (unsigned)a.nsplit), 256, 0, st>>>(a);
  } else {
    const int64_t wgs = (int64_t)a.q_tiles * a.q_split + (int64_t)a.w_tiles * a.w_split;
    k_ce_bwd<T, DP, NC><<<(unsigned)wgs, 256, 0, st>>>(a);
  }
  MONO_HIP(hipGetLastError());
  return 0;
}
template <int W>
int launch(int dtype, const Args& a, hipStream_t st) {
  if (dtype == MONO_ROW_BF16) {
    if (a.D <= 16) return launch1<W, bf16, 16, 2>(a, st);
    if (a.D <= 32) return launch1<W, bf16, 32, 2>(a, st);
    if (a.D <= 64) return launch1<W, bf16, 64, 2>(a, st);
    if (a.D <= 128) return launch1<W, bf16, 128, 1>(a, st);
    return launch1<W, bf16, 256, 1>(a, st);
  }
  if (a.D <= 16) return launch1<W, float, 16, 1>(a, st);
  if (a.D <= 32) return launch1<W, float, 32, 1>(a, st);
  if (a.D <= 64) return launch1<W, float, 64, 1>(a, st);
  if (a.D <= 128) return launch1<W, float, 128, 1>(a, st);
  return launch1<W, float, 256, 1>(a, st);
}
int64_t round16(int64_t b) { return (b + 15) & ~(int64_t)15; }
}  // namespace
}  // namespace mono

extern "C" {
using namespace mono;

int64_t mono_softmax_cross_entropy_workspace(const mono_softmax_ce_args* p) {
  if (check(p, "mono_softmax_cross_entropy_workspace")) return -1;
  return 2 * round16((int64_t)fwd_pieces(p) * p->n * 4);
}

int mono_softmax_cross_entropy(const mono_softmax_ce_args* p, void* stream) {
  MONO_TRY(check(p, "mono_softmax_cross_entropy"));
  if (p->n == 0) return 0;
  MONO_REQUIRE(p->query && p->rows && p->labels && p->loss && p->lse,
               "mono_softmax_cross_entropy: an array is NULL");
  MONO_REQUIRE(p->workspace_bytes >= mono_softmax_cross_entropy_workspace(p),
               "mono_softmax_cross_entropy: workspace of %lld bytes is too small", (long long)p->workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  Args a = base_args(p);
  a.nsplit = fwd_pieces(p);
  a.q_tiles = (int)tiles_of(p, p->n);
  a.part = (float*)p->workspace;
  a.part2 = (float*)((char*)p->workspace + round16((int64_t)a.nsplit * p->n * 4));
  MONO_TRY(launch<kFwd>(p->dtype, a, st));
  const int grid = grid_for(p->n, 4, 1 << 20);
  if (p->dtype == MONO_ROW_BF16) k_ce_loss<bf16><<<grid, 256, 0, st>>>(a);
  else k_ce_loss<float><<<grid, 256, 0, st>>>(a);
  MONO_HIP(hipGetLastError());
  return 0;
}

namespace {
// where the partial gradients lie in the workspace; returns its bytes
int64_t place_parts(const mono_softmax_ce_args* p, Args* a) {
  const bool rows = p->grad_rows || p->grad_bias;
  a->q_split = p->grad_query ? query_pieces(p) : 1;
  a->w_split = rows ? rows_pieces(p) : 1;
  a->q_tiles = p->grad_query ? (int)tiles_of(p, p->n) : 0;
  a->w_tiles = rows ? (int)tiles_of(p, p->vocab) : 0;
  int64_t at = 0;
  const auto take = [&](int n_part, int64_t each) {
    float* to = (float*)((char*)p->workspace + at);
    if (n_part > 1) at += round16(n_part * each * 4);
    return to;
  };
  a->q_part = take(a->q_split, p->n * p->dim);
  a->w_part = take(p->grad_rows ? a->w_split : 1, p->vocab * p->dim);
  a->b_part = take(p->grad_bias ? a->w_split : 1, p->vocab);
  return at;
}
}  // namespace

int64_t mono_softmax_cross_entropy_gradient_workspace(const mono_softmax_ce_args* p) {
  if (check_grad(p, "mono_softmax_cross_entropy_gradient_workspace")) return -1;
  Args a;
  return place_parts(p, &a);
}

int mono_softmax_cross_entropy_gradient(const mono_softmax_ce_args* p, void* stream) {
  MONO_TRY(check_grad(p, "mono_softmax_cross_entropy_gradient"));
  Args a = base_args(p);
  MONO_REQUIRE(p->rows && (p->n == 0 || (p->query && p->labels && p->lse && p->grad_loss)),
               "mono_softmax_cross_entropy_gradient: an array is NULL");
  MONO_REQUIRE(p->workspace_bytes >= place_parts(p, &a),
               "mono_softmax_cross_entropy_gradient: workspace of %lld bytes is too small",
               (long long)p->workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  if (a.q_tiles + a.w_tiles == 0) return 0;
  MONO_TRY(launch<kBwd>(p->dtype, a, st));
  if (a.q_split > 1 || a.w_split > 1) {
    const int64_t per = (p->dim + 3) / 4;
    const int grid = grid_for((a.q_split > 1 ? p->n * per : 0) + (a.w_split > 1 ? p->vocab * (per + 1) : 0), 256);
    if (p->dtype == MONO_ROW_BF16) k_ce_join<bf16><<<grid, 256, 0, st>>>(a);
    else k_ce_join<float><<<grid, 256, 0, st>>>(a);
    MONO_HIP(hipGetLastError());
  }
  return 0;
}
}
