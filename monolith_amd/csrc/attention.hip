// attention.hip — attention over ragged embedding rows: forward, backward, and the form whose
// batch shares a prefix. The tile scheme is described in seq_dev.h.
//
// The query heads of one key head lie side by side as columns of a tile ("virtual rows" token * G +
// head), so a group's keys are read once for all of its heads and a single token still fills part of
// a tile. Which sequence a workgroup's tile belongs to is found from the splits on the device, by
// the rule that sequence b's tiles start at floor(start_b / BM) + b: that leaves every sequence room
// for ceil(length / BM) tiles, needs no pass over the splits and no copy of them to the host.
#include <algorithm>
#include <type_traits>

#include "mono_common.h"
#include "seq_dev.h"

namespace mono {
namespace {
using namespace seq;

enum Mode { kSplits = 0, kOnePerSeq = 1, kWhole = 2 };

struct Args {
  const void *q, *k, *v, *go, *o;
  int64_t qs, qh, ks, kh, vs, vh, gs, gh;
  void *out, *rest, *dq, *dk, *dv;
  float *lse, *delta;
  float *part, *part2, *part_lse;  // split partials
  const int64_t *qsp, *ksp;
  const uint8_t* mask;
  int B, nq, nk, H, Hkv, G, D, qmode, kmode, causal, shared;
  int qbatch;                      // kWhole with query splits: their sequences; other queries see nothing
  int nsplit, slot0;
  int chunk;                       // pooled rows: keys of a wave, 0 = a split of a sequence's keys
  float scale, scale2;
  int vec_q, vec_k, vec_v, vec_g, vec_o;
};

struct Seg {
  int lo, n, b;  // first row, rows, sequence (-1: rows of no sequence)
};

__device__ inline int split_at(const int64_t* sp, int i, int n) {
  const int64_t s = sp[i];
  return s < 0 ? 0 : s > n ? n : (int)s;
}

__device__ inline Seg segment(const int64_t* sp, int mode, int b, int n) {
  if (mode == kWhole) return {0, n, b};
  if (mode == kOnePerSeq) return {b, 1, b};
  const int lo = split_at(sp, b, n), hi = split_at(sp, b + 1, n);
  return {lo, hi > lo ? hi - lo : 0, b};
}

// The sequence of tile `tile` (BM virtual rows each, G to a row) and the tile's place in it. Rows in
// front of the first split and behind the last count as two more sequences.
__device__ inline Seg find_tile(const int64_t* sp, int mode, int B, int n, int G, int BM, int tile,
                                int* local) {
  if (mode == kWhole) {
    *local = tile;
    return {0, n, 0};
  }
  if (mode == kOnePerSeq) {
    const int per = (G + BM - 1) / BM;
    *local = tile % per;
    return {tile / per, 1, tile / per};
  }
  // the last of segments 0 .. B + 1 (segment i starts at start(i)) whose tiles start at or before this
  // one, 64 candidates at a time: every step is one load's latency at the head of each workgroup
  int lo = 0, len = B + 2;
  const int lane = threadIdx.x & 63;
  while (len > 1) {
    const int step = (len + 63) / 64, i = lo + lane * step;
    bool at = false;
    if (i < lo + len) at = i == 0 || ((int64_t)split_at(sp, i - 1, n) * G) / BM + i <= tile;
    const uint64_t found = __ballot(at);
    const int last = found ? 63 - __builtin_clzll(found) : 0;
    len = min(step, len - last * step);
    lo += last * step;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int start = lo == 0 ? 0 : split_at(sp, lo - 1, n);
  const int end = lo == B + 1 ? n : split_at(sp, lo, n);
  *local = tile - (int)(((int64_t)start * G) / BM) - lo;
  return {start, end > start ? end - start : 0, lo == 0 || lo == B + 1 ? -1 : lo - 1};
}
int64_t tiles_for(int mode, int64_t B, int64_t n, int64_t G, int BM) {
  if (mode == kWhole) return (n * G + BM - 1) / BM;
  if (mode == kOnePerSeq) return B * ((G + BM - 1) / BM);
  return n * G / BM + B + 2;
}

// rows of a streamed tile: 64 where one takes the registers of 64 bytes a thread or less on its way to LDS
// (the forward, which keeps one product less, also for bf16 rows of 128)
template <typename T, int DP, int NW, bool FWD = false>
struct Tile {
  static constexpr int BN = NW > 1 && DP * sizeof(T) <= (FWD && sizeof(T) == 2 ? 256 : 128) ? 64 : 32, NR = BN / 32;
};

// v where a column's key (rows y of a tile, from its row 0 on) is not below lim or not alive
__device__ inline void hide(f16v& s, int lim, const uint8_t* alive, float v, int lane) {
  lim -= 4 * (lane >> 5);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t bytes = alive ? *(const uint32_t*)(alive + 8 * q + 4 * (lane >> 5)) : 0x01010101u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (8 * q + i >= lim || !(bytes & (0xffu << (8 * i)))) s[4 * q + i] = v;
  }
}

// ---- forward -------------------------------------------------------------------------------
// out_i = sum_j p_ij v_j, p the softmax over the allowed keys, in one pass: running maximum m and sum l
// per row, the accumulators rescaled when a maximum moves. A workgroup has 128 rows (4 waves of 32) so that
// a tile of keys in LDS serves four waves; a wave skips the tiles that none of its rows sees. Bound by
// the vector unit's exponential, multiply-add, maximum and sum per logit beside 4 dim / 1024 matrix
// instructions, and by the clock that the card keeps under such a load. Dense bf16 rows, 2048 keys, 64
// elements: 610 TFLOP/s, 128 elements 800 (a library matrix product of 8192: 1133); fp32 183 (151). Ragged
// causal rows (58602 rows of 8 x 64, 112 to 2048 a sequence): 183 us, 347 TFLOP/s, and there neither unit is the
// bound: vector unit 49% of the time, matrix unit 16%. Some five tiles a workgroup, two of them on the diagonal, and
// four memory latencies before the first. (Sorting the tiles by their work changed nothing.)
template <typename T, int DP, int NC, int NW>
__global__ __launch_bounds__(NW * 64, DP * sizeof(T) <= 256 ? 2 : 1) void k_attn_fwd(Args a) {
  constexpr int BM = NC * NW * 32, BN = Tile<T, DP, NW, true>::BN, NR = Tile<T, DP, NW, true>::NR, NT = NW * 64;
  typedef Stage<T, DP, BN, NT> St;
  typedef Mma<T, DP, St::PLANE> M;
  __shared__ __align__(16) bf16 lk[St::LDS];
  __shared__ __align__(16) bf16 lv[St::LDS];
  __shared__ __align__(16) uint8_t lm[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kvh = blockIdx.x % a.Hkv, split = blockIdx.y;
  int local;
  const Seg sq = find_tile(a.qsp, a.qmode, a.B, a.nq, a.G, BM, blockIdx.x / a.Hkv, &local);
  const int64_t nrow = (int64_t)sq.n * a.G;
  int64_t r0 = (int64_t)local * BM;
  if (r0 >= nrow) return;
  if (a.causal) r0 = (nrow - 1) / BM * BM - r0;  // a sequence's last rows see the most keys: first
  Seg sk = {0, 0, -1};
  if (sq.b >= 0) sk = segment(a.ksp, a.kmode, sq.b, a.nk);
  // every column's row, and the keys it sees: [0, klim) of its sequence
  int tok[NC], head[NC], klim[NC];
  bool ok[NC];
  typename M::Frag qf[NC][M::KF];
  int kmin = sk.n, kmax = 0, tfirst = 0, tlast = a.nq;
  if (a.qmode == kWhole && a.qsp) {  // (behind the shared prefix: rows of no sequence)
    tfirst = split_at(a.qsp, 0, a.nq);
    tlast = split_at(a.qsp, a.qbatch, a.nq);
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int64_t r = r0 + (wave * NC + c) * 32 + (lane & 31);
    ok[c] = r < nrow;
    tok[c] = ok[c] ? (int)(r / a.G) : 0;
    head[c] = kvh * a.G + (ok[c] ? (int)(r % a.G) : 0);
    const bool sees = sq.lo + tok[c] >= tfirst && sq.lo + tok[c] < tlast;
    int lim = sees ? sk.n : 0;
    if (a.causal) lim = min(lim, max(0, sk.n - sq.n + tok[c] + 1));
    klim[c] = ok[c] ? lim : 0;
    if (ok[c]) kmin = min(kmin, lim), kmax = max(kmax, lim);
    M::load_cols(qf[c], (const T*)a.q + (int64_t)(sq.lo + tok[c]) * a.qs + (int64_t)head[c] * a.qh, ok[c] && sees,
                 a.D, a.vec_q, lane);
  }
#pragma unroll
  for (int x = 16; x; x >>= 1) {
    kmin = min(kmin, __shfl_xor(kmin, x));
    kmax = max(kmax, __shfl_xor(kmax, x));
  }
  int kend = sk.n;
  if (a.causal) {
    const int last = (int)((min(r0 + BM, nrow) - 1) / a.G);
    kend = min(kend, max(0, sk.n - sq.n + last + 1));
  }
  int kbeg = 0;
  if (a.nsplit > 1) {
    const int chunk = ((kend + a.nsplit - 1) / a.nsplit + BN - 1) / BN * BN;
    kbeg = min(kend, split * chunk);
    kend = min(kend, kbeg + chunk);
  }
  const Rows<T> kr = {(const T*)a.k + (int64_t)sk.lo * a.ks + (int64_t)kvh * a.kh, a.ks, a.D, a.vec_k != 0};
  const Rows<T> vr = {(const T*)a.v + (int64_t)sk.lo * a.vs + (int64_t)kvh * a.vh, a.vs, a.D, a.vec_v != 0};
  const uint8_t* mb = a.mask ? a.mask + sk.lo : nullptr;

  f16v acc[M::NDT][NC];
  float m[NC], l[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m[c] = neg_inf();
    l[c] = 0.f;
#pragma unroll
    for (int d = 0; d < M::NDT; ++d) acc[d][c] = all_of(0.f);
  }
  St stk, stv;
  uint8_t mk = 0;
  auto fetch = [&](int y0) {
    const auto word = [&](int row) { return (uint32_t)mb[row]; };
    stk.load(kr, y0, kend, tid, mb, word);
    stv.load(vr, y0, kend, tid, mb, word);
    if (mb && tid < BN) mk = y0 + tid < kend ? mb[y0 + tid] : 0;
  };
  if (kbeg < kend) fetch(kbeg);
  for (int y0 = kbeg; y0 < kend; y0 += BN) {
    __syncthreads();
    stk.store(lk, tid, mb, 0);
    stv.store(lv, tid, mb, 0);
    if (mb && tid < BN) lm[tid] = mk;
    __syncthreads();
    if (y0 + BN < kend) fetch(y0 + BN);
    if (y0 >= kmax) continue;  // (per wave: every later tile only has keys that none of its rows sees)
    f16v s[NR][NC];
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) M::template scores<NC>(lk, rt, qf, s[rt], all_of(0.f), lane);
    if (mb || y0 + BN > min(kmin, kend)) {
#pragma unroll
      for (int rt = 0; rt < NR; ++rt)
#pragma unroll
        for (int c = 0; c < NC; ++c)
          hide(s[rt][c], min(klim[c], kend) - y0 - 32 * rt, mb ? lm + 32 * rt : nullptr, neg_inf(), lane);
    }
    // m is the running maximum of the products themselves: scale > 0, so the softmax's base is m * scale
    float alpha[NC];
    bool moved = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float mx = m[c];
#pragma unroll
      for (int rt = 0; rt < NR; ++rt)
#pragma unroll
        for (int r = 0; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[rt][c][r]), s[rt][c][r + 1]);
      mx = col_max(mx);
      const float base = mx == neg_inf() ? 0.f : mx * a.scale2;
      alpha[c] = exp2_hw(fmaf(m[c], a.scale2, -base));
      moved |= mx != m[c];
      m[c] = mx;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int rt = 0; rt < NR; ++rt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = exp2_hw(fmaf(s[rt][c][r], a.scale2, -base));
          s[rt][c][r] = p;
          sum[r & 1] += p;
        }
      l[c] = fmaf(l[c], alpha[c], sum[0] + sum[1]);
    }
    if (__any(moved)) {
#pragma unroll
      for (int d = 0; d < M::NDT; ++d)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[d][c] *= alpha[c];
    }
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) M::template accumulate<NC>(lv, rt, s[rt], acc, lane);
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float lt = col_sum(l[c]);
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    const float lse = lt == 0.f ? neg_inf() : fmaf(m[c], a.scale2, __log2f(lt));
    if (!ok[c]) continue;
    const int64_t row = (int64_t)(sq.lo + tok[c]) * a.H + head[c];
    if (a.part) {
      const int64_t at = (int64_t)(a.slot0 + split) * a.nq * a.H + row;
      if (lane < 32) a.part_lse[at] = lse;
      store_col(a.part + at * a.D, a.D, acc, c, inv, a.vec_o, lane);
    } else {
      if (a.lse && lane < 32) a.lse[row] = lse;
      store_col((T*)a.out + row * a.D, a.D, acc, c, inv, a.vec_o, lane, a.rest ? (T*)a.rest + row * a.D : nullptr);
    }
  }
}

// Pooled rows in parts of `chunk` keys: only a sequence of more than one part has partial results. It has
// ceil(length / chunk) <= floor(2 length / chunk) of them, so they lie from floor(2 start / chunk) on without
// meeting the next one's.
__device__ __host__ inline int64_t pool_part(int64_t start, int chunk) { return 2 * start / chunk; }

// Where the parts of a row lie: part s at first + s * step; of() returns how many there are, 0 where the row
// is whole and written already.
struct Parts {
  int n;                // parts of a row (chunk = 0)
  int64_t rows;         // rows of a part
  const int64_t* ksp;   // chunk > 0: the parts of the pooled rows, by the splits
  int chunk, B, nk, H;
  __device__ inline int of(int64_t row, int64_t* first, int64_t* step) const {
    if (!chunk) {
      *first = row;
      *step = rows;
      return n;
    }
    const int b = (int)(row / H), lo = split_at(ksp, b, nk), hi = split_at(ksp, b + 1, nk);
    *first = pool_part(lo, chunk) * H + row % H;
    *step = H;
    return hi - lo > chunk ? (int)(((int64_t)hi - lo + chunk - 1) / chunk) : 0;
  }
};
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(const float* part, const float* part_lse, Parts parts,
                                                   int64_t rows, int D, T* out, T* rest, float* lse, int vec) {
  const int d4 = (D + 3) / 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * d4; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / d4;
    const int d0 = (int)(i % d4) * 4;
    int64_t first, step;
    const int n = parts.of(row, &first, &step);
    if (n == 0) continue;
    float m = neg_inf();
    for (int s = 0; s < n; ++s) m = fmaxf(m, part_lse[first + s * step]);
    const float base = m == neg_inf() ? 0.f : m;
    f4 t = {0.f, 0.f, 0.f, 0.f};
    float z = 0.f;
    for (int s = 0; s < n; ++s) {
      const float w = exp2_hw(part_lse[first + s * step] - base);
      const float* p = part + (first + s * step) * D + d0;
      z += w;
      if (vec) {
        t += w * *(const f4*)p;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d0 + j < D) t[j] = fmaf(w, p[j], t[j]);
      }
    }
    t *= z == 0.f ? 0.f : 1.f / z;
    store4(out + row * D, d0, D, t, vec);
    if (rest) store4(rest + row * D, d0, D, rest_of<T>(t), vec);
    if (lse && d0 == 0) lse[row] = z == 0.f ? neg_inf() : m + __log2f(z);
  }
}

// The same for many parts of few rows: a workgroup per row, its threads as groups of d4 that take every
// so many-th part. The weights come first, 1024 parts at a time, so that the parts' rows are loads that
// wait for nothing: one thread after the other through 625 parts, each behind its weight, took 30 us.
template <typename T, bool VEC>
__global__ __launch_bounds__(1024) void k_attn_join_many(const float* part, const float* part_lse, Parts parts,
                                                         int D, T* out, T* rest, float* lse) {
  __shared__ f4 sums[1024];
  __shared__ float ws[1024], red[16];
  const int tid = threadIdx.x, d4 = (D + 3) / 4, groups = 1024 / d4, group = tid / d4, d0 = tid % d4 * 4;
  const int64_t row = blockIdx.x;
  int64_t first, step;
  const int n = parts.of(row, &first, &step);
  if (n == 0) return;
  float m = neg_inf();
  for (int s = tid; s < n; s += 1024) m = fmaxf(m, part_lse[first + s * step]);
  m = over_lanes<1, 64, Max>(m);
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) m = fmaxf(m, red[i]);
  const float base = m == neg_inf() ? 0.f : m;
  f4 t = {0.f, 0.f, 0.f, 0.f};
  float z = 0.f;
  for (int s0 = 0; s0 < n; s0 += 1024) {
    const int here = min(1024, n - s0);
    __syncthreads();
    ws[tid] = tid < here ? exp2_hw(part_lse[first + (s0 + tid) * step] - base) : 0.f;
    z += ws[tid];
    __syncthreads();
    const float* p = part + (first + s0 * step) * D + d0;
    if (group < groups) {
#pragma unroll 8
      for (int s = group; s < here; s += groups) {
        if (VEC) {
          t += ws[s] * *(const f4*)(p + s * step * D);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (d0 + j < D) t[j] = fmaf(ws[s], p[s * step * D + j], t[j]);
        }
      }
    }
  }
  z = over_lanes<1, 64, Sum>(z);
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = z;
  sums[tid] = t;
  __syncthreads();
  if (group) return;
  z = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) z += red[i];
  for (int g = 1; g < groups; ++g) t += sums[g * d4 + tid];
  t *= z == 0.f ? 0.f : 1.f / z;
  store4(out + row * D, d0, D, t, VEC);
  if (rest) store4(rest + row * D, d0, D, rest_of<T>(t), VEC);
  if (lse && tid == 0) lse[row] = z == 0.f ? neg_inf() : m + __log2f(z);
}

// ---- backward ------------------------------------------------------------------------------
// dQ, then dK and dV: two passes that each make the logits again, 7 products instead of the 5 of one pass
// that adds dQ up with atomics, but every sum has one order and the result is the same from call to call.
// The same rows: 224 + 256 us, 463 and 593 TFLOP/s of executed products; 2048 keys without a mask: 660.
//
// dQ: the forward's tiles again. With p = exp2(s - lse) from the forward's statistics and
// delta = g.o, ds = p (g.v - delta), dq = scale sum ds k. Also writes delta for the pass over keys. A bf16
// result's rounding would shift delta, and with it every ds of the row the same way (gradients 2.5e-3 off
// instead of 2.4e-3, of which their own rounding is 1.7e-3): o is taken with its rest.
template <typename T, int DP, int NC, int NW>
__global__ __launch_bounds__(NW * 64, DP <= 64 || (sizeof(T) == 2 && NW > 1) ? 2 : 1) void k_attn_dq(Args a) {
  constexpr int BM = NC * NW * 32, BN = Tile<T, DP, NW>::BN, NR = Tile<T, DP, NW>::NR, NT = NW * 64;
  typedef Stage<T, DP, BN, NT> St;
  typedef Mma<T, DP, St::PLANE> M;
  __shared__ __align__(16) bf16 lk[St::LDS];
  __shared__ __align__(16) bf16 lv[St::LDS];
  __shared__ __align__(16) uint8_t lm[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kvh = blockIdx.x % a.Hkv, split = blockIdx.y;
  int local;
  const Seg sq = find_tile(a.qsp, a.qmode, a.B, a.nq, a.G, BM, blockIdx.x / a.Hkv, &local);
  const int64_t nrow = (int64_t)sq.n * a.G;
  int64_t r0 = (int64_t)local * BM;
  if (r0 >= nrow) return;
  if (a.causal) r0 = (nrow - 1) / BM * BM - r0;  // a sequence's last rows see the most keys: first
  Seg sk = {0, 0, -1};
  if (sq.b >= 0) sk = segment(a.ksp, a.kmode, sq.b, a.nk);
  int tok[NC], head[NC], klim[NC];
  bool ok[NC];
  float lse[NC], delta[NC];
  typename M::Frag qf[NC][M::KF], gf[NC][M::KF];
  int kmin = sk.n, kmax = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int64_t r = r0 + (wave * NC + c) * 32 + (lane & 31);
    ok[c] = r < nrow;
    tok[c] = ok[c] ? (int)(r / a.G) : 0;
    head[c] = kvh * a.G + (ok[c] ? (int)(r % a.G) : 0);
    int lim = sk.n;
    if (a.causal) lim = min(lim, max(0, sk.n - sq.n + tok[c] + 1));
    klim[c] = ok[c] ? lim : 0;
    if (ok[c]) kmin = min(kmin, lim), kmax = max(kmax, lim);
    const int64_t t = sq.lo + tok[c], row = t * a.H + head[c];
    M::load_cols(qf[c], (const T*)a.q + t * a.qs + (int64_t)head[c] * a.qh, ok[c], a.D, a.vec_q, lane);
    M::load_cols(gf[c], (const T*)a.go + t * a.gs + (int64_t)head[c] * a.gh, ok[c], a.D, a.vec_g, lane);
    typename M::Frag of[M::KF];
    M::load_cols(of, (const T*)a.o + row * a.D, ok[c], a.D, a.vec_o, lane);
    delta[c] = M::dot(gf[c], of);
    if (a.rest) {
      M::load_cols(of, (const T*)a.rest + row * a.D, ok[c], a.D, a.vec_o, lane);
      delta[c] += M::dot(gf[c], of);
    }
    delta[c] = col_sum(delta[c]);
    const float e = ok[c] ? a.lse[row] : neg_inf();
    lse[c] = e == neg_inf() ? __builtin_inff() : e;  // a row without keys: every weight is 0
    if (ok[c] && lane < 32 && split == 0) a.delta[row] = delta[c];
  }
#pragma unroll
  for (int x = 16; x; x >>= 1) {
    kmin = min(kmin, __shfl_xor(kmin, x));
    kmax = max(kmax, __shfl_xor(kmax, x));
  }
  int kend = sk.n;
  if (a.causal) {
    const int last = (int)((min(r0 + BM, nrow) - 1) / a.G);
    kend = min(kend, max(0, sk.n - sq.n + last + 1));
  }
  int kbeg = 0;
  if (a.nsplit > 1) {
    const int chunk = ((kend + a.nsplit - 1) / a.nsplit + BN - 1) / BN * BN;
    kbeg = min(kend, split * chunk);
    kend = min(kend, kbeg + chunk);
  }
  const Rows<T> kr = {(const T*)a.k + (int64_t)sk.lo * a.ks + (int64_t)kvh * a.kh, a.ks, a.D, a.vec_k != 0};
  const Rows<T> vr = {(const T*)a.v + (int64_t)sk.lo * a.vs + (int64_t)kvh * a.vh, a.vs, a.D, a.vec_v != 0};
  const uint8_t* mb = a.mask ? a.mask + sk.lo : nullptr;
  f16v acc[M::NDT][NC];
#pragma unroll
  for (int d = 0; d < M::NDT; ++d)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[d][c] = all_of(0.f);
  St stk, stv;
  uint8_t mk = 0;
  auto fetch = [&](int y0) {
    const auto word = [&](int row) { return (uint32_t)mb[row]; };
    stk.load(kr, y0, kend, tid, mb, word);
    stv.load(vr, y0, kend, tid, mb, word);
    if (mb && tid < BN) mk = y0 + tid < kend ? mb[y0 + tid] : 0;
  };
  if (kbeg < kend) fetch(kbeg);
  for (int y0 = kbeg; y0 < kend; y0 += BN) {
    __syncthreads();
    stk.store(lk, tid, mb, 0);
    stv.store(lv, tid, mb, 0);
    if (mb && tid < BN) lm[tid] = mk;
    __syncthreads();
    if (y0 + BN < kend) fetch(y0 + BN);
    if (y0 >= kmax) continue;
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) {
      f16v s[NC], dp[NC];
      M::template scores<NC>(lk, rt, qf, s, all_of(0.f), lane);
      M::template scores<NC>(lv, rt, gf, dp, all_of(0.f), lane);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[c][r] = exp2_hw(fmaf(s[c][r], a.scale2, -lse[c])) * (dp[c][r] - delta[c]);
      if (mb || y0 + BN > min(kmin, kend)) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
          hide(s[c], min(klim[c], kend) - y0 - 32 * rt, mb ? lm + 32 * rt : nullptr, 0.f, lane);
      }
      M::template accumulate<NC>(lk, rt, s, acc, lane);
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (!ok[c]) continue;
    const int64_t row = (int64_t)(sq.lo + tok[c]) * a.H + head[c];
    if (a.part) {
      const int64_t at = (int64_t)split * a.nq * a.H + row;
      store_col(a.part + at * a.D, a.D, acc, c, a.scale, a.vec_o, lane);
    } else {
      store_col((T*)a.dq + row * a.D, a.D, acc, c, a.scale, a.vec_o, lane);
    }
  }
}

// dK, dV: a tile of keys keeps its sums while the queries of its sequence stream by, the heads of
// the group one after the other, so a shared key head's gradient is one sum in one order.
template <typename T, int DP, int NC, int NW>
__global__ __launch_bounds__(NW * 64, DP * sizeof(T) <= 128 ? 2 : 1) void k_attn_dkv(Args a) {
  constexpr int BM = NC * NW * 32, BN = Tile<T, DP, NW>::BN, NR = Tile<T, DP, NW>::NR, NT = NW * 64;
  typedef Stage<T, DP, BN, NT> St;
  typedef Mma<T, DP, St::PLANE> M;
  __shared__ __align__(16) bf16 lq[St::LDS];
  __shared__ __align__(16) bf16 lg[St::LDS];
  __shared__ __align__(16) float ll[BN], ld[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kvh = blockIdx.x % a.Hkv, split = blockIdx.y;
  int local;
  const Seg sk = find_tile(a.ksp, a.kmode, a.B, a.nk, 1, BM, blockIdx.x / a.Hkv, &local);
  const int j0 = local * BM;
  if (j0 >= sk.n) return;
  Seg sq = {0, 0, -1};
  if (sk.b >= 0) sq = segment(a.qsp, a.qmode, sk.b, a.nq);
  // every column's key, and the queries that see it: [qlim, n) of its sequence
  int qlim[NC], key[NC];
  bool ok[NC];
  typename M::Frag kf[NC][M::KF], vf[NC][M::KF];
  int qmax = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int j = j0 + (wave * NC + c) * 32 + (lane & 31);
    ok[c] = j < sk.n;
    key[c] = sk.lo + (ok[c] ? j : 0);
    const bool seen = ok[c] && (!a.mask || a.mask[key[c]]);
    qlim[c] = seen ? (a.causal ? max(0, j - (sk.n - sq.n)) : 0) : 0x7fffffff;
    if (ok[c]) qmax = max(qmax, qlim[c]);
    M::load_cols(kf[c], (const T*)a.k + (int64_t)key[c] * a.ks + (int64_t)kvh * a.kh, seen, a.D, a.vec_k, lane);
    M::load_cols(vf[c], (const T*)a.v + (int64_t)key[c] * a.vs + (int64_t)kvh * a.vh, seen, a.D, a.vec_v, lane);
  }
#pragma unroll
  for (int x = 16; x; x >>= 1) qmax = max(qmax, __shfl_xor(qmax, x));
  f16v ak[M::NDT][NC], av[M::NDT][NC];
#pragma unroll
  for (int d = 0; d < M::NDT; ++d)
#pragma unroll
    for (int c = 0; c < NC; ++c) ak[d][c] = av[d][c] = all_of(0.f);
  // tiles of queries, head after head
  const int tfirst = a.causal ? max(0, j0 - (sk.n - sq.n)) / BN : 0;
  const int nt = max(0, (sq.n + BN - 1) / BN - tfirst);
  int64_t ibeg = 0, iend = (int64_t)nt * a.G;
  if (a.nsplit > 1) {
    const int64_t chunk = (iend + a.nsplit - 1) / a.nsplit;
    ibeg = min(iend, split * chunk);
    iend = min(iend, ibeg + chunk);
  }
  // A query without keys has weights of 0, but a product with them would still carry on what its row and its
  // gradient hold, NaN say: rows of zeros then. There is none where the queries are no more than the keys and no
  // key is masked.
  const bool some_empty = a.mask || (a.causal && sq.n > sk.n);
  St stq, stg;
  float el = 0.f, ed = 0.f;
  const float inv_scale2 = 1.f / a.scale2;
  auto fetch = [&](int64_t it) {
    const auto all = [](int) { return 1u; };
    const int head = kvh * a.G + (int)(it / nt), y0 = (int)(tfirst + it % nt) * BN;
    const Rows<T> qr = {(const T*)a.q + (int64_t)sq.lo * a.qs + (int64_t)head * a.qh, a.qs, a.D, a.vec_q != 0};
    const Rows<T> gr = {(const T*)a.go + (int64_t)sq.lo * a.gs + (int64_t)head * a.gh, a.gs, a.D, a.vec_g != 0};
    stq.load(qr, y0, sq.n, tid, false, all);
    stg.load(gr, y0, sq.n, tid, false, all);
    if (tid < BN) {
      el = neg_inf();
      ed = 0.f;
      if (y0 + tid < sq.n) {
        const int64_t row = (int64_t)(sq.lo + y0 + tid) * a.H + head;
        el = a.lse[row];
        ed = a.delta[row];
      }
    }
  };
  if (ibeg < iend) fetch(ibeg);
  for (int64_t it = ibeg; it < iend; ++it) {
    __syncthreads();
    stq.store(lq, tid, false, 0);
    stg.store(lg, tid, false, 0);
    if (tid < BN) {  // a query without keys, and none: every weight is 0
      const bool empty = el == neg_inf();
      ll[tid] = empty ? neg_inf() : -el * inv_scale2;
      ld[tid] = empty ? 0.f : -ed;
    }
    __syncthreads();
    const int y0 = (int)(tfirst + it % nt) * BN;
    if (some_empty) {
      const auto empty = [&](int row) { return ll[row] == neg_inf(); };
      if (__any(y0 + (lane & (BN - 1)) < sq.n && empty(lane & (BN - 1)))) {  // (every wave finds the same)
        St::clear(lq, tid, empty);
        St::clear(lg, tid, empty);
        __syncthreads();
      }
    }
    if (it + 1 < iend) fetch(it + 1);
    const bool need = y0 < qmax;
#pragma unroll
    for (int rt = 0; rt < NR; ++rt) {
      f16v p[NC], ds[NC];
      // the rows' statistics are where the products start from: s - lse / scale and dp - delta
      M::template scores<NC>(lq, rt, kf, p, by_rows(ll + 32 * rt, lane), lane);
      M::template scores<NC>(lg, rt, vf, ds, by_rows(ld + 32 * rt, lane), lane);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) p[c][r] = exp2_hw(p[c][r] * a.scale2);
      if (need) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int lim = qlim[c] - y0 - 32 * rt - 4 * (lane >> 5);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) < lim) p[c][r] = 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) ds[c] *= p[c];
      M::template accumulate<NC>(lg, rt, p, av, lane);
      M::template accumulate<NC>(lq, rt, ds, ak, lane);
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (!ok[c]) continue;
    const int64_t row = (int64_t)key[c] * a.Hkv + kvh;
    if (a.shared)
#pragma unroll
      for (int d = 0; d < M::NDT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) ak[d][c][r] = fmaf(ak[d][c][r], a.scale, av[d][c][r]);
    const float f = a.shared ? 1.f : a.scale;
    if (a.part) {
      const int64_t at = ((int64_t)split * a.nk * a.Hkv + row) * a.D;
      store_col(a.part + at, a.D, ak, c, f, a.vec_o, lane);
      if (!a.shared) store_col(a.part2 + at, a.D, av, c, 1.f, a.vec_o, lane);
    } else {
      store_col((T*)a.dk + row * a.D, a.D, ak, c, f, a.vec_o, lane);
      if (!a.shared) store_col((T*)a.dv + row * a.D, a.D, av, c, 1.f, a.vec_o, lane);
    }
  }
}

// out = the parts' sums, first to last
template <typename T>
__global__ __launch_bounds__(256) void k_sum_parts(const float* part, Parts parts, int64_t total, int D, T* out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    int64_t first, step;
    const int n = parts.of(i / D, &first, &step);
    if (n == 0) continue;
    const float* p = part + first * D + i % D;
    float t = 0.f;
#pragma unroll 8
    for (int s = 0; s < n; ++s) t += p[s * step * D];
    out[i] = (T)t;
  }
}

// ---- one query per sequence -------------------------------------------------------------------
// A pooled row reads every key once and computes 4 D operations for it: memory bound, and a matrix tile
// would hold one column. One wave walks the keys of a sequence (or of its split): LPR lanes hold a key's
// row, 16 bytes each, so a wave takes R = 64 / LPR keys at once and U times that per turn; every group
// of LPR lanes keeps softmax statistics of its own, joined behind the loop. GT query heads of the key
// head share what is read. 16384 rows of 825261 keys x 32 floats: 36 us, 2.9 TB/s (a large read reaches 4.0);
// the next keys' loads ahead of the present ones' sums took as long (37 us, 104 registers for 54).
template <typename T>
struct Chunk {
  static constexpr int E = 16 / sizeof(T);
  float x[E];
  __device__ inline void set(u4 w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t t = w[i];
      if constexpr (sizeof(T) == 4) {
        x[i] = __uint_as_float(t);
      } else {
        x[2 * i] = __uint_as_float(t << 16);
        x[2 * i + 1] = __uint_as_float(t & 0xffff0000u);
      }
    }
  }
  __device__ inline void clear() {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = 0.f;
  }
  __device__ inline float dot(const Chunk& o) const {
    float t = x[0] * o.x[0];
#pragma unroll
    for (int i = 1; i < E; ++i) t = fmaf(x[i], o.x[i], t);
    return t;
  }
  __device__ inline void add(float w, const Chunk& o) {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = fmaf(w, o.x[i], x[i]);
  }
  template <typename O>
  __device__ inline void store(O* row, int e0, int D, bool vec, float f) const {
#pragma unroll
    for (int i = 0; i < E; i += 4)
      if (e0 + i < D) store4(row, e0 + i, D, f4{x[i] * f, x[i + 1] * f, x[i + 2] * f, x[i + 3] * f}, vec);
  }
};
template <int LPR>
__device__ inline float row_sum(float t) {
  return over_lanes<1, LPR, Sum>(t);
}

// the keys of a split
__device__ inline void split_range(int n, int nsplit, int split, int step, int* beg, int* end) {
  const int chunk = ((n + nsplit - 1) / nsplit + step - 1) / step * step;
  *beg = (int)min((int64_t)n, (int64_t)split * chunk);
  *end = (int)min((int64_t)n, (int64_t)*beg + chunk);
}

// A wave's work: a key head of a sequence, or a part of its keys. With chunk = 0 every sequence has
// nsplit equal parts, and part p of row b lies at p * n_query + b. Otherwise a part is `chunk` keys. Every
// sequence's first part is the wave of its number; the others are found by search, and few: part k > 0 of a
// sequence that starts at s is the extra e = floor(s / chunk) + k, whose first possible key e * chunk lies
// in that sequence and in no other.
struct PoolItem {
  Seg sk;
  int kvh, beg, end;
  int64_t part;  // times heads: the row of the partial results
  bool whole;    // all of the sequence's keys: no partial results
};
__device__ __host__ inline int64_t pool_items(int64_t B, int64_t Hkv, int64_t nk, int nsplit, int chunk) {
  return (chunk ? nk / chunk + 1 + B : B * nsplit) * Hkv;
}
__device__ inline PoolItem pool_item(const Args& a, int64_t item, int step) {
  PoolItem w;
  w.kvh = (int)(item % a.Hkv);
  item /= a.Hkv;
  if (a.chunk) {
    const int extras = a.nk / a.chunk + 1;
    int b = (int)(item - extras), k = 0;
    if (b < 0) {  // (the long sequences' later parts first)
      const int64_t at = item * a.chunk;
      int lo = 0, len = a.B;
      const int lane = threadIdx.x & 63;
      while (len > 1) {
        const int step64 = (len + 63) / 64, i = lo + lane * step64;
        const uint64_t found = __ballot(i < lo + len && split_at(a.ksp, i, a.nk) <= at);
        const int last = found ? 63 - __builtin_clzll(found) : 0;
        len = min(step64, len - last * step64);
        lo += last * step64;
      }
      b = __builtin_amdgcn_readfirstlane(lo);
      k = (int)item - split_at(a.ksp, b, a.nk) / a.chunk;
      if (k < 1 || a.B == 0) b = -1;
    }
    w.sk = {0, 0, -1};
    if (b >= 0) w.sk = segment(a.ksp, kSplits, b, a.nk);
    const int64_t beg = (int64_t)k * a.chunk;
    if (k > 0 && beg >= w.sk.n) w.sk.b = -1;
    w.beg = (int)min(beg, (int64_t)w.sk.n);
    w.end = (int)min(beg + a.chunk, (int64_t)w.sk.n);
    w.part = pool_part(w.sk.lo, a.chunk) + k;
    w.whole = w.sk.n <= a.chunk;
  } else {
    const int split = (int)(item % a.nsplit), b = (int)(item / a.nsplit);
    w.sk = segment(a.ksp, kSplits, b, a.nk);
    split_range(w.sk.n, a.nsplit, split, step, &w.beg, &w.end);
    w.part = (int64_t)split * a.nq + b;
    w.whole = !a.part;
  }
  return w;
}

template <typename T, int DP, int GT>
__global__ __launch_bounds__(256) void k_pool_fwd(Args a) {
  constexpr int E = 16 / sizeof(T), LPR = DP / E, R = 64 / LPR, U = sizeof(T) == 4 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= pool_items(a.B, a.Hkv, a.nk, a.nsplit, a.chunk)) return;
  const PoolItem w = pool_item(a, item, R);
  if (w.sk.b < 0) return;
  const int kvh = w.kvh, b = w.sk.b, beg = w.beg, end = w.end;
  const Seg sk = w.sk;
  const int sub = lane / LPR, e0 = lane % LPR * E;
  const T* kb = (const T*)a.k + (int64_t)sk.lo * a.ks + (int64_t)kvh * a.kh;
  const T* vb = (const T*)a.v + (int64_t)sk.lo * a.vs + (int64_t)kvh * a.vh;
  const uint8_t* mb = a.mask ? a.mask + sk.lo : nullptr;
  const bool same = a.k == a.v && a.ks == a.vs && a.kh == a.vh;
  Chunk<T> q[GT], acc[GT];
  float m[GT], l[GT];
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    const int head = kvh * a.G + g;
    q[g].set(load_chunk((const T*)a.q + (int64_t)b * a.qs + (int64_t)head * a.qh, e0, a.D, a.vec_q));
    acc[g].clear();
    m[g] = neg_inf();
    l[g] = 0.f;
  }
  for (int j0 = beg; j0 < end; j0 += R * U) {
    u4 kw[U], vw[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * R + sub;
      in[u] = j < end && (!mb || mb[j]);
      kw[u] = vw[u] = u4{0u, 0u, 0u, 0u};
      if (in[u]) {
        kw[u] = load_chunk(kb + (int64_t)j * a.ks, e0, a.D, a.vec_k);
        if (!same) vw[u] = load_chunk(vb + (int64_t)j * a.vs, e0, a.D, a.vec_v);
      }
    }
    Chunk<T> kc[U], vc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      kc[u].set(kw[u]);
      vc[u].set(same ? kw[u] : vw[u]);
    }
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float s[U], mx = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float t = row_sum<LPR>(q[g].dot(kc[u]));
        s[u] = in[u] ? t : neg_inf();
        mx = fmaxf(mx, s[u]);
      }
      const float base = mx == neg_inf() ? 0.f : mx * a.scale2;
      const float alpha = exp2_hw(fmaf(m[g], a.scale2, -base));
      m[g] = mx;
      l[g] *= alpha;
#pragma unroll
      for (int i = 0; i < E; ++i) acc[g].x[i] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = exp2_hw(fmaf(s[u], a.scale2, -base));
        l[g] += p;
        acc[g].add(p, vc[u]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    const float mx = over_lanes<LPR, 64, Max>(m[g]);
    const float base = mx == neg_inf() ? 0.f : mx * a.scale2;
    const float share = exp2_hw(fmaf(m[g], a.scale2, -base));
    const float lt = over_lanes<LPR, 64, Sum>(l[g] * share);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[g].x[i] = over_lanes<LPR, 64, Sum>(acc[g].x[i] * share);
    if (sub) continue;
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    const float lse = lt == 0.f ? neg_inf() : fmaf(mx, a.scale2, __log2f(lt));
    const int64_t row = (int64_t)b * a.H + kvh * a.G + g;
    if (!w.whole) {
      const int64_t at = (a.chunk ? 0 : (int64_t)a.slot0 * a.nq * a.H) + w.part * a.H + kvh * a.G + g;
      if (lane == 0) a.part_lse[at] = lse;
      acc[g].store(a.part + at * a.D, e0, a.D, a.vec_o, inv);
    } else {
      if (a.lse && lane == 0) a.lse[row] = lse;
      acc[g].store((T*)a.out + row * a.D, e0, a.D, a.vec_o, inv);
      if (a.rest) {
        Chunk<T> rest;
#pragma unroll
        for (int i = 0; i < E; ++i) rest.x[i] = acc[g].x[i] * inv - (float)(T)(acc[g].x[i] * inv);
        rest.store((T*)a.rest + row * a.D, e0, a.D, a.vec_o, 1.f);
      }
    }
  }
}

// The gradient in one pass over the keys: a wave that holds the query and its output's gradient makes
// a key's weight again and writes the key's and value's gradients at once, which no other row shares;
// the query's gradient is summed on the way. All GT = G heads of the key head together. The same rows:
// 52 us, 4.1 TB/s read and written.
template <typename T, int DP, int GT>
__global__ __launch_bounds__(256) void k_pool_bwd(Args a) {
  constexpr int E = 16 / sizeof(T), LPR = DP / E, R = 64 / LPR, U = 2;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t items = pool_items(a.B, a.Hkv, a.nk, a.nsplit, a.chunk);
  const int sub = lane / LPR, e0 = lane % LPR * E;
  Chunk<T> zero;
  zero.clear();
  if (item >= items) {  // the waves behind the last: rows of no sequence get zeros
    if (!a.dk) return;
    const int first = split_at(a.ksp, 0, a.nk), last = split_at(a.ksp, a.B, a.nk);
    const int64_t others = ((int64_t)first + max(0, a.nk - last)) * a.Hkv, step = ((int64_t)gridDim.x * 4 - items) * R;
    for (int64_t i = (item - items) * R + sub; i < others; i += step) {
      const int64_t at = i < (int64_t)first * a.Hkv ? i : i - (int64_t)first * a.Hkv + (int64_t)last * a.Hkv;
      zero.store((T*)a.dk + at * a.D, e0, a.D, a.vec_o, 0.f);
      if (!a.shared) zero.store((T*)a.dv + at * a.D, e0, a.D, a.vec_o, 0.f);
    }
    return;
  }
  const PoolItem w = pool_item(a, item, R);
  if (w.sk.b < 0) return;
  const int kvh = w.kvh, b = w.sk.b, beg = w.beg, end = w.end;
  const Seg sk = w.sk;
  const T* kb = (const T*)a.k + (int64_t)sk.lo * a.ks + (int64_t)kvh * a.kh;
  const T* vb = (const T*)a.v + (int64_t)sk.lo * a.vs + (int64_t)kvh * a.vh;
  const uint8_t* mb = a.mask ? a.mask + sk.lo : nullptr;
  const bool same = a.k == a.v && a.ks == a.vs && a.kh == a.vh;
  Chunk<T> q[GT], go[GT], dq[GT];
  float lse[GT], delta[GT];
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    const int head = kvh * a.G + g;
    const int64_t row = (int64_t)b * a.H + head;
    Chunk<T> o;
    q[g].set(load_chunk((const T*)a.q + (int64_t)b * a.qs + (int64_t)head * a.qh, e0, a.D, a.vec_q));
    go[g].set(load_chunk((const T*)a.go + (int64_t)b * a.gs + (int64_t)head * a.gh, e0, a.D, a.vec_g));
    o.set(load_chunk((const T*)a.o + row * a.D, e0, a.D, a.vec_o));
    delta[g] = go[g].dot(o);
    if (a.rest) {
      o.set(load_chunk((const T*)a.rest + row * a.D, e0, a.D, a.vec_o));
      delta[g] += go[g].dot(o);
    }
    delta[g] = row_sum<LPR>(delta[g]);
    const float e = a.lse[row];
    lse[g] = e == neg_inf() ? __builtin_inff() : e;
    dq[g].clear();
  }
  for (int j0 = beg; j0 < end; j0 += R * U) {
    u4 kw[U], vw[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * R + sub;
      in[u] = j < end && (!mb || mb[j]);
      kw[u] = vw[u] = u4{0u, 0u, 0u, 0u};
      if (in[u]) {
        kw[u] = load_chunk(kb + (int64_t)j * a.ks, e0, a.D, a.vec_k);
        if (!same) vw[u] = load_chunk(vb + (int64_t)j * a.vs, e0, a.D, a.vec_v);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * R + sub;
      Chunk<T> kc, vc, dk, dv;
      kc.set(kw[u]);
      vc.set(same ? kw[u] : vw[u]);
      dk.clear();
      dv.clear();
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        const float s = row_sum<LPR>(q[g].dot(kc)), dp = row_sum<LPR>(go[g].dot(vc));
        const float p = in[u] ? exp2_hw(fmaf(s, a.scale2, -lse[g])) : 0.f;
        const float ds = p * (dp - delta[g]) * a.scale;
        if (in[u]) {
          dq[g].add(ds, kc);
          dk.add(ds, q[g]);
          if (a.shared) dk.add(p, go[g]);
          else dv.add(p, go[g]);
        }
      }
      if (a.dk && j < end) {
        const int64_t at = ((int64_t)(sk.lo + j) * a.Hkv + kvh) * a.D;
        dk.store((T*)a.dk + at, e0, a.D, a.vec_o, 1.f);
        if (!a.shared) dv.store((T*)a.dv + at, e0, a.D, a.vec_o, 1.f);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < GT; ++g) {
#pragma unroll
    for (int i = 0; i < E; ++i) dq[g].x[i] = over_lanes<LPR, 64, Sum>(dq[g].x[i]);
    if (sub) continue;
    const int64_t row = (int64_t)b * a.H + kvh * a.G + g;
    if (!w.whole) {
      dq[g].store(a.part + (w.part * a.H + kvh * a.G + g) * a.D, e0, a.D, a.vec_o, 1.f);
    } else {
      dq[g].store((T*)a.dq + row * a.D, e0, a.D, a.vec_o, 1.f);
    }
  }
}

// ---- host ----------------------------------------------------------------------------------
struct Shape {
  int nc, nw, bm;
};
// Short sequences (64 rows of a key head or fewer on average) leave most of a 128-row tile empty: one
// wave with 32 columns per workgroup then. 49152 causal rows of 8 heads in sequences of random length, forward and
// with its gradient, one wave against four: bf16 of 64 elements, 32 rows on average 55 us against 106 and 316 against
// 481, 64 rows 55 against 80 and 331 against 393, 128 rows 63 against 75 and 371 against 387, 192 rows 73 against 79 and
// 413 against 402; fp32 of 32 elements 77 against 140 and 294 against 616, 81 against 103 and 307 against 459, 107
// against 106 and 387 against 464, 137 against 120 and 486 against 525. (fp32 rows of more than 32 elements: a tile's
// way to LDS alone would take a wave's registers.)
Shape shape_for(int dtype, int D, double rows_per_seq) {
  if (rows_per_seq <= 64 && (dtype == MONO_ROW_BF16 || D <= 32)) return {1, 1, 32};
  return {1, 4, 128};
}
// Few tiles are split along the streamed axis into as many workgroups as the card holds at once (a
// rest would run alone on it: prefix_lifelong took 256 us in 768 workgroups of which it holds 512), in
// pieces of 64 rows or more.
int splits_for(int64_t tiles, int nw, int D, double stream_rows) {
  const int64_t want = 256 * (nw == 1 ? 12 : D <= 32 ? 4 : D <= 64 ? 3 : 2);
  if (tiles <= 0 || tiles >= want) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want / tiles, (int64_t)(stream_rows / 64)), 256));
}

bool aligned_rows(const mono_rows& r, int dtype, int D) {
  const int e = dtype == MONO_ROW_BF16 ? 8 : 4;
  return D % e == 0 && r.row_stride % e == 0 && r.head_stride % e == 0 && ((uintptr_t)r.ptr & 15) == 0;
}

int check(const mono_attention_args* p, const char* who) {
  MONO_REQUIRE(p != nullptr, "%s: args is NULL", who);
  MONO_REQUIRE(p->dtype == MONO_ROW_FP32 || p->dtype == MONO_ROW_BF16, "%s: unknown row type %d", who, p->dtype);
  MONO_REQUIRE(p->dim >= 1 && p->dim <= 128, "%s: dim must be in [1, 128], got %d", who, p->dim);
  MONO_REQUIRE(p->heads >= 1 && p->kv_heads >= 1 && p->heads % p->kv_heads == 0,
               "%s: heads (%d) must be a positive multiple of kv_heads (%d)", who, p->heads, p->kv_heads);
  MONO_REQUIRE(p->scale >= 1e-20f && p->scale <= 1e20f, "%s: scale must be in [1e-20, 1e20], got %g", who,
               (double)p->scale);
  MONO_REQUIRE(p->batch >= 0 && p->n_query >= 0 && p->n_key >= 0 && p->n_prefix >= 0, "%s: negative size", who);
  constexpr int64_t kMost = (1LL << 31) - 65536;
  MONO_REQUIRE(p->n_query <= kMost / p->heads && p->n_key <= kMost / p->kv_heads &&
                   p->n_prefix <= kMost / p->kv_heads && p->batch <= kMost / p->kv_heads,
               "%s: more than 2^31 rows", who);
  MONO_REQUIRE(((uintptr_t)p->workspace & 15) == 0, "%s: workspace must be 16-byte aligned", who);
  MONO_REQUIRE(p->query_splits || p->n_query == p->batch,
               "%s: without query_splits there is one query per sequence (n_query %lld, batch %lld)", who,
               (long long)p->n_query, (long long)p->batch);
  return 0;
}

Args base_args(const mono_attention_args* p) {
  Args a{};
  a.q = p->query.ptr, a.qs = p->query.row_stride, a.qh = p->query.head_stride;
  a.k = p->key.ptr, a.ks = p->key.row_stride, a.kh = p->key.head_stride;
  a.v = p->value.ptr, a.vs = p->value.row_stride, a.vh = p->value.head_stride;
  a.go = p->grad_out.ptr, a.gs = p->grad_out.row_stride, a.gh = p->grad_out.head_stride;
  a.o = p->out, a.out = p->out, a.rest = p->out_rest, a.lse = p->lse;
  a.dq = p->grad_query, a.dk = p->grad_key, a.dv = p->grad_value;
  a.qsp = p->query_splits, a.ksp = p->key_splits, a.mask = p->key_mask;
  a.B = (int)p->batch, a.nq = (int)p->n_query, a.nk = (int)p->n_key;
  a.H = p->heads, a.Hkv = p->kv_heads, a.G = p->heads / p->kv_heads, a.D = p->dim;
  a.qmode = p->query_splits ? kSplits : kOnePerSeq;
  a.kmode = kSplits;
  a.causal = p->causal, a.shared = p->kv_shared;
  a.nsplit = 1;
  a.scale = p->scale, a.scale2 = p->scale * kLog2e;
  a.vec_q = aligned_rows(p->query, p->dtype, p->dim);
  a.vec_k = aligned_rows(p->key, p->dtype, p->dim);
  a.vec_v = aligned_rows(p->value, p->dtype, p->dim);
  a.vec_g = aligned_rows(p->grad_out, p->dtype, p->dim);
  a.vec_o = p->dim % (p->dtype == MONO_ROW_BF16 ? 8 : 4) == 0 && (((uintptr_t)p->out | (uintptr_t)p->out_rest | (uintptr_t)p->grad_query |
             (uintptr_t)p->grad_key | (uintptr_t)p->grad_value) & 15) == 0;
  return a;
}

// how one kernel's work is cut
struct Plan {
  bool pool;  // one query per sequence, by the kernels of their own
  Shape sh;
  int64_t tiles;
  int nsplit;
  int chunk;  // pool: keys of a wave where long sequences are cut
  int64_t slots;  // chunk > 0: partial results per head
  int64_t part_rows(int64_t rows, int64_t heads) const { return chunk ? slots * heads : nsplit > 1 ? nsplit * rows : 0; }
  bool parted() const { return chunk || nsplit > 1; }
};
Plan plan_tiles(int dtype, int D, int mode, int64_t B, int64_t n, int64_t G, int64_t heads,
                double stream_rows) {
  Plan pl{};
  const double per = mode == kWhole ? (double)n * G : (double)n * G / std::max<int64_t>(1, B);
  pl.sh = shape_for(dtype, D, per);
  pl.tiles = tiles_for(mode, B, n, G, pl.sh.bm);
  pl.nsplit = splits_for(pl.tiles * heads, pl.sh.nw, D, stream_rows);
  return pl;
}
double average(int64_t n, int64_t B) { return (double)n / std::max<int64_t>(1, B); }

// One query per sequence: a wave per sequence and key head while a few heads share the keys; a group of
// more than 4 heads fills enough of a matrix tile. How the lengths differ the host does not know, so
// sequences are cut into `chunk` keys, and whole ones cost no more than a look by the join: 1024, or what
// fills the card's 4096 waves where few sequences are long on average (equal numbers of parts left the
// longest of pool_lifelong's 7 histories of 9411 to 120000 keys alone at the end, 36 us for 28). One history
// of 100000 keys among 16384 of 40: 84 us and 97 for the gradient, 2993 and 5467 if one wave walks it; where
// there is none the look costs 4 us each way. No more keys than one chunk in all: nothing to cut. Behind a prefix,
// whose parts are joined in any case: equal parts by the average length, so that one candidate with a very long history
// of its own among many short ones is one wave's walk there, as it is one tile's in the tile kernels.
bool is_pool(const mono_attention_args* p) { return !p->query_splits && p->heads / p->kv_heads <= 4; }
Plan plan_pool(const mono_attention_args* p, bool equal) {
  Plan pl{};
  pl.pool = true;
  pl.nsplit = 1;
  const int64_t waves = std::max<int64_t>(1, p->batch * p->kv_heads), want = 256 * 16;
  const int64_t by_len = (int64_t)(average(p->n_key, p->batch) / 128);
  if (equal) {
    if (waves < want && by_len >= 2) pl.nsplit = (int)std::min<int64_t>(std::min<int64_t>(want / waves, by_len), 256);
    return pl;
  }
  const int64_t chunk = waves >= want || by_len < 2
                            ? 1024 : (std::max<int64_t>(128, p->n_key * p->kv_heads / want) + 63) / 64 * 64;
  if (p->n_key <= chunk) return pl;
  pl.chunk = (int)chunk;
  pl.slots = pool_part(p->n_key, pl.chunk) + 1;
  return pl;
}
Plan plan_fwd(const mono_attention_args* p, bool behind_prefix = false) {
  if (is_pool(p)) return plan_pool(p, behind_prefix);
  return plan_tiles(p->dtype, p->dim, p->query_splits ? kSplits : kOnePerSeq, p->batch, p->n_query,
                    p->heads / p->kv_heads, p->kv_heads, average(p->n_key, p->batch));
}
Plan plan_dkv(const mono_attention_args* p) {
  return plan_tiles(p->dtype, p->dim, kSplits, p->batch, p->n_key, 1, p->kv_heads,
                    average(p->n_query, p->batch) * (p->heads / p->kv_heads));
}

enum Which { kFwd, kDq, kDkv };
template <int W, typename T, int DP, int NC, int NW>
int launch1(const Args& a, const Plan& pl, hipStream_t st) {
  const dim3 grid((unsigned)(pl.tiles * a.Hkv), (unsigned)a.nsplit);
  if (W == kFwd) k_attn_fwd<T, DP, NC, NW><<<grid, NW * 64, 0, st>>>(a);
  else if (W == kDq) k_attn_dq<T, DP, NC, NW><<<grid, NW * 64, 0, st>>>(a);
  else k_attn_dkv<T, DP, NC, NW><<<grid, NW * 64, 0, st>>>(a);
  MONO_HIP(hipGetLastError());
  return 0;
}
// the pooled kernels; backward: 64 more workgroups for the rows of no sequence
template <int W, typename T, int DP, int GT>
int launch_pool2(const Args& a, hipStream_t st) {
  const int64_t wgs = (pool_items(a.B, a.Hkv, a.nk, a.nsplit, a.chunk) + 3) / 4;
  MONO_REQUIRE(wgs < (1LL << 24) - 64, "attention: too many sequences");
  if (W == kFwd) k_pool_fwd<T, DP, GT><<<(unsigned)wgs, 256, 0, st>>>(a);
  else k_pool_bwd<T, DP, GT><<<(unsigned)wgs + 64, 256, 0, st>>>(a);
  MONO_HIP(hipGetLastError());
  return 0;
}
template <int W, typename T, int DP>
int launch_pool1(const Args& a, hipStream_t st) {
  if (W == kFwd && a.B == 0) return 0;
  if (a.G == 1) return launch_pool2<W, T, DP, 1>(a, st);
  if (a.G == 2) return launch_pool2<W, T, DP, 2>(a, st);
  if (a.G == 3) return launch_pool2<W, T, DP, 3>(a, st);
  return launch_pool2<W, T, DP, 4>(a, st);
}
template <int W>
int launch_pool(int dtype, const Args& a, hipStream_t st) {
  if (dtype == MONO_ROW_BF16) {
    if (a.D <= 16) return launch_pool1<W, bf16, 16>(a, st);
    if (a.D <= 32) return launch_pool1<W, bf16, 32>(a, st);
    if (a.D <= 64) return launch_pool1<W, bf16, 64>(a, st);
    return launch_pool1<W, bf16, 128>(a, st);
  }
  if (a.D <= 16) return launch_pool1<W, float, 16>(a, st);
  if (a.D <= 32) return launch_pool1<W, float, 32>(a, st);
  if (a.D <= 64) return launch_pool1<W, float, 64>(a, st);
  return launch_pool1<W, float, 128>(a, st);
}
template <int W, typename T, int DP>
int launch2(const Args& a, const Plan& pl, hipStream_t st) {
  if (pl.tiles * a.Hkv == 0) return 0;
  MONO_REQUIRE(pl.tiles * a.Hkv < (1LL << 24), "attention: too many tiles");
  constexpr bool half = sizeof(T) == 2;
  if constexpr (half || DP <= 32)
    if (pl.sh.nw == 1) return launch1<W, T, DP, 1, 1>(a, pl, st);
  return launch1<W, T, DP, 1, 4>(a, pl, st);
}
template <int W>
int launch(int dtype, const Args& a, const Plan& pl, hipStream_t st) {
  if (pl.pool) return launch_pool<W>(dtype, a, st);
  if (dtype == MONO_ROW_BF16) {
    if (a.D <= 16) return launch2<W, bf16, 16>(a, pl, st);
    if (a.D <= 32) return launch2<W, bf16, 32>(a, pl, st);
    if (a.D <= 64) return launch2<W, bf16, 64>(a, pl, st);
    return launch2<W, bf16, 128>(a, pl, st);
  }
  if (a.D <= 16) return launch2<W, float, 16>(a, pl, st);
  if (a.D <= 32) return launch2<W, float, 32>(a, pl, st);
  if (a.D <= 64) return launch2<W, float, 64>(a, pl, st);
  return launch2<W, float, 128>(a, pl, st);
}

int64_t round16(int64_t b) { return (b + 15) & ~(int64_t)15; }
// partial rows and their statistics
int64_t parts_bytes(int64_t rows, int64_t D) { return round16(rows * D * 4) + round16(rows * 4); }

Parts parts_of(const mono_attention_args* p, int n, int64_t rows, int chunk) {
  return Parts{n, rows, p->key_splits, chunk, (int)p->batch, (int)p->n_key, p->heads};
}
int join(const mono_attention_args* p, const float* part, const float* part_lse, int n_part, int chunk, hipStream_t st) {
  const int64_t rows = p->n_query * p->heads;
  if (rows == 0) return 0;
  const int vec = p->dim % 4 == 0 && (((uintptr_t)p->out | (uintptr_t)p->out_rest) & 15) == 0;
  const bool many = (chunk && rows <= 4096) || n_part >= 16;
  const unsigned grid = many ? (unsigned)rows : (unsigned)grid_for(rows * ((p->dim + 3) / 4), 256, 1 << 20);
  const Parts parts = parts_of(p, n_part, rows, chunk);
  const auto go = [&](auto* out) {
    typedef typename std::remove_pointer<decltype(out)>::type T;
    T* rest = (T*)p->out_rest;
    if (!many) k_attn_join<T><<<grid, 256, 0, st>>>(part, part_lse, parts, rows, p->dim, out, rest, p->lse, vec);
    else if (vec) k_attn_join_many<T, true><<<grid, 1024, 0, st>>>(part, part_lse, parts, p->dim, out, rest, p->lse);
    else k_attn_join_many<T, false><<<grid, 1024, 0, st>>>(part, part_lse, parts, p->dim, out, rest, p->lse);
  };
  if (p->dtype == MONO_ROW_BF16) go((bf16*)p->out);
  else go((float*)p->out);
  MONO_HIP(hipGetLastError());
  return 0;
}
int sum_parts(int dtype, const float* part, const Parts& parts, int64_t total, int D, void* out, hipStream_t st) {
  if (total == 0) return 0;
  const int grid = grid_for(total, 256);
  if (dtype == MONO_ROW_BF16) k_sum_parts<bf16><<<grid, 256, 0, st>>>(part, parts, total, D, (bf16*)out);
  else k_sum_parts<float><<<grid, 256, 0, st>>>(part, parts, total, D, (float*)out);
  MONO_HIP(hipGetLastError());
  return 0;
}

// the two launches of the shared prefix: over the prefix, where the whole batch is one sequence, and
// over every sequence's own keys
struct PrefixPlan {
  Plan pre, own;
  int slots;
};
PrefixPlan plan_prefix(const mono_attention_args* p) {
  PrefixPlan r;
  const int64_t G = p->heads / p->kv_heads;
  r.pre = plan_tiles(p->dtype, p->dim, kWhole, 1, p->n_query, G, p->kv_heads, (double)p->n_prefix);
  r.slots = r.pre.nsplit;
  if (p->key_splits) {
    r.own = plan_fwd(p, true);
    r.slots += r.own.nsplit;
  }
  return r;
}
}  // namespace
}  // namespace mono

extern "C" {
using namespace mono;

int64_t mono_ragged_attention_workspace(const mono_attention_args* p) {
  if (check(p, "mono_ragged_attention_workspace")) return -1;
  return parts_bytes(plan_fwd(p).part_rows(p->n_query * p->heads, p->heads), p->dim);
}

int mono_ragged_attention(const mono_attention_args* p, void* stream) {
  MONO_TRY(check(p, "mono_ragged_attention"));
  MONO_REQUIRE(p->key_splits, "mono_ragged_attention: key_splits is NULL");
  if (p->n_query == 0) return 0;
  MONO_REQUIRE(p->query.ptr && p->out && (p->n_key == 0 || (p->key.ptr && p->value.ptr)),
               "mono_ragged_attention: a rows array is NULL");
  const Plan pl = plan_fwd(p);
  const int64_t rows = pl.part_rows(p->n_query * p->heads, p->heads);
  MONO_REQUIRE(p->workspace_bytes >= parts_bytes(rows, p->dim),
               "mono_ragged_attention: workspace of %lld bytes is too small", (long long)p->workspace_bytes);
  Args a = base_args(p);
  a.nsplit = pl.nsplit;
  a.chunk = pl.chunk;
  if (pl.parted()) {
    a.part = (float*)p->workspace;
    a.part_lse = (float*)((char*)p->workspace + round16(rows * p->dim * 4));
  }
  MONO_TRY(launch<kFwd>(p->dtype, a, pl, (hipStream_t)stream));
  return pl.parted() ? join(p, a.part, a.part_lse, pl.nsplit, pl.chunk, (hipStream_t)stream) : 0;
}

int64_t mono_ragged_attention_gradient_workspace(const mono_attention_args* p) {
  if (check(p, "mono_ragged_attention_gradient_workspace")) return -1;
  const Plan q = plan_fwd(p), k = plan_dkv(p);
  const int64_t nk = p->n_key * p->kv_heads;
  return round16(p->n_query * p->heads * 4) +
         std::max(round16(q.part_rows(p->n_query * p->heads, p->heads) * p->dim * 4),
                  q.pool ? 0 : 2 * round16(k.part_rows(nk, 0) * p->dim * 4));
}

int mono_ragged_attention_gradient(const mono_attention_args* p, void* stream) {
  MONO_TRY(check(p, "mono_ragged_attention_gradient"));
  MONO_REQUIRE(p->key_splits, "mono_ragged_attention_gradient: key_splits is NULL");
  MONO_REQUIRE(!p->grad_key || p->kv_shared || p->grad_value,
               "mono_ragged_attention_gradient: grad_value is NULL");
  MONO_REQUIRE(p->workspace_bytes >= mono_ragged_attention_gradient_workspace(p),
               "mono_ragged_attention_gradient: workspace of %lld bytes is too small",
               (long long)p->workspace_bytes);
  MONO_REQUIRE(p->n_query == 0 || (p->query.ptr && p->out && p->lse && p->grad_out.ptr && p->grad_query),
               "mono_ragged_attention_gradient: a rows array of the queries is NULL");
  MONO_REQUIRE(p->n_key == 0 || (p->key.ptr && p->value.ptr), "mono_ragged_attention_gradient: key or value is NULL");
  hipStream_t st = (hipStream_t)stream;
  const Plan plq = plan_fwd(p), plk = plan_dkv(p);
  const int64_t rows = p->n_query * p->heads, krows = p->n_key * p->kv_heads;
  float* scratch = (float*)((char*)p->workspace + round16(rows * 4));
  Args a = base_args(p);
  a.delta = (float*)p->workspace;
  a.nsplit = plq.nsplit;
  a.chunk = plq.chunk;
  a.part = plq.parted() ? scratch : nullptr;
  MONO_TRY(launch<kDq>(p->dtype, a, plq, st));
  if (a.part)
    MONO_TRY(sum_parts(p->dtype, a.part, parts_of(p, plq.nsplit, rows, plq.chunk), rows * p->dim, p->dim,
                       p->grad_query, st));
  if (!p->grad_key || plq.pool) return 0;  // (the pooled pass has written the keys' gradients)
  a.nsplit = plk.nsplit;
  a.part = plk.nsplit > 1 ? scratch : nullptr;
  a.part2 = a.part ? (float*)((char*)scratch + round16(plk.nsplit * krows * p->dim * 4)) : nullptr;
  MONO_TRY(launch<kDkv>(p->dtype, a, plk, st));
  if (a.part) {
    const Parts parts = parts_of(p, plk.nsplit, krows, 0);
    MONO_TRY(sum_parts(p->dtype, a.part, parts, krows * p->dim, p->dim, p->grad_key, st));
    if (!p->kv_shared) MONO_TRY(sum_parts(p->dtype, a.part2, parts, krows * p->dim, p->dim, p->grad_value, st));
  }
  return 0;
}

int64_t mono_shared_prefix_attention_workspace(const mono_attention_args* p) {
  if (check(p, "mono_shared_prefix_attention_workspace")) return -1;
  const int64_t slots = plan_prefix(p).slots;
  return slots > 1 ? parts_bytes(slots * p->n_query * p->heads, p->dim) : 0;
}

int mono_shared_prefix_attention(const mono_attention_args* p, void* stream) {
  MONO_TRY(check(p, "mono_shared_prefix_attention"));
  if (p->n_query == 0) return 0;
  MONO_REQUIRE(p->query.ptr && p->out && (!p->key_splits || p->n_key == 0 || (p->key.ptr && p->value.ptr)) &&
                   (p->n_prefix == 0 || (p->prefix_key.ptr && p->prefix_value.ptr)),
               "mono_shared_prefix_attention: a rows array is NULL");
  const PrefixPlan pl = plan_prefix(p);
  const int64_t rows = p->n_query * p->heads;
  MONO_REQUIRE(p->workspace_bytes >= (pl.slots > 1 ? parts_bytes(pl.slots * rows, p->dim) : 0),
               "mono_shared_prefix_attention: workspace of %lld bytes is too small",
               (long long)p->workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  Args a = base_args(p);
  if (pl.slots > 1) {
    a.part = (float*)p->workspace;
    a.part_lse = (float*)((char*)p->workspace + round16(pl.slots * rows * p->dim * 4));
  }
  if (p->key_splits) {
    a.nsplit = pl.own.nsplit;
    a.slot0 = pl.pre.nsplit;
    MONO_TRY(launch<kFwd>(p->dtype, a, pl.own, st));
  }
  a.k = p->prefix_key.ptr, a.ks = p->prefix_key.row_stride, a.kh = p->prefix_key.head_stride;
  a.v = p->prefix_value.ptr, a.vs = p->prefix_value.row_stride, a.vh = p->prefix_value.head_stride;
  a.vec_k = aligned_rows(p->prefix_key, p->dtype, p->dim);
  a.vec_v = aligned_rows(p->prefix_value, p->dtype, p->dim);
  a.mask = p->prefix_mask;
  a.nk = (int)p->n_prefix;
  a.qmode = a.kmode = kWhole;
  a.qbatch = a.B;
  a.B = 1;
  a.causal = 0;
  a.nsplit = pl.pre.nsplit;
  a.slot0 = 0;
  MONO_TRY(launch<kFwd>(p->dtype, a, pl.pre, st));
  return pl.slots > 1 ? join(p, a.part, a.part_lse, pl.slots, 0, st) : 0;
}
}
