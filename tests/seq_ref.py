"""64-bit restatements of the sequence and loss operators with a bound on every element's error.

The bounds count roundings. `half` is half a step of the rows' type relative to the value (bf16 2^-8,
fp32 2^-24), e is what 32-bit sums and exponentials leave of a weight p relative to it: a logit of
products whose magnitudes sum to S is off by (dim + 2) roundings of S, its exponent's base change and
the subtraction of the maximum by two more, the hardware exponential by one step (two roundings), the
weight's numerator and the softmax's sum each carry this once, and a sum of n terms n roundings."""
import numpy as np

U32 = 2.0 ** -24
HALF = {"bf16": 2.0 ** -8, "fp32": 2.0 ** -24}


def _weight_error(S, dim, n):
  return 2 * U32 * ((dim + 2) * S + 2 * 1.4427 * S + 4) + 2 * U32 * (n + 8)


def attention(q, k, v, segments, keep, scale, dtype, g=None):
  """q [nq, H, D], k, v [nk, Hkv, D] float64; segments: list of (query rows, key rows) index arrays;
  keep(c, nq, nk) -> bool [nq, nk]. Returns {name: (value, bound)}."""
  half = HALF[dtype]
  nq, H, D = q.shape
  G = H // k.shape[1]
  out, lim = np.zeros_like(q), np.zeros_like(q)
  res = {}
  if g is not None:
    dq, bq = np.zeros_like(q), np.zeros_like(q)
    dk, bk = np.zeros_like(k), np.zeros_like(k)
    dv, bv = np.zeros_like(v), np.zeros_like(v)
  for c, (qi, ki) in enumerate(segments):
    if len(qi) == 0 or len(ki) == 0:
      continue
    ok = keep(c, len(qi), len(ki))
    for h in range(H):
      j = h // G
      Q, K, V = q[qi, h], k[ki, j], v[ki, j]
      # what lies in a masked row does not take part, whatever it is
      seen = ok.any(0)
      K, V = np.where(seen[:, None], K, 0), np.where(seen[:, None], V, 0)
      s = np.where(ok, Q @ K.T * scale, -np.inf)
      m = s.max(1, keepdims=True)
      m[~np.isfinite(m)] = 0
      p = np.exp(s - m)
      z = p.sum(1, keepdims=True)
      p /= np.where(z == 0, 1, z)
      S = (np.abs(Q) @ np.abs(K).T * scale)[ok].max() if ok.any() else 0.0
      e = _weight_error(S, D, len(ki))
      A = p @ np.abs(V)
      o = p @ V
      out[qi, h] = o
      # weights rounded to the type, sums in 32 bits, one rounding of the result
      off = (half + e) * A
      lim[qi, h] = off + half * (np.abs(o) + off)
      if g is None:
        continue
      Gr = g[qi, h]
      dp = Gr @ V.T
      dpa = np.abs(Gr) @ np.abs(V).T
      delta = (Gr * o).sum(1, keepdims=True)
      ga = (np.abs(Gr) * A).sum(1, keepdims=True)
      # delta is taken from the rounded result
      ddelta = (np.abs(Gr) * lim[qi, h]).sum(1, keepdims=True) + (D + 2) * U32 * ga
      ds = p * (dp - delta)
      spread = p * (dpa + ga)
      dds = half * np.abs(ds) + p * (ddelta + (D + 2) * U32 * dpa) * (1 + half) + (e + 2 * U32) * spread
      n = len(qi) * G
      x = scale * (ds @ K)
      off = scale * ((dds + (len(ki) + 2) * U32 * spread) @ np.abs(K))
      dq[qi, h], bq[qi, h] = x, off + half * (np.abs(x) + off)
      dk[ki, j] += scale * (ds.T @ Q)
      bk[ki, j] += scale * ((dds + (n + 2) * U32 * spread).T @ np.abs(Q))
      dv[ki, j] += p.T @ Gr
      bv[ki, j] += ((half + e + (n + 2) * U32) * p).T @ np.abs(Gr)
  res["out"] = (out, lim)
  if g is not None:
    res["dq"] = (dq, bq)
    res["dk"] = (dk, bk + half * (np.abs(dk) + bk))
    res["dv"] = (dv, bv + half * (np.abs(dv) + bv))
    both, off = dk + dv, bk + bv
    res["dkv"] = (both, off + 2 * U32 * (np.abs(dk) + np.abs(dv)) + half * (np.abs(both) + off))
  return res


def segments(query_splits, key_splits):
  """Index arrays of every sequence; query_splits None: one query each."""
  out = []
  for b in range(len(key_splits) - 1):
    qi = np.arange(b, b + 1) if query_splits is None else np.arange(query_splits[b], query_splits[b + 1])
    out.append((qi, np.arange(key_splits[b], key_splits[b + 1])))
  return out


def keep_rule(segs, mask, causal):
  def keep(c, nq, nk):
    ok = np.ones((nq, nk), bool)
    if causal:
      ok &= np.arange(nk)[None] <= np.arange(nq)[:, None] + nk - nq
    if mask is not None:
      ok &= mask[segs[c][1]][None]
    return ok
  return keep


def cross_entropy(q, w, labels, bias, scale, dtype, g=None):
  """loss (fp32) and gradients of softmax cross entropy; bias None or [V]."""
  half = HALF[dtype]
  n, D = q.shape
  V = w.shape[0]
  b = np.zeros(V) if bias is None else bias
  alive = b != -np.inf
  w = np.where(alive[:, None], w, 0)
  b0 = np.where(alive, b, 0)
  l = np.where(alive, scale * (q @ w.T) + b0, -np.inf)
  S = (scale * np.abs(q) @ np.abs(w).T + np.abs(b0)).max() if n else 0.0
  e = _weight_error(S, D, V)
  m = l.max(1, keepdims=True)
  m[~np.isfinite(m)] = 0
  z = np.exp(l - m).sum(1, keepdims=True)
  with np.errstate(divide="ignore"):
    lse = np.log(z) + m
  known = (labels >= 0) & (labels < V)
  lab = np.where(known, labels, 0)
  out = known & ~alive[lab]
  live = known & ~out
  loss = np.where(live, lse[:, 0] - np.where(live, l[np.arange(n), lab], 0), 0.0)
  loss[out] = np.inf
  loss[~known & (labels != -1)] = np.nan
  # the sum's relative error is the logarithm's absolute one; the logarithm in base 2, its change of
  # base, the logit and the difference each round values of at most S + log V
  top = S + np.log(V) + 1
  res = {"loss": (loss, np.full(n, e + U32 * (D + 12) * top))}
  if g is not None:
    gl = np.where(live, g, 0.0)[:, None]
    p = np.where(live[:, None], np.exp(l - np.where(live[:, None], lse, 0)), 0)
    hot = np.zeros_like(p)
    hot[np.arange(n)[live], lab[live]] = 1
    x = scale * ((p - hot) * gl) @ w
    off = scale * np.abs(gl) * (((half + e + (V + 2) * U32) * p + 4 * U32 * hot) @ np.abs(w))
    res["dq"] = (x, off + half * (np.abs(x) + off))
    ds = (p - hot) * gl
    dds = np.abs(gl) * (e * p + 4 * U32 * (p + hot)) + half * np.abs(ds)
    x = scale * ds.T @ q
    off = scale * (dds + (n + 2) * U32 * np.abs(gl) * (p + hot)).T @ np.abs(q)
    res["dw"] = (x, off + half * (np.abs(x) + off))
    x = ds.sum(0)
    res["db"] = (x, (np.abs(gl) * (e * p + (n + 6) * U32 * (p + hot))).sum(0))
  return res


def check(got, want, what):
  """got (torch) within the bound of want (value, bound), element by element."""
  value, bound = want
  got = got.detach().to("cpu").double().numpy()
  assert got.shape == value.shape, (what, got.shape, value.shape)
  special = ~np.isfinite(value)
  assert np.array_equal(np.isnan(got), np.isnan(value)), what
  assert np.array_equal(got[special & ~np.isnan(value)], value[special & ~np.isnan(value)]), what
  err = np.abs(got[~special] - value[~special])
  lim = bound[~special] + 1e-30
  if err.size:
    worst = (err / lim).max()
    assert worst <= 1.0, "%s: an element is off by %.3g times its bound (%d of %d over)" % (
        what, worst, int((err > lim).sum()), err.size)
