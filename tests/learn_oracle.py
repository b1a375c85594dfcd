"""The operators of include/omk_learn.h in 64 bits, plainly, and how far a result in fewer bits may be from them.

What is allowed counts roundings.  U = 2^-24 is half a step of a 32-bit float.  For a row with largest logit m and
d = m - x:
  exp(x - m)   the difference is rounded (d U), its product with log2(e) twice (the constant and the product, 2 d U), and
               2^y is good to a step (2 U): (3 d + 2) U relative, and an absolute 2^-126 where it underflows
  S            terms that are off by (3 dbar + 2) U on the average, dbar = sum p d, and a tree of sums:
               (3 dbar + 2 + n/64 + 16) U (a lane adds n/64 of them one after another at most, then come the lanes and wavefronts)
  p            the sum of both, and a reciprocal and a product: (3 (d + dbar) + n/64 + 24) U
  log S        S's, and 2 U for the logarithm (which is taken in 64 bits)
"""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # relative to the value
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}


class Rows:
    """Logits [rows, actions] (float64, as the given type holds them), legal [rows, actions] or None."""

    def __init__(self, x, legal=None):
        self.x = np.where(legal, x, -np.inf) if legal is not None else x.copy()
        n = self.x.shape[1]
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            top = self.x.max(1)
            self.some = ~(top == -np.inf)
            self.top = np.where(self.some, top, 0.0)
            self.d = self.top[:, None] - self.x
            e = np.exp(-self.d)
            self.sum = e.sum(1)
            self.p = np.where(self.some[:, None], e / np.where(self.some, self.sum, 1.0)[:, None], 0.0)
            self.log_sum = np.where(self.some, np.log(np.where(self.some, self.sum, 1.0)), 0.0)
            self.dbar = np.where(self.p > 0, self.p * self.d, 0.0).sum(1)
            self.entropy = np.where(self.some, self.log_sum + self.dbar, 0.0)
        self.chain = n / 64 + 24
        finite_d = np.where(np.isfinite(self.d), self.d, 0.0)
        self.p_rel = (3 * (finite_d + self.dbar[:, None]) + self.chain) * U
        self.log_sum_off = (3 * self.dbar + self.chain + 4) * U

    def priors_off(self):
        return self.p * self.p_rel + 2.0 ** -126

    def entropy_off(self):
        # sum e d / S: its terms' errors, weighted with d; then the rounding of the two and of their difference
        d = np.where(self.p > 0, self.d, 0.0)
        d2 = (self.p * d * (3 * d + self.chain)).sum(1) * U
        return self.log_sum_off * (1 + self.dbar) + d2 + (self.entropy + 2 * self.dbar) * 2 * U

    def taken(self, moves):
        """(log-probability in 64 bits, rows that count, how far it may be off before it is rounded)."""
        rows, n = self.x.shape
        inside = (moves >= 0) & (moves < n)
        chosen = self.x[np.arange(rows), np.where(inside, moves, 0)]
        counts = inside & self.some & ~(chosen == -np.inf)
        with np.errstate(invalid="ignore"):
            lp = chosen - self.top - self.log_sum
        return np.where(counts, lp, 0.0), counts, self.log_sum_off

    def gradient(self, moves, slope, slope_off, kind):
        """(gradient, how far it may be off) of rows whose loss has the derivative `slope` by the move's log-probability
        (0: left out), itself known to slope_off."""
        rows, n = self.x.shape
        one = np.zeros((rows, n))
        here = (slope != 0) | (slope_off != 0)
        one[np.nonzero(here)[0], moves[here]] = 1.0
        with np.errstate(invalid="ignore"):
            g = np.where(here[:, None], slope[:, None] * (one - self.p), 0.0)
            off = np.abs(slope)[:, None] * (self.p * (self.p_rel + 2 * U) + one * 2 * U) + slope_off[:, None] * np.abs(one - self.p)
            off = off + 2.0 ** -126 * np.abs(slope)[:, None] + np.abs(g) * HALF_STEP[kind] * (1 + 1e-6) + TINY[kind]
        return g, np.where(here[:, None], off, 0.0)


def policy_loss(rows, moves, old, advantage, ref, weight, clip_low, clip_high, kl_weight, scale):
    """dict of (value, off) for logprob, kl, loss and slope."""
    lp, counts, off = rows.taken(moves)
    # (rows that count nothing may hold anything in their other columns)
    old, advantage = np.where(counts, old, 0.0), np.where(counts, advantage, 0.0)
    weight = np.where(counts, 1.0 if weight is None else weight, 0.0)
    shift = lp - old
    ratio = np.exp(shift)
    low, high = 1.0 - clip_low, 1.0 + clip_high
    clipped = np.where(advantage > 0, ratio > high, (advantage < 0) & (ratio < low))
    row = -np.minimum(ratio * advantage, np.clip(ratio, low, high) * advantage)
    slope = np.where(clipped, 0.0, -advantage * ratio)
    # expf is good to two steps, its argument is rounded; a product
    ratio_rel = off + np.abs(shift) * U + 6 * U
    row_off = np.where(clipped, np.abs(row) * 3 * U, np.abs(row) * ratio_rel)
    slope_off = np.where(clipped, 0.0, np.abs(slope) * ratio_rel)
    kl, kl_off = np.zeros_like(lp), np.zeros_like(lp)
    if ref is not None:
        d = np.where(counts, ref - lp, 0.0)
        kl = np.expm1(d) - d
        d_off = off + np.abs(d) * U
        # exp(d + t) - (d + t) - 1 is (exp(d) - d - 1) + (exp(d) - 1) t + exp(d) t^2 / 2 + .., |t| <= d_off: where d is 0 the
        # second term is all there is
        kl_off = np.abs(np.expm1(d)) * d_off + np.exp(np.abs(d)) * d_off ** 2 + kl * 12 * U + (np.exp(d) + np.abs(d) + 1) * 4 * U * (np.abs(d) >= 0.25)
        row, row_off = row + kl_weight * kl, row_off + kl_weight * (kl_off + 3 * U * kl)
        slope = slope - kl_weight * np.expm1(d)
        # exp(d) - 1 as d and exp(d) - d - 1 added: the rounding of exp(d) (two steps) and of the differences, of magnitudes up to
        # exp(d) + |d| + 1
        slope_off = slope_off + kl_weight * (np.exp(d) * d_off + 6 * U * np.abs(np.expm1(d)) +
                                             (np.abs(d) >= 0.25) * 6 * U * (np.exp(d) + np.abs(d) + 1))
    w = weight * scale
    slope_off = slope_off + 3 * U * np.abs(slope)
    # a ratio within rounding of a border may fall on either side of it: the loss has the same value there, but not the slope
    border = np.minimum(np.abs(shift - np.log(high)), np.abs(shift - np.log(low)) if low > 0 else np.inf)
    slope_off = np.where(border < 2 * off, slope_off + np.abs(advantage) * ratio, slope_off) * np.abs(w)
    loss = (w * row).sum()
    loss_off = (np.abs(w) * (row_off + 4 * U * np.abs(row))).sum() + abs(loss) * 2 * U
    return dict(logprob=(lp, off + np.abs(lp) * U), kl=(np.where(counts, kl, 0.0), kl_off), loss=(loss, loss_off),
                slope=(np.where(counts, w * slope, 0.0), np.where(counts, slope_off, 0.0)))


def preference_loss(rows, moves, begin, ref, beta, smoothing, scale):
    lp, counts, off = rows.taken(moves)
    n = len(lp)
    begin = np.clip(begin, 0, n)
    lines = len(begin) - 1
    sums = np.array([lp[begin[k]:begin[k + 1]].sum() for k in range(lines)])
    sums_off = np.array([(off + np.abs(lp) * U)[begin[k]:begin[k + 1]].sum() for k in range(lines)])
    gain = sums - (0.0 if ref is None else ref)
    u = beta * (gain[0::2] - gain[1::2])
    u_off = np.abs(beta) * (sums_off[0::2] + sums_off[1::2]) + np.abs(u) * 2 * U
    softplus = lambda t: np.maximum(t, 0) + np.log1p(np.exp(-np.abs(t)))  # noqa: E731
    pair = (1 - smoothing) * softplus(-u) + smoothing * softplus(u)
    sig = lambda t: np.exp(-softplus(-t))  # noqa: E731
    bracket = (1 - smoothing) * sig(-u) - smoothing * sig(u)
    slope = -beta * scale * bracket
    # the bracket's derivative is at most 1/4; expf, a sum, a quotient, two products and a difference round
    slope_off = np.abs(beta * scale) * (np.minimum(0.25, sig(u) * sig(-u)) * u_off * 1.01 + 16 * U * ((1 - smoothing) * sig(-u) + smoothing * sig(u)))
    loss = scale * pair.sum()
    loss_off = abs(scale) * (u_off + pair * 12 * U).sum() + abs(loss) * 2 * U
    row_slope, row_off = np.zeros(n), np.zeros(n)
    for k in range(lines):
        at = slice(begin[k], begin[k + 1])
        row_slope[at] = slope[k // 2] * (1 if k % 2 == 0 else -1)
        row_off[at] = slope_off[k // 2]
    return dict(loss=(loss, loss_off), margin=(u, u_off), logprob=(sums, sums_off + np.abs(sums) * U),
                slope=(np.where(counts, row_slope, 0.0), np.where(counts, row_off, 0.0)))
