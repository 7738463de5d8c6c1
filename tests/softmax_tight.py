"""Tolerances of the vocabulary softmax's gradient that do not forgive a cancellation.

Those of test_gpu_vocab_softmax.Exact, with the target's coefficient taken as what it is, G_t = g (1 - p_t) - h p_t (log p_t + H),
not as the difference of g and g p_t.  u = 2^-24.
  1 - p_t          the sum of the other ids' probabilities, each off by tol_p of itself, or (p_t below a half) 1 - p_t, off by
                   p_t tol_p, which is less: (1 - p_t) tol_p either way
  G, in bf16       2^-8 of |G| itself, the target's included (db sums G in float32: none)
  float32          an element goes into the products as two float16 (2^-22 of itself, in the sums' terms) of a value scaled by a power
                   of two that its row shares with rows no more than 2^8 (2^9 with the rounding to powers of two) larger: 2^-37 of the
                   scale's largest, hence 2^-28 of the row's largest element m_j.  A weight c_j is off by 2^-37 of the
                   largest |c_k| 2^9 m_k / (2^9 m_j), times an element of at most m_j: 2^-28 of max_k |c_k| m_k.
                   Together N 2^-27 max_j |c_j| m_j for N terms.
  small p          below 2^-126 they may be 0: N 2^-126 of the largest gradient times the largest element"""
import math

import torch

from .test_gpu_vocab_softmax import F32, U, Exact


class Tight(Exact):
    def gradient(self, g, h, dtype):
        """-> ((dx, tolerance), (dw, tolerance), (db, tolerance))"""
        n, V = self.s.shape
        zero = torch.zeros(n, dtype=torch.float64, device=self.s.device)
        g = zero if g is None else torch.where(self.has, g.double(), 0.0)
        h = zero if h is None else torch.where(self.empty, 0.0, h.double())
        spread = h.abs()[:, None] * (self.finite.abs() + self.H[:, None])
        G = -self.p * (g[:, None] + h[:, None] * (self.finite + self.H[:, None]))
        of_h = self.p * (self.tol_p * spread + h.abs()[:, None] * (self.tol_lse + self.tol_H)[:, None])
        of_g = self.p * self.tol_p * g.abs()[:, None]
        mass = self.p * (g.abs()[:, None] + spread)
        rows = torch.nonzero(self.has).view(-1)
        t = self.t[rows]
        others = self.p.clone()
        others[rows, t] = 0.0
        rest = torch.where(self.empty, 1.0, others.sum(1))[rows]                # 1 - p_t, to the last bit
        p, log_p = self.p[rows, t], self.finite[rows, t]
        G[rows, t] = g[rows] * rest - h[rows] * p * (log_p + self.H[rows])
        of_g[rows, t] = g[rows].abs() * rest * self.tol_p[rows, t]
        mass[rows, t] = g[rows].abs() * rest + p * spread[rows, t]
        err = of_g + of_h + 4 * U * mass
        self.G = G
        step = torch.finfo(dtype).eps / 2
        half = 0.0 if dtype == F32 else 2.0 ** -8

        def through(value, tol, m, other):
            length = other.shape[0]
            out = value @ other
            off = (tol + half * value.abs() * (1 + half) + half * tol) @ other.abs() + (8 * math.sqrt(length) + 16) * U * m @ other.abs()
            if dtype == F32:
                off = off + length * 2.0 ** -27 * (m * other.abs().amax(1)[None, :]).amax(1, keepdim=True)
            off = off + length * 2.0 ** -126 * float((g.abs() + h.abs()).max()) * (self.w.abs().max() + self.x.abs().max())
            return out, off + step * out.abs() * (1 + step) + step * off + 1e-37
        tr = lambda a: a.t().contiguous()
        db = G.sum(0)
        tdb = err.sum(0) + (8 * math.sqrt(n) + 16) * U * mass.sum(0) + 2 * U * db.abs() + 1e-37
        return through(G, err, mass, self.w), through(tr(G), tr(err), tr(mass), self.x), (db, tdb)
