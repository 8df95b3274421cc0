"""Plain 64-bit forms of the operators that keep a cache small, and the error their kernels may have."""
import numpy as np
import torch


def visible(pos, m, window, sinks, live=None):
    """[len(pos), m]: which of m keys the queries at positions pos see."""
    p, j = torch.as_tensor(np.asarray(pos), dtype=torch.int64)[:, None], torch.arange(m)[None]
    see = j <= p
    if window > 0:
        see = see & ((j < sinks) | (j > p - window))
    return see if live is None else see & live[None]


def softmax(s, see):
    """Softmax of s over its last dimension among the visible entries; zeros where there are none."""
    s = torch.where(see, s, -torch.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(s.shape[:-1] + (1,))
    w = torch.where(see, torch.exp(s - torch.where(top == -torch.inf, 0.0, top)), 0.0)
    total = w.sum(-1, keepdim=True)
    return torch.where(total > 0, w / total, 0.0)


def weight_sums(q, k, pos, window, sinks, live=None):
    """One sequence in float64: q [n, Hq, D] at positions pos, k [m, Hk, D]. (the weights summed over rows and group
    [Hk, m], what the kernel's roundings may add up to there).

    * a score is D products and a few scalings in 32 bits: D + 16 roundings of e = sum_d |q_d k_jd| / sqrt(D); a
      weight's exponent holds one such score and the row's lse, which is off by as much, and their difference is
      rounded once, at most e + log2(m) + 1 in size: 2 (D + 24) 2^-24 e and 4 (log2(m) + 1) 2^-24 relative;
    * two exp2 and the row's sum, merged over tiles: 4 of 2^-22 and m additions;
    * the sum over rows and group: one rounding per row of what is there so far;
    * weights below 2^-126 are gone: rows of them."""
    n, Hq, D = q.shape
    m, Hk, _ = k.shape
    G = Hq // Hk
    q, k = q.double().cpu(), k.double().cpu()
    see = visible(pos, m, window, sinks, live)
    out, tol = torch.zeros(Hk, m, dtype=torch.float64), torch.zeros(Hk, m, dtype=torch.float64)
    for h in range(Hk):
        for g in range(G):
            s = (q[:, h * G + g] @ k[:, h].t()) / D ** 0.5
            e = torch.where(see, q[:, h * G + g].abs() @ k[:, h].abs().t() / D ** 0.5, 0.0).amax(-1, keepdim=True) \
                if m else s
            w = softmax(s, see)
            out[h] += w.sum(0)
            rel = 2 * (D + 24) * 2.0 ** -24 * e + (4 * (np.log2(max(m, 2)) + 1) + m + n * G) * 2.0 ** -24 + 2.0 ** -20
            tol[h] += (w * rel).sum(0) + n * 2.0 ** -126
    return out, tol
