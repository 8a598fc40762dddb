"""Plain 64-bit forms of the paged-cache operators, the layouts their tests
use, and the error bounds of the kernels' arithmetic."""
import math

import torch


def layout(counts, pos, page, num_extra=2, seed=0, max_pages=None, device="cuda", live=None):
    """A table of shuffled pages covering every position below pos + count of
    each sequence (only those that meet live(b) = [(a, e), ...] if given):
    (table, num_pages)."""
    g = torch.Generator().manual_seed(seed)
    need = []
    for b, (n, p) in enumerate(zip(counts, pos)):
        spans = live(b) if live else [(0, max(0, p + n))]
        need.append(sorted({i for a, e in spans if e > a for i in range(a // page, (e - 1) // page + 1)}))
    if max_pages is None:
        max_pages = max([1] + [i + 1 for l in need for i in l])
    total = sum(len(l) for l in need)
    order = torch.randperm(total + num_extra, generator=g).tolist()
    table = torch.full((len(counts), max_pages), -1, dtype=torch.int32)
    for b, l in enumerate(need):
        for i in l:
            table[b, i] = order.pop()
    return table.to(device), total + num_extra


def sees(i, j, window, sinks):
    """Whether the row at position i sees key j (tensors)."""
    m = j <= i
    if window:
        m = m & ((j > i - window) | (j < sinks))
    return m


def attention(q, k, v, table, counts, pos, window=0, sinks=0):
    """softmax(q k) v over the pages in 64 bits -> (out, bound): bound is
    sum p |v| and the scores' spread, from which the tests' tolerances come."""
    H, Dh = q.shape[1:]
    Hkv, ps = k.shape[1], k.shape[2]
    G = H // Hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    size = 0.0  # largest sum |q_d k_d| of a visible pair
    r = 0
    for b, (n, p) in enumerate(zip(counts, pos)):
        for i in range(p, p + n):
            if i >= 0:
                j = torch.arange(0, i + 1, device=q.device)
                j = j[sees(i, j, window, sinks)]
                pg = table[b, j // ps].long()
                held = (pg >= 0) & (pg < k.shape[0])
                j, pg = j[held], pg[held]
                if j.numel():
                    kk = k[pg, :, j % ps].double().transpose(0, 1)  # [Hkv][keys][Dh]
                    vv = v[pg, :, j % ps].double().transpose(0, 1)
                    qq = q[r].double().view(Hkv, G, Dh)
                    x = torch.softmax(qq @ kk.transpose(1, 2), -1)
                    out[r] = (x @ vv).view(H, Dh)
                    mass[r] = (x @ vv.abs()).view(H, Dh)
                    size = max(size, (qq.abs() @ kk.abs().transpose(1, 2)).max().item())
            r += 1
    return out, (mass, size)


def attention_tolerance(dtype, ref, bound, Dh, keys, p_eps):
    """Elementwise error bound of the kernels, from their arithmetic:
    - the output's rounding: eps/2 of the value;
    - P: `p_eps` relative each (hi + lo halves, or one 16-bit rounding);
    - a score: Dh products summed in fp32, off by Dh 2^-24 sum |q k|, and its
      product with log2 e and the difference to the maximum, 2^-22 of the
      score; an error d of a score moves the result by at most 2 d sum p |v|;
    - exp2: 2^-21 relative, in numerator and normaliser;
    - the sums over `keys` keys in fp32: keys 2^-24 relative, twice."""
    mass, size = bound
    eps = torch.finfo(dtype).eps / 2
    c = p_eps + 2 * (Dh * 2.0 ** -24 + 2.0 ** -22) * size + 2 * 2.0 ** -21 + 2 * keys * 2.0 ** -24
    tiny = torch.finfo(dtype).smallest_normal * eps * 2
    return eps * (ref.abs() + c * mass) + c * mass + tiny


def rope(qkv, H, Hkv, Dh, positions, theta, q_norm, k_norm, eps):
    """(q, k, v) in 64 bits of rows at `positions` (list)."""
    x = qkv.double().view(-1, H + 2 * Hkv, Dh)
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]

    def norm(t, w):
        return t if w is None else t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * w.double()

    j = torch.arange(Dh // 2, dtype=torch.float64, device=qkv.device)
    a = torch.tensor(positions, dtype=torch.float64, device=qkv.device)[:, None] * theta ** (-2 * j / Dh)
    c, s = a.cos()[:, None], a.sin()[:, None]

    def rot(t):
        lo, hi = t[..., :Dh // 2], t[..., Dh // 2:]
        return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)

    return rot(norm(q, q_norm)) / math.sqrt(Dh), rot(norm(k, k_norm)), v


def rope_tolerance(dtype, ref):
    """The output's rounding, and the fp32 norm (a sum of at most 256 squares:
    2^-24 each, halved by the root), sines (2^-22 of the pair's length) and
    products: 2^-18 of the head's largest value in all."""
    big = ref.abs().amax(-1, keepdim=True)
    return torch.finfo(dtype).eps / 2 * ref.abs() * 1.001 + 2.0 ** -18 * 2 * big + torch.finfo(dtype).smallest_normal


def spec_picks(target, draft, drafts, u, temperature):
    """Picks [k + 1][batch] of the definition, in 64 bits, row by row."""
    k, B, V = target.shape[0] - 1, target.shape[1], target.shape[2]
    picks = torch.full((k + 1, B), -1, dtype=torch.int32)

    def dist(x):
        return torch.softmax(x.double() / temperature, 0)

    for b in range(B):
        n, w = 0, None
        while n < k:
            p, q, d = dist(target[n, b]), dist(draft[n, b]), int(drafts[b, n])
            inside = 0 <= d < V
            if not (inside and float(u[b, n].double()) * float(q[d]) < float(p[d])):
                w = (p - q).clamp_min(0)
                break
            picks[n, b] = d
            n += 1
        if w is None:
            w = dist(target[k, b])
        c = w.cumsum(0)
        goal = u[b, k].double() * c[-1]
        picks[n, b] = int((c <= goal).sum().clamp_max(V - 1))
    return picks
