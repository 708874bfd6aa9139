"""Paged caches and 64-bit plain forms for the tests of the paged operators."""
import math

import torch


class Batch:
    """Sequences of a call: new tokens and cache lengths, pages in random order.

    Rows of the pool that no sequence owns hold `junk`; so do `tail` rows of the
    token buffers behind the last sequence."""

    def __init__(self, new, kv, nh, nkv, hd, page, dtype, order="rows", seed=0, junk=float("nan"), tail=0,
                 interleave=False, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.new, self.kv, self.nh, self.nkv, self.hd, self.page = new, kv, nh, nkv, hd, page
        need = [-(-x // page) for x in kv]
        self.n_pages = sum(need) + 2
        perm = torch.randperm(self.n_pages, generator=g)
        table = torch.full((len(new), max(need + [1]) + 1), -7, dtype=torch.int32)
        at = 0
        for i, m in enumerate(need):
            table[i, :m] = perm[at:at + m]
            at += m
        shape = (self.n_pages, page, nkv, hd) if order == "rows" else (self.n_pages, nkv, page, hd)
        if interleave:   # k and v of a page side by side in one pool
            pool = torch.full((shape[0], 2) + shape[1:], junk, dtype=dtype)
            pools = [pool[:, 0], pool[:, 1]]
        else:
            pools = [torch.full(shape, junk, dtype=dtype) for _ in range(2)]
        views = pools if order == "rows" else [p.transpose(1, 2) for p in pools]
        self.where = []
        for i, n in enumerate(kv):
            t = torch.arange(n)
            self.where.append((table[i].long()[t // page], t % page))
            for p in views:
                p[self.where[i]] = torch.randn(n, nkv, hd, generator=g).to(dtype)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        self.used, self.T = cu[-1], cu[-1] + tail
        self.q = torch.randn(self.T, nh, hd, generator=g)
        self.kn = torch.randn(self.T, nkv, hd, generator=g)
        self.vn = torch.randn(self.T, nkv, hd, generator=g)
        self.hk, self.hv = views
        self.cu = torch.tensor(cu, dtype=torch.int32)
        self.kv_len = torch.tensor(kv, dtype=torch.int32)
        self.table = table
        if device:
            if interleave:
                d = pool.to(device)
                dp = [d[:, 0], d[:, 1]]
            else:
                dp = [p.to(device) for p in pools]
            self.k, self.v = dp if order == "rows" else [p.transpose(1, 2) for p in dp]
            self.dq, self.dkn, self.dvn = self.q.to(device), self.kn.to(device), self.vn.to(device)

    def cache(self):
        from ternative_b200 import PagedCache
        return PagedCache(self.k, self.v)

    def batch(self, max_new=None, max_kv=None):
        from ternative_b200 import PagedBatch
        return PagedBatch(self.cu.cuda(), self.kv_len.cuda(), self.table.cuda(), self.T,
                          max(self.new) if max_new is None else max_new, max(self.kv) if max_kv is None else max_kv)

    def attention(self, scale=None, window=0, limit=None):
        """(out, lse, bound) in 64 bits; `limit` masks keys from a position on (a page that does not exist).
        bound: how far 32-bit arithmetic may be off, per output row (see `attention_bound`)."""
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        g = self.nh // self.nkv
        out = torch.zeros(self.used, self.nh, self.hd, dtype=torch.float64)
        lse = torch.full((self.used, self.nh), -math.inf, dtype=torch.float64)
        tol = torch.zeros(self.used, self.nh, dtype=torch.float64)
        r = 0
        for i, (n, kv) in enumerate(zip(self.new, self.kv)):
            k, v = self.hk[self.where[i]].double(), self.hv[self.where[i]].double()
            for j in range(n):
                p = kv - n + j
                lo = max(0, p - window + 1) if window else 0
                hi = min(p + 1, limit[i]) if limit else p + 1
                for h in range(self.nh):
                    if hi <= lo:
                        continue
                    q, kk, vv = self.q[r, h].double(), k[lo:hi, h // g], v[lo:hi, h // g]
                    z = kk @ q * scale
                    w = torch.softmax(z, 0)
                    out[r, h], lse[r, h] = w @ vv, torch.logsumexp(z, 0)
                    tol[r, h] = attention_bound(q, kk, vv, scale)
                r += 1
        return out, lse, tol


U = 2.0 ** -24   # half a step of F32


def attention_bound(q, k, v, scale):
    """A score is a sum of hd products in F32 (at most (hd + 4) U times the sum of their magnitudes S, splitting an
    operand into planes included); the exponential adds 2^-21, a probability's planes 2^-21, the sums over n keys n U;
    a relative error e of every probability moves the weighted mean by at most 2 e max |v|."""
    S = float(((k.abs() @ q.abs()) * abs(scale)).max())
    n, hd = k.shape
    return 2 * float(v.abs().max()) * ((hd + 4) * U * S + 2.0 ** -20 + n * U)


def rope_frequencies(rot, theta, scaling, factor, original, low=1.0, high=4.0, fast=32.0, slow=1.0):
    f, m = [], 1.0
    for i in range(rot // 2):
        w = theta ** (-2.0 * i / rot)
        if scaling == "linear":
            w /= factor
        elif scaling == "bands":
            turns = original * w / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            w = w * keep + w / factor * (1 - keep)
        elif scaling == "yarn":
            def pair(t):
                return rot * math.log(original / (t * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
            ramp = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            w = w / factor * ramp + w * (1 - ramp)
            m = 0.1 * math.log(factor) + 1.0
        f.append(w)
    return torch.tensor(f, dtype=torch.float64), m


def rope(x, pos, rot, pairs, f, m):
    """x [T][heads][hd] in 64 bits, turned by pos * f."""
    x = x.double().clone()
    a = pos.double()[:, None, None] * f
    c, s = a.cos() * m, a.sin() * m
    i = torch.arange(rot // 2)
    u, w = (2 * i, 2 * i + 1) if pairs == "interleaved" else (i, i + rot // 2)
    p, q = x[..., u].clone(), x[..., w].clone()
    x[..., u], x[..., w] = p * c - q * s, q * c + p * s
    return x
