"""Cases that time and check the operators of a serving step over a paged KV cache:

* ``rope``: rotary positions of the new tokens' q and k (half and interleaved pairs, part of the
  head, scaled for long contexts) with the append of k and v to the paged cache,
* ``attention``: attention of new tokens (one a sequence, or a chunk) over the paged cache,
* ``lora``: the low-rank adapters of many requests beside a projection that they share.

Each has a plain form in elementary torch operations and the framework's own call (``own``).
"""
import math

import torch

own = False

# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------


def _rope(name, n, new, kv, heads, hd, rot, pairs, scaling, page, dtype, order):
    return {"name": name, "op": "rope", "n": n, "new": new, "kv": kv, "nh": heads[0], "nkv": heads[1], "hd": hd,
            "rot": rot, "pairs": pairs, "scaling": scaling, "page": page, "dtype": dtype, "order": order}


def _attention(name, n, new, kv, heads, hd, window, page, dtype, order):
    return {"name": name, "op": "attention", "n": n, "new": new, "kv": kv, "nh": heads[0], "nkv": heads[1], "hd": hd,
            "window": window, "page": page, "dtype": dtype, "order": order}


def _lora(name, M, K, N, weight, adapters, rank, mixed, dtype):
    return {"name": name, "op": "lora", "M": M, "K": K, "N": N, "weight": weight, "adapters": adapters, "rank": rank,
            "mixed": mixed, "dtype": dtype}


def listed():
    return [
        # eight sequences, each with its next token, before a decode step's attention
        _rope("rope-decode-8", 8, 1, 512, (20, 5), 128, 128, "half", "none", 16, "f32", "rows"),
        # a long prompt's chunk at far positions, frequencies scaled by wavelength
        _rope("rope-prompt-far", 1, 2048, 33333, (32, 8), 128, 128, "interleaved", "bands", 64, "f16", "rows"),
        # chunks of several prompts and single tokens together, half of each head rotated, odd pages
        _rope("rope-mixed-partial", 7, 700, 5000, (20, 5), 128, 64, "half", "yarn", 5, "f16", "heads"),
        # one short conversation: latency
        _attention("attention-decode-1", 1, 1, 130, (20, 5), 128, 0, 16, "f32", "rows"),
        # a full serving batch, lengths from short to the model's longest
        _attention("attention-decode-32", 32, 1, 4096, (20, 5), 128, 0, 16, "f16", "rows"),
        # few long documents: the split over the cache matters
        _attention("attention-decode-long", 4, 1, 61000, (32, 8), 128, 0, 64, "f16", "rows"),
        # prompt chunks after long prefixes: the tensor cores' case
        _attention("attention-chunk", 4, 512, 6000, (32, 8), 128, 0, 64, "f16", "heads"),
        # ragged chunks over a 32-bit cache, a sliding window, pages that end inside any tile
        _attention("attention-chunk-window", 6, 300, 2500, (20, 5), 128, 1024, 24, "f32", "rows"),
        # one request's token through one projection: latency
        _lora("lora-decode-1", 1, 2560, 2560, "f16", 1, 16, False, "f32"),
        # eight requests, an adapter each, through a wide projection
        _lora("lora-decode-8", 8, 4096, 14336, "f16", 8, 16, False, "f16"),
        # sixteen requests on INT8 weights, adapters of several ranks, some requests without one
        _lora("lora-decode-16-int8", 16, 6912, 2560, "i8", 5, 64, True, "f32"),
        # prompt chunks of several requests and single tokens in one call
        _lora("lora-chunk", 1400, 2560, 6912, "f16", 6, 64, True, "f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "attention", "attention", "lora", "lora"])
    if op == "lora":
        K = rng.choice([256, 512, 2560, 4096, 6912, 64 * rng.randint(3, 80)])
        N = rng.choice([512, 640, 2560, 6912, 4096, _log(rng, 100, 8000)])
        M = _log(rng, 1, 1400)
        M = max(1, min(M, 1400 * 2560 * 6912 // (K * N)))
        rank = rng.choice([4, 8, 16, 32, 64, rng.randint(1, 64)])
        case = _lora("", M, K, N, rng.choice(["f16", "f16", "i8"]), _log(rng, 1, 12), rank, rng.random() < 0.5,
                     rng.choice(["f32", "f16"]))
    else:
        heads = rng.choice([(20, 5), (32, 8), (4, 2), (2, 1), (8, 8), (16, 2)])
        hd = rng.choice([64, 128, 128])
        page = rng.choice([1, 5, 16, 16, 24, 64, 128])
        dtype = rng.choice(["f32", "f16", "f16"])
        order = rng.choice(["rows", "heads"])
        decode = rng.random() < 0.5
        new = rng.choice([1, 1, 1, 2, 5]) if decode else _log(rng, 6, 1024)
        n = _log(rng, 1, 48) if decode else _log(rng, 1, max(1, 2048 // new))
        kv = max(new, _log(rng, 32, min(30000, 130000 // n)))
        if op == "rope":
            case = _rope("", n, new, kv, heads, hd, rng.choice([hd, hd, hd // 2, hd // 4]),
                         rng.choice(["half", "interleaved"]), rng.choice(["none", "linear", "bands", "yarn"]), page,
                         dtype, order)
        else:
            if not decode:
                kv = max(new, min(kv, 5_000_000 // (n * new)))
            case = _attention("", n, new, kv, heads, hd, rng.choice([0, 0, 0, _log(rng, 16, 4096)]), page, dtype, order)
    del case["name"]
    return case


def _lens(case):
    """New tokens and cache lengths (those tokens among them) of a case's sequences: from short to the longest."""
    n, new, kv = case["n"], case["new"], case["kv"]
    t = [new if i == 0 else 1 + (i * 7919 + 13) % new for i in range(n)]
    return t, [kv if i == 0 else t[i] + (i * 104729 + 31) % (kv - t[i] + 1) for i in range(n)]


def _ranks(case):
    r = case["rank"]
    return [max(1, r >> (i % 3)) if case["mixed"] else r for i in range(case["adapters"])]


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _paged(case, g):
    """A paged cache in use: its pools, the sequences' pages in no order, the lengths after the new tokens."""
    t, kv = _lens(case)
    page, nkv, hd = case["page"], case["nkv"], case["hd"]
    need = [-(-x // page) for x in kv]
    n_pages = sum(need) + 3
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(case["n"], max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = perm[at:at + m]
        at += m
    dtype = torch.float16 if case["dtype"] == "f16" else torch.float32
    rows = case["order"] == "rows"
    shape = (n_pages, page, nkv, hd) if rows else (n_pages, nkv, page, hd)
    pools = [torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype) for _ in range(2)]
    k, v = pools if rows else [p.transpose(1, 2) for p in pools]
    cu = [0]
    for x in t:
        cu.append(cu[-1] + x)
    return {"k": k, "v": v, "table": table, "cu": _ints(cu), "kv_len": _ints(kv), "T": cu[-1], "max_new": max(t),
            "max_kv": max(kv)}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    s = {"case": case}
    if case["op"] == "lora":
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = randn(M, K)
        if case["weight"] == "i8":
            s["w"] = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
            s["row_scales"] = (0.5 + torch.rand(N, generator=g, device="cuda")) * (0.03 / 127)
        else:
            s["w"] = (randn(N, K) * 0.02).half()
        dtype = torch.float16 if case["dtype"] == "f16" else torch.float32
        ranks = _ranks(case)
        s["A"] = [(randn(r, K) / math.sqrt(K)).to(dtype) for r in ranks]
        s["B"] = [(randn(N, r) * 0.02).to(dtype) for r in ranks]
        s["rank"] = _ints(ranks)
        s["scale"] = torch.tensor([2.0 * case["rank"] / r for r in ranks], dtype=torch.float32, device="cuda")
        # the rows of one request stand together: runs of equal ids, -1 where a request has no adapter
        runs = min(M, 16) if M > 16 else M
        ids = torch.randint(-1 if M > 1 else 0, case["adapters"], (runs,), generator=g, device="cuda")
        cut = torch.sort(torch.randint(0, M, (M - runs,), generator=g, device="cuda") % runs)[0]
        s["adapter"] = ids[torch.sort(torch.cat([torch.arange(runs, device="cuda"), cut]))[0]].to(torch.int32)
        return s
    s |= _paged(case, g)
    T, nh, nkv, hd = s["T"], case["nh"], case["nkv"], case["hd"]
    s["q"] = randn(T, nh, hd)
    if case["op"] == "rope":
        s["kn"], s["vn"] = randn(T, nkv, hd), randn(T, nkv, hd)
    return s


# ---------------------------------------------------------------------------------------------
# Rotary frequencies (64 bits): pair i turns by pos * f[i]; `m` scales cosine and sine
# ---------------------------------------------------------------------------------------------

THETA, FACTOR, ORIGINAL, LOW, HIGH, FAST, SLOW = 500000.0, 8.0, 8192, 1.0, 4.0, 32.0, 1.0


def _frequencies(rot, scaling):
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    f = THETA ** (-i / rot)
    if scaling == "linear":
        return f / FACTOR, 1.0
    if scaling == "bands":   # whole turns within the original context: kept, blended, divided
        turns = ORIGINAL * f / (2 * math.pi)
        keep = ((turns - LOW) / (HIGH - LOW)).clamp(0, 1)
        return f * keep + f / FACTOR * (1 - keep), 1.0
    if scaling == "yarn":    # a ramp over the pairs between the ones of FAST and of SLOW turns

        def pair(turns):
            return rot * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(THETA))

        lo, hi = max(math.floor(pair(FAST)), 0), min(math.ceil(pair(SLOW)), rot - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f / FACTOR * ramp + f * (1 - ramp), 0.1 * math.log(FACTOR) + 1.0
    return f, 1.0


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------


def _places(s):
    """Sequence and cache position of every new token."""
    cu = s["cu"].long()
    token = torch.arange(s["T"], device="cuda")
    seq = torch.searchsorted(cu[1:], token, right=True)
    return seq, s["kv_len"].long()[seq] - cu[1:][seq] + token


def _rotate(x, cos, sin, rot, pairs):
    c, n = cos[:, None, :], sin[:, None, :]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs == "interleaved" else (x[..., :rot // 2], x[..., rot // 2:rot])
    y, z = a * c - b * n, b * c + a * n
    turned = torch.stack([y, z], -1).flatten(-2) if pairs == "interleaved" else torch.cat([y, z], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rope(s):
    c = s["case"]
    seq, pos = _places(s)
    f, m = _frequencies(c["rot"], c["scaling"])
    angle = pos.double()[:, None] * f
    cos, sin = (angle.cos() * m).float(), (angle.sin() * m).float()
    page, row = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    s["k"][page, row] = _rotate(s["kn"], cos, sin, c["rot"], c["pairs"]).to(s["k"].dtype)
    s["v"][page, row] = s["vn"].to(s["v"].dtype)
    return {"q": _rotate(s["q"], cos, sin, c["rot"], c["pairs"]), "k": s["k"], "v": s["v"]}


def _plain_attention(s):
    c = s["case"]
    nh, nkv, hd, group = c["nh"], c["nkv"], c["hd"], c["nh"] // c["nkv"]
    seq, pos = _places(s)
    cu = s["cu"].long()
    at = torch.arange(s["T"], device="cuda") - cu[seq]
    q = torch.zeros(c["n"], s["max_new"], nh, hd, device="cuda")
    q[seq, at] = s["q"]
    where = torch.full((c["n"], s["max_new"]), -1, dtype=torch.long, device="cuda")
    where[seq, at] = pos
    key = torch.arange(s["max_kv"], device="cuda")
    page, row = s["table"].long()[:, key // c["page"]], (key % c["page"])[None, :]
    k, v = s["k"][page, row].float(), s["v"][page, row].float()                       # [n, kv, nkv, hd]
    q = q.view(c["n"], s["max_new"], nkv, group, hd).permute(0, 2, 3, 1, 4).reshape(c["n"], nkv, -1, hd)
    scores = (q @ k.permute(0, 2, 3, 1)) / math.sqrt(hd)                               # [n, nkv, group * new, kv]
    seen = key <= where[..., None]
    if c["window"]:
        seen &= key > where[..., None] - c["window"]
    scores.view(c["n"], nkv, group, s["max_new"], -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v.permute(0, 2, 1, 3)) / total.clamp_min(1e-38)
    out = out.view(c["n"], nkv, group, s["max_new"], hd).permute(0, 3, 1, 2, 4).reshape(c["n"], s["max_new"], nh, hd)
    lse = (top + total.log()).view(c["n"], nh, s["max_new"]).transpose(1, 2)
    return {"out": out[seq, at], "lse": lse[seq, at]}


def _plain_lora(s):
    w = s["w"].float() * s["row_scales"][:, None] if "row_scales" in s else s["w"].float()
    ids = torch.repeat_interleave(torch.arange(len(s["A"]), device="cuda"), s["rank"].long(),
                                  output_size=sum(_ranks(s["case"])))
    t = s["x"] @ torch.cat(s["A"]).float().T
    t = t * (s["adapter"].long()[:, None] == ids) * s["scale"][ids]
    return s["x"] @ w.T + t @ torch.cat(s["B"], 1).float().T


# ---------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------

_backend = None


def _handles(s):
    """The descriptors that a program keeps beside its buffers: addresses and sizes."""
    global _backend
    from ternative_b200 import CUDABackend, DeviceWeight, LoraTable, PagedBatch, PagedCache, RopeConfig, TVB_F16, TVB_I8_ROW

    c = s["case"]
    if _backend is None:
        _backend = CUDABackend()
    if c["op"] == "lora":
        s["table"] = LoraTable(s["A"], s["B"], s["rank"], s["scale"], max_rank=max(_ranks(c)))
        s["weight"] = (DeviceWeight(s["w"].data_ptr(), TVB_I8_ROW, s["row_scales"].data_ptr()) if "row_scales" in s
                       else DeviceWeight(s["w"].data_ptr(), TVB_F16))
    else:
        s["cache"] = PagedCache(s["k"], s["v"])
        s["batch"] = PagedBatch(s["cu"], s["kv_len"], s["table"], n_tokens=s["T"], max_new=s["max_new"], max_kv=s["max_kv"])
    if c["op"] == "rope":
        s["rope"] = RopeConfig(rot_dim=c["rot"], theta=THETA, pairs=c["pairs"], scaling=c["scaling"], factor=FACTOR,
                               original_len=ORIGINAL, low_turns=LOW, high_turns=HIGH, fast_turns=FAST, slow_turns=SLOW)
    s["handles"] = True


def _own(s):
    c = s["case"]
    if "handles" not in s:
        _handles(s)
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "lora":
        y = torch.empty(c["M"], c["N"], device="cuda")
        _backend.matmul_lora_d(y, s["x"], c["M"], c["K"], s["weight"], c["N"], s["table"], s["adapter"], stream=stream)
        return y
    if c["op"] == "rope":
        q = torch.empty_like(s["q"])
        _backend.rope_append_paged_d(q, s["q"], s["kn"], s["vn"], s["cache"], s["batch"], s["rope"], c["nh"], c["nkv"],
                                     c["hd"], stream=stream)
        return {"q": q, "k": s["k"], "v": s["v"]}
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["T"], c["nh"], device="cuda")
    _backend.attention_paged_d(out, s["q"], s["cache"], s["batch"], c["nh"], c["nkv"], c["hd"], 1 / math.sqrt(c["hd"]),
                               window=c["window"], lse=lse, stream=stream)
    return {"out": out, "lse": lse}


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "attention": _plain_attention, "lora": _plain_lora}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------


def work(case):
    size = 2 if case["dtype"] == "f16" else 4
    if case["op"] == "lora":
        M, K, N = case["M"], case["K"], case["N"]
        ranks = _ranks(case)
        used = sum(ranks[:max(1, min(len(ranks), M))])
        mean = sum(ranks) / len(ranks)
        wsize = N * K + 4 * N if case["weight"] == "i8" else 2 * N * K
        return {"bytes": wsize + size * used * (K + N) + 4 * M * (K + N), "flops": 2.0 * M * N * K + 2.0 * M * mean * (K + N)}
    new, kv = _lens(case)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if case["op"] == "rope":
        T = sum(new)
        return {"bytes": T * hd * (8 * nh + 2 * nkv * (4 + size)), "flops": 3.0 * T * (nh + nkv) * case["rot"]}
    w = case["window"] or max(kv)
    rows = sum(min(b, a + w - 1) for a, b in zip(new, kv))
    pairs = sum(min(w, b - j) for a, b in zip(new, kv) for j in range(a))
    return {"bytes": sum(new) * nh * (8 * hd + 4) + 2 * size * rows * nkv * hd, "flops": 4.0 * hd * nh * pairs}


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits, sequence by sequence and adapter by adapter
# ---------------------------------------------------------------------------------------------


def _exact_turn(x, angle, m, rot, pairs):
    """Pairs as complex numbers, each times m * exp(i * angle)."""
    x = x.double()
    head = x[..., :rot]
    z = head.unflatten(-1, (-1, 2)) if pairs == "interleaved" else head.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.full_like(angle, m), angle)[:, None, :]
    z = torch.view_as_real(z)
    z = z if pairs == "interleaved" else z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), x[..., rot:]], -1)


def _exact_angles(first, count, rot, scaling):
    f, m = [], 1.0
    for i in range(rot // 2):
        w = THETA ** (-2.0 * i / rot)
        if scaling == "linear":
            w /= FACTOR
        elif scaling == "bands":
            length = 2 * math.pi / w
            if length > ORIGINAL / LOW:
                w /= FACTOR
            elif length >= ORIGINAL / HIGH:
                b = (ORIGINAL / length - LOW) / (HIGH - LOW)
                w = (1 - b) * w / FACTOR + b * w
        elif scaling == "yarn":
            lo = max(0, math.floor(rot * math.log(ORIGINAL / (FAST * 2 * math.pi), THETA) / 2))
            hi = min(rot - 1, math.ceil(rot * math.log(ORIGINAL / (SLOW * 2 * math.pi), THETA) / 2))
            r = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            w = w / FACTOR * r + w * (1 - r)
            m = 1.0 + 0.1 * math.log(FACTOR)
        f.append(w)
    pos = torch.arange(first, first + count, dtype=torch.float64, device="cuda")
    return torch.outer(pos, torch.tensor(f, dtype=torch.float64, device="cuda")), m


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lora":
        x, w = s["x"].double(), s["w"].double()
        if "row_scales" in s:
            w *= s["row_scales"].double()[:, None]
        y = x @ w.T
        for i in range(case["adapters"]):
            at = torch.nonzero(s["adapter"] == i).flatten()
            y[at] += s["scale"][i].double() * ((x[at] @ s["A"][i].double().T) @ s["B"][i].double().T)
        return y
    new, kv = _lens(case)
    page, group = case["page"], case["nh"] // case["nkv"]
    rows = []
    for i in range(case["n"]):
        t = torch.arange(kv[i], device="cuda")
        rows.append((s["table"][i].long()[torch.div(t, page, rounding_mode="floor")], t % page))
    at = 0
    if case["op"] == "rope":
        q, k, v = [], s["k"].double(), s["v"].double()
        for i in range(case["n"]):
            angle, m = _exact_angles(kv[i] - new[i], new[i], case["rot"], case["scaling"])
            q.append(_exact_turn(s["q"][at:at + new[i]], angle, m, case["rot"], case["pairs"]))
            to = (rows[i][0][-new[i]:], rows[i][1][-new[i]:])
            k[to] = _exact_turn(s["kn"][at:at + new[i]], angle, m, case["rot"], case["pairs"])
            v[to] = s["vn"][at:at + new[i]].double()
            at += new[i]
        return {"q": torch.cat(q), "k": k, "v": v}
    out, lse = [], []
    for i in range(case["n"]):
        q = s["q"][at:at + new[i]].double()
        at += new[i]
        pos = torch.arange(kv[i] - new[i], kv[i], device="cuda")[:, None]
        t = torch.arange(kv[i], device="cuda")[None, :]
        hide = (t > pos) | (t <= pos - case["window"]) if case["window"] else t > pos
        o, e = [], []
        for h in range(case["nh"]):
            k, v = s["k"][rows[i][0], rows[i][1], h // group].double(), s["v"][rows[i][0], rows[i][1], h // group].double()
            z = (q[:, h] @ k.T / math.sqrt(case["hd"])).masked_fill(hide, -math.inf)
            e.append(torch.logsumexp(z, 1))
            o.append(torch.softmax(z, 1) @ v)
        out.append(torch.stack(o, 1))
        lse.append(torch.stack(e, 1))
    return {"out": torch.cat(out), "lse": torch.cat(lse)}
