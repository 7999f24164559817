"""The operators of a decoder block beside the LM head and the sampling step, as cases to be measured.

attention  one new token per sequence over a paged key-value cache (kept in 16 bits, or as 8- or 4-bit codes)
kv         new tokens' keys and values written into such a cache, and a range of it read back
linear     act(LayerNorm(x) W^T + b) + r

With `own` false, run() computes them from elementary torch operations in 32 bits; with `own` true, by the
framework's calls.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

HEADS, HEAD_DIM, WIDTH = 20, 64, 1280          # the T2S decoder: d 1280, MLP 5120, 8194 tokens
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _package():
    """The package directory is no identifier: it is imported under the name c4s."""
    if "c4s" not in sys.modules:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-confucius4-tts_b200")
        spec = importlib.util.spec_from_file_location("c4s", os.path.join(path, "__init__.py"),
                                                      submodule_search_locations=[path])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["c4s"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["c4s"]


def listed():
    att = {"op": "attention", "type": "bf16", "bits": 16, "group": 64, "q_heads": HEADS, "kv_heads": HEADS,
           "dim": HEAD_DIM, "page": 16, "layout": "head", "ragged": False, "window": 0}
    kv = {"op": "kv", "type": "bf16", "read": "bf16", "bits": 8, "group": 64, "kv_heads": HEADS, "dim": HEAD_DIM,
          "page": 16, "layout": "head", "batch": 64, "ragged": True, "before": 100, "step": False}
    lin = {"op": "linear", "type": "bf16", "out": "bf16", "norm": False, "bias": True, "act": "none",
           "residual": False}
    return [
        # one stream in the middle of an utterance: a call of a few microseconds, the latency of each layer's step
        {**att, "name": "attention-stream", "batch": 1, "len": 700},
        # 64 streams at different places, cache in 8-bit groups as the weights are
        {**att, "name": "attention-streams-q8", "batch": 64, "len": 1600, "bits": 8, "page": 32, "ragged": True},
        # a full batch of streams, cache in token-major pages
        {**att, "name": "attention-batch", "batch": 256, "len": 1500, "page": 64, "layout": "token", "ragged": True},
        # few long contexts whose key heads are shared by four query heads
        {**att, "name": "attention-long-shared", "batch": 2, "len": 50001, "type": "fp16", "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 128},
        # long contexts in 4-bit codes, the last 20000 positions visible, pages that no tile fits
        {**att, "name": "attention-long-q4", "batch": 4, "len": 30011, "bits": 4, "group": 32, "q_heads": 20,
         "kv_heads": 4, "dim": 96, "page": 100, "window": 20000},
        # what a decode step of 64 streams adds to one layer's cache: one token each
        {**kv, "name": "kv-step-q8", "tokens": 1, "before": 777, "step": True},
        # prompts of 64 streams into a 16-bit cache, and the dense copy that a prompt's own attention reads
        {**kv, "name": "kv-prompts", "tokens": 1500, "bits": 16, "before": 0},
        # long contexts into 8-bit codes, read back whole in 32 bits
        {**kv, "name": "kv-long-q8", "type": "fp16", "read": "fp32", "batch": 4, "tokens": 32768, "kv_heads": 8,
         "dim": 128, "page": 64, "layout": "token", "ragged": False, "before": 5},
        # one stream's query, key and value projection
        {**lin, "name": "linear-step", "rows": 1, "inner": WIDTH, "outer": 3 * WIDTH, "norm": True},
        # the second MLP product of 64 streams, added to the stream
        {**lin, "name": "linear-streams", "rows": 64, "inner": 4 * WIDTH, "outer": WIDTH, "residual": True},
        # the first MLP product of a full batch
        {**lin, "name": "linear-batch", "rows": 256, "inner": WIDTH, "outer": 4 * WIDTH, "type": "fp16",
         "out": "fp16", "norm": True, "act": "gelu"},
        # the same for the prompts' tokens
        {**lin, "name": "linear-prompts", "rows": 4099, "inner": WIDTH, "outer": 4 * WIDTH, "norm": True,
         "act": "gelu"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "kv", "linear", "linear"])
    typ = rng.choice(["bf16", "fp16"])
    if op == "linear":
        rows = _log(rng, 1, 4096)
        inner = 8 * _log(rng, 8, 1024)
        outer = _log(rng, 1, 8194)
        while rows * inner * outer > 4096 * WIDTH * 4 * WIDTH:
            rows = max(1, rows // 2)
        norm = rng.random() < 0.4
        return {"op": op, "type": typ, "out": typ if norm or rng.random() < 0.7 else "fp32", "norm": norm,
                "bias": rng.random() < 0.8, "act": rng.choice(["none", "none", "gelu", "gelu_erf", "silu", "relu"]),
                "residual": rng.random() < 0.5, "rows": rows, "inner": inner, "outer": outer}
    dim = rng.choice([64, 64, 96, 128])
    bits = rng.choice([16, 8, 4])
    group = 32 if dim == 96 or rng.random() < 0.3 else 64
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 16, 20])
    page = rng.choice([1, 8, 16, 16, 25, 32, 64, 100, 128, 256])
    layout = rng.choice(["head", "token"])
    if op == "kv":
        batch, tokens = _log(rng, 1, 200), _log(rng, 1, 8192)
        while batch * tokens * kv_heads * dim > 60_000_000:
            tokens = max(1, tokens // 2)
        return {"op": op, "type": typ, "read": rng.choice([typ, typ, "fp32"]), "bits": bits, "group": group,
                "kv_heads": kv_heads, "dim": dim, "page": page, "layout": layout, "batch": batch, "tokens": tokens,
                "ragged": rng.random() < 0.6, "before": rng.choice([0, 0, 7, 100, 1001]),
                "step": tokens == 1}
    shared = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
    batch, length = _log(rng, 1, 256), _log(rng, 1, 60000)
    while batch * length * kv_heads * dim * min(16, max(2, shared)) > 250_000_000:
        length, batch = max(1, length * 2 // 3), max(1, batch * 2 // 3)
    return {"op": op, "type": typ, "bits": bits, "group": group, "q_heads": kv_heads * shared, "kv_heads": kv_heads,
            "dim": dim, "page": page, "layout": layout, "batch": batch, "len": length,
            "ragged": rng.random() < 0.6, "window": rng.choice([0, 0, 0, 1 + length // 3])}


def _lengths(case, most):
    """The sequences' lengths, the same for every seed but for their order."""
    r = random.Random("%d %d" % (case["batch"], most))
    if not case["ragged"]:
        return [most] * case["batch"]
    n = [r.randint(0 if case["batch"] > 8 and case["op"] == "attention" else 1, most) for _ in range(case["batch"])]
    n[0] = most
    return n


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _cache_rows(n, case, gen, dev):
    """Rows of keys or values as projections give them: a few channels much larger than the rest."""
    x = torch.randn((*n, case["dim"]), generator=gen, device=dev, dtype=torch.float32)
    big = torch.ones(case["dim"], device=dev)
    big[3::29] = 6.0
    return x.mul_(big * 0.7)


def _encode(x, bits, group):
    """Codes (one a byte, or two), scales and biases of rows x in groups: the code is the step nearest to the value,
    the even one where two are as near. That border is looked for in 64 bits, a part of the rows at a time."""
    top = 2 ** bits - 1
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    q = torch.empty(g.shape, dtype=torch.uint8, device=x.device)
    for i in range(0, g.shape[0], 1 << 14):
        a = lo[i:i + (1 << 14)].double()
        t = (g[i:i + (1 << 14)].double() - a) * top / (hi[i:i + (1 << 14)].double() - a)
        q[i:i + (1 << 14)] = torch.round(t).nan_to_num_(0).to(torch.uint8)
    q = q.flatten(-2)
    if bits == 4:
        q = q[..., 0::2] | (q[..., 1::2] << 4)
    return q, torch.cat([(hi - lo) / torch.full_like(lo, top), lo], -1)


def _decode(q, sb, bits, group):
    """The 32-bit values that codes stand for."""
    if bits == 4:
        q = torch.stack([q & 15, q >> 4], -1).flatten(-2)
    g = q.float().unflatten(-1, (-1, group))
    return (g * sb[..., :1] + sb[..., 1:]).flatten(-2)


def _pool(case, pages, dev, typ):
    """An empty cache of `pages` pages: (codes or rows, scale and bias pairs or None), heads before tokens or after."""
    h, d, ps, bits = case["kv_heads"], case["dim"], case["page"], case["bits"]
    swap = case["layout"] == "token"

    def make(tail, dtype):
        x = torch.zeros((pages, ps, h, *tail) if swap else (pages, h, ps, *tail), dtype=dtype, device=dev)
        return x.transpose(1, 2) if swap else x
    if bits == 16:
        return make((d,), typ), None
    return make((d * bits // 8,), torch.uint8), make((d // case["group"], 2), torch.float32)


def _tables(case, caps, gen, dev):
    """Pages of the cache in no order, a row of them for each sequence, -1 behind its last."""
    need = [-(-c // case["page"]) for c in caps]
    total, width = sum(need), max(1, max(need))
    perm = torch.randperm(total + 3, generator=gen, device=dev).to(torch.int32)
    table = torch.full((len(caps), width), -1, dtype=torch.int32, device=dev)
    at = torch.arange(width, device=dev)[None, :] < torch.tensor(need, device=dev)[:, None]
    table[at] = perm[:total]
    return table, total + 3


def _handle(state):
    """The context that a program keeps."""
    if own:
        c4s = _package()
        state["ctx"] = c4s.SamplingContext(max_vocab=64, device=_device().index, max_rows=1)
        if "k" in state:
            state["cache"] = c4s.KVCache(state["k"], state["v"], state["k_sb"], state["v_sb"],
                                         bits=state["case"]["bits"])
        if state["op"] == "attention":
            state["work"] = state["ctx"].attention_workspace(state["q"].shape[0], state["q"].shape[1],
                                                             state["q"].shape[2])
    return state


def _inputs(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    typ = TYPES[case["type"]]

    def randn(*n):
        return torch.randn(n, generator=gen, device=dev, dtype=torch.float32)
    s = {"op": case["op"], "case": case}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        s["x"] = (randn(m, k) * 1.5 + 0.1).to(typ)
        s["w"] = (randn(n, k) / math.sqrt(k)).to(typ)
        s["bias"] = randn(n) * 0.1 if case["bias"] else None
        s["residual"] = (randn(m, n) * 2.0).to(TYPES[case["out"]]) if case["residual"] else None
        s["gamma"], s["beta"] = (1 + 0.1 * randn(k), 0.05 * randn(k)) if case["norm"] else (None, None)
        return s
    order = random.Random(seed)
    if case["op"] == "attention":
        lens = _lengths(case, case["len"])
        order.shuffle(lens)
        caps = lens
        table, pages = _tables(case, caps, gen, dev)
        pools = []
        for _ in "kv":
            rows, sb = _pool(case, pages, dev, typ)
            for a in range(0, pages, 512):      # a part at a time, for the memory that the 32-bit rows take
                x = _cache_rows(rows[a:a + 512].shape[:3], case, gen, dev).to(typ)
                if sb is None:
                    rows[a:a + 512] = x
                else:
                    rows[a:a + 512], sb[a:a + 512] = _encode(x.float(), case["bits"], case["group"])
            pools += [rows, sb]
        s["k"], s["k_sb"], s["v"], s["v_sb"] = pools
        n = torch.tensor(lens, dtype=torch.int32, device=dev)
        # what lies behind a sequence's end in its last page is whatever was there before
        last = table.gather(1, ((n.long() - 1).clamp(min=0) // case["page"])[:, None])[:, 0].long()
        used = (n.long() - 1) % case["page"]
        behind = torch.arange(case["page"], device=dev)[None, :] > used[:, None]
        behind &= (n > 0)[:, None]
        b, slot = behind.nonzero(as_tuple=True)
        for x in (s["k"], s["v"]) if case["bits"] == 16 else (s["k_sb"], s["v_sb"]):
            x[last[b], :, slot] = float("nan")
        s["table"], s["lens"] = table, n
        s["start"] = (n - case["window"]).clamp(min=0) if case["window"] else None
        # queries as the fused projection leaves them: a part of its rows
        b, hq, d = case["batch"], case["q_heads"], case["dim"]
        qkv = (randn(b, (hq + 2 * case["kv_heads"]) * d) * 0.8).to(typ)
        s["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        return s
    lens = _lengths(case, case["tokens"])
    order.shuffle(lens)
    before = [order.randint(0, case["before"]) if case["before"] else 0 for _ in lens]
    table, pages = _tables(case, [a + n for a, n in zip(before, lens)], gen, dev)
    s["k"], s["k_sb"] = _pool(case, pages, dev, typ)
    s["v"], s["v_sb"] = _pool(case, pages, dev, typ)
    s["table"] = table
    s["pos"] = torch.tensor(before, dtype=torch.int32, device=dev)
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    s["total"] = off[-1]
    s["tok_off"] = None if case["step"] else torch.tensor(off, dtype=torch.int64, device=dev)
    s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device=dev), torch.tensor(lens, device=dev))
    first = torch.tensor(off[:-1], device=dev)
    s["at"] = torch.arange(off[-1], device=dev) - first[s["seq"]] + s["pos"].long()[s["seq"]]
    h, d = case["kv_heads"], case["dim"]
    kv = torch.empty((off[-1], 3, h, d), dtype=typ, device=dev)     # the fused projection's rows
    kv[:, 1] = _cache_rows((off[-1], h), case, gen, dev)
    kv[:, 2] = _cache_rows((off[-1], h), case, gen, dev)
    s["new_k"], s["new_v"] = kv[:, 1], kv[:, 2]
    return s


def prepare(case, seed):
    return _handle(_inputs(case, seed))


def _act(y, act):
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if act == "gelu_erf":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "silu":
        return y / (1 + torch.exp(-y))
    return torch.relu(y) if act == "relu" else y


def _plain_linear(s):
    case, x = s["case"], s["x"].float()
    if case["norm"]:
        x = x - x.mean(-1, keepdim=True)
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * s["gamma"] + s["beta"]
    y = x @ s["w"].float().T
    y = _act(y if s["bias"] is None else y + s["bias"], case["act"])
    y = y if s["residual"] is None else y + s["residual"].float()
    return y.to(TYPES[case["out"]])


def _plain_attention(s):
    case, lens = s["case"], s["lens"].long()
    b, hq, d = s["q"].shape
    h = case["kv_heads"]
    pos = torch.arange(max(1, case["len"]), device=lens.device)
    page = s["table"].long()[:, (pos // case["page"]).clamp(max=s["table"].shape[1] - 1)].clamp(min=0)
    slot = (pos % case["page"]).expand(b, -1)
    seen = pos[None, :] < lens[:, None]
    if s["start"] is not None:
        seen &= pos[None, :] >= s["start"][:, None]

    def rows(x, sb):
        x = x[page, :, slot]                                        # batch, position, head, row
        x = x.float() if sb is None else _decode(x, sb[page, :, slot], case["bits"], case["group"])
        return torch.where(seen[:, :, None, None], x, 0.0).transpose(1, 2)
    q = s["q"].float().unflatten(1, (h, hq // h))
    a = q @ rows(s["k"], s["k_sb"]).transpose(2, 3) / math.sqrt(d)
    a = torch.where(seen[:, None, None, :], a, float("-inf"))
    top = a.amax(-1, keepdim=True)
    p = torch.exp(a - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = p @ rows(s["v"], s["v_sb"]) / torch.where(total == 0, 1.0, total)
    return o.flatten(1, 2).to(s["q"].dtype)


def _plain_kv(s):
    case, seq, at = s["case"], s["seq"], s["at"]
    page, slot = s["table"].long()[seq, at // case["page"]], at % case["page"]
    out = []
    for new, x, sb in ((s["new_k"], s["k"], s["k_sb"]), (s["new_v"], s["v"], s["v_sb"])):
        if sb is None:
            x[page, :, slot] = new
            got = x[page, :, slot].float()
        else:
            x[page, :, slot], sb[page, :, slot] = _encode(new.float(), case["bits"], case["group"])
            got = _decode(x[page, :, slot], sb[page, :, slot], case["bits"], case["group"])
        out.append(got.to(TYPES[case["read"]]))
    return out


def run(s):
    case = s["case"]
    if not own:
        return {"linear": _plain_linear, "attention": _plain_attention, "kv": _plain_kv}[s["op"]](s)
    ctx = s["ctx"]
    if s["op"] == "linear":
        return ctx.linear(s["x"], s["w"], bias=s["bias"], act=case["act"], residual=s["residual"],
                          layer_norm=case["norm"], gamma=s["gamma"], beta=s["beta"], eps=1e-5,
                          out_dtype=TYPES[case["out"]])
    if s["op"] == "attention":
        return ctx.paged_attention(s["q"], s["cache"], s["table"], s["lens"], start=s["start"], work=s["work"])
    ctx.kv_write(s["cache"], s["table"], s["new_k"], s["new_v"], s["pos"], tok_off=s["tok_off"])
    return list(ctx.kv_read(s["cache"], s["table"], s["pos"], tok_off=s["tok_off"], total=s["total"],
                            dtype=TYPES[case["read"]]))


def work(case):
    size = 4 if case.get("out") == "fp32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        return {"bytes": 2 * (m * k + n * k) + size * m * n * (2 if case["residual"] else 1) + 4 * n,
                "flops": 2 * m * k * n}
    d, h, bits = case["dim"], case["kv_heads"], case["bits"]
    row = 2 * d if bits == 16 else d * bits // 8 + 8 * (d // case["group"])
    if case["op"] == "attention":
        lens = [min(n, case["window"] or n) for n in _lengths(case, case["len"])]
        io = 4 * case["batch"] * case["q_heads"] * d
        return {"bytes": 2 * sum(lens) * h * row + io, "flops": 4 * sum(lens) * case["q_heads"] * d}
    rows = 2 * sum(_lengths(case, case["tokens"])) * h
    return {"bytes": rows * (2 * d + 2 * row + d * (4 if case["read"] == "fp32" else 2)), "flops": 6 * rows * d}


def exact(case, seed):
    s = _inputs(case, seed)
    f64 = torch.float64
    if case["op"] == "linear":
        outs = []
        w = s["w"].to(f64)
        for i in range(0, case["rows"], 1024):
            x = s["x"][i:i + 1024].to(f64)
            if case["norm"]:
                var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
                x = (x - mean) * torch.rsqrt(var + 1e-5)
                x = x * s["gamma"].to(f64) + s["beta"].to(f64)
            y = torch.einsum("mk,nk->mn", x, w)
            if s["bias"] is not None:
                y += s["bias"].to(f64)
            if case["act"] == "gelu":
                y = torch.nn.functional.gelu(y, approximate="tanh")
            elif case["act"] == "gelu_erf":
                y = torch.nn.functional.gelu(y)
            elif case["act"] == "silu":
                y = y * torch.sigmoid(y)
            elif case["act"] == "relu":
                y = y.clamp(min=0)
            if s["residual"] is not None:
                y += s["residual"][i:i + 1024].to(f64)
            outs.append(y)
        return torch.cat(outs)
    ps, bits, g = case["page"], case["bits"], case["group"]
    if case["op"] == "kv":
        def values(x):
            x = x.to(f64)
            if bits == 16:
                return x
            x = x.reshape(*x.shape[:-1], -1, g)
            low = x.min(-1, keepdim=True).values
            span = (x.max(-1, keepdim=True).values - low).clamp(min=1e-300)
            code = torch.round((x - low) * (2 ** bits - 1) / span)
            return (code * span / (2 ** bits - 1) + low).flatten(-2)
        return [values(s["new_k"]), values(s["new_v"])]
    lens = s["lens"].tolist()
    if sum(lens) > 400_000:
        return None
    shared = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=f64, device=s["q"].device)

    def sequence(x, sb, pages, a, n):
        x = x[pages].transpose(1, 2).flatten(0, 1)[a:n]
        if sb is None:
            return x.to(f64)
        p = sb[pages].transpose(1, 2).flatten(0, 1)[a:n].to(f64)
        if bits == 4:
            x = torch.stack([x % 16, x // 16], dim=-1).flatten(-2)
        p = p.repeat_interleave(g, dim=2)
        return x.to(f64) * p[..., 0] + p[..., 1]
    for b, n in enumerate(lens):
        a = max(0, n - case["window"]) if case["window"] else 0
        if a >= n:
            continue
        pages = s["table"][b, :-(-n // ps)].long()
        k, v = sequence(s["k"], s["k_sb"], pages, a, n), sequence(s["v"], s["v_sb"], pages, a, n)
        q = s["q"][b].to(f64).reshape(case["kv_heads"], shared, -1)
        a64 = torch.einsum("hgd,nhd->hgn", q, k) * case["dim"] ** -0.5
        out[b] = torch.einsum("hgn,nhd->hgd", torch.softmax(a64, dim=-1), v).flatten(0, 1)
    return out
