"""Timed cases of the 8-bit key/value cache operators: append, single-token attention, prompt attention, eviction.

With `own` false each case runs in its plain form, elementary torch operations in 32 bits (64 where a value stands next to a
rounding border); with `own` true the same case runs through the package's KvCache8.  `exact` gives the outputs in 64 bits.

The cache holds a K and a V vector of D numbers per position and K/V head.  Sixteen consecutive positions of one head form a
block with one scale for K and one for V:
    amax  = largest magnitude in the block's rows          scale = f32(amax / 127)     inverse = f32(127 / amax)
    code  = rint(x * inverse), in [-127, 127]              value = f32(code * scale)
The rows of the last, still open block are kept in 32 bits beside it, so that a later append rounds them once, not twice.
"""
import math

import torch

own = False
BLOCK = 16
_pkg = None
_ctx = {}


def listed():
    return [
        # the smallest call of a decode loop: one token joins a nearly full 512-position cache of a 7B layer
        dict(name="append-one-7b", op="append", heads=32, kv_heads=32, dim=128, pos=511, n=1),
        # a long prompt enters the cache at once, behind a few tokens that are already there; an odd length
        dict(name="append-long-odd", op="append", heads=32, kv_heads=32, dim=128, pos=5, n=16381),
        # the small test model at a short context: nothing but latency
        dict(name="decode-tiny-64", op="decode", heads=8, kv_heads=8, dim=64, T=64, mass=False),
        # one decode step of a 7B layer at its full context of 512, attention weights counted for a later eviction
        dict(name="decode-7b-512-mass", op="decode", heads=32, kv_heads=32, dim=128, T=512, mass=True),
        # one decode step of a 13B layer at 2047 positions, an odd length
        dict(name="decode-13b-2047", op="decode", heads=40, kv_heads=40, dim=128, T=2047, mass=False),
        # a long conversation, a K/V head for every query head, weights counted
        dict(name="decode-65535-mass", op="decode", heads=32, kv_heads=32, dim=128, T=65535, mass=True),
        # a very long context with eight query heads on each K/V head
        dict(name="decode-131071-grouped", op="decode", heads=64, kv_heads=8, dim=128, T=131071, mass=False),
        # a short follow-up turn over a long cache: few rows, a long axis
        dict(name="prefill-17-over-8192", op="prefill", heads=32, kv_heads=8, dim=128, past=8192, n=17, mass=False),
        # a 512-token prompt of a 7B layer from the start, weights counted
        dict(name="prefill-512-7b-mass", op="prefill", heads=32, kv_heads=32, dim=128, past=0, n=512, mass=True),
        # a large chunk of a long prompt behind three earlier ones, grouped heads
        dict(name="prefill-2048-over-6144", op="prefill", heads=32, kv_heads=8, dim=128, past=6144, n=2048, mass=False),
        # a 512-position cache is full: half of it goes, the first four and the last 32 positions stay
        dict(name="evict-7b-512-to-256", op="evict", heads=32, kv_heads=32, dim=128, T=512, keep=256, sink=4, recent=32),
        # a long prompt's cache shrinks to a small budget before decoding
        dict(name="evict-32768-to-4099", op="evict", heads=32, kv_heads=32, dim=128, T=32768, keep=4099, sink=4, recent=512),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dim = rng.choice([64, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32, 32, 40])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
    while kv_heads * group > 64:
        group = rng.choice([1, 2, 3, 4, 5, 8, 16])
        kv_heads = rng.choice([1, 2, 4, 8, 16, 32, 40])
    case = dict(op=rng.choice(["append", "decode", "decode", "prefill", "prefill", "evict"]), heads=kv_heads * group, kv_heads=kv_heads, dim=dim)
    width = kv_heads * dim
    if case["op"] == "append":
        n = 1 if rng.random() < 0.3 else _log(rng, 2, 16381 * 4096 // max(4096, width))
        return case | dict(pos=rng.randrange(0, 2048), n=n)
    if case["op"] == "decode":
        return case | dict(T=_log(rng, 1, min(131071, 65535 * 4096 // width)), mass=rng.random() < 0.5)
    if case["op"] == "prefill":
        n = _log(rng, 1, 2048)
        total = 32 * 2048 * 7168 // case["heads"]  # scores of the largest listed case, over the heads
        past = 0 if rng.random() < 0.3 else _log(rng, 1, max(1, min(16384, total // n - n)))
        return case | dict(past=past, n=n, mass=rng.random() < 0.3)
    T = _log(rng, 2, min(65536, 32768 * 4096 // width))
    keep = max(1, min(int(T * rng.uniform(0.1, 1.0)), 2 * 4099 * 4096 // width // 2))
    sink = min(keep, rng.choice([0, 1, 4, 16]))
    return case | dict(T=T, keep=keep, sink=sink, recent=int((keep - sink) * rng.random() * 0.5))


def work(case):
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":  # rows in, codes and scales out, and the touched rows' values given back
        rows = case["pos"] % BLOCK + case["n"]
        return {"bytes": 2 * g * d * (4 * case["n"] + 5 * rows) + 8 * g * -(-rows // BLOCK), "flops": 4 * g * d * rows}
    if case["op"] == "decode":
        T = case["T"]
        return {"bytes": 2 * g * T * d + 8 * g * -(-T // BLOCK) + 8 * h * d + (8 * g * T if case["mass"] else 0), "flops": 4 * h * T * d}
    if case["op"] == "prefill":
        n, T = case["n"], case["past"] + case["n"]
        pairs = n * case["past"] + n * (n + 1) // 2
        return {"bytes": 2 * g * T * d + 8 * g * -(-T // BLOCK) + 8 * n * h * d + (8 * g * T if case["mass"] else 0), "flops": 4 * h * pairs * d}
    T, keep = case["T"], case["keep"]  # weights and kept rows in; codes, scales, weights, indices and the kept rows' values out
    return {"bytes": 4 * g * T + 2 * g * keep * d * (1 + 5) + 8 * g * (-(-T // BLOCK) + -(-keep // BLOCK)) + 8 * g * keep, "flops": 4 * g * keep * d}


def _inputs(case, seed):
    """Keys with a few strong channels, values and queries around one, weights with a heavy tail: what a trained layer shows."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    rows = {"append": lambda: case["pos"] % BLOCK + case["n"], "decode": lambda: case["T"], "prefill": lambda: case["past"] + case["n"], "evict": lambda: case["T"]}[case["op"]]()
    x = {"k": normal(rows, g, d) * (0.4 + 0.6 * normal(g, d).square()), "v": normal(rows, g, d) * (0.3 + 0.4 * normal(g, 1).abs())}
    if case["op"] == "decode":
        x["q"] = normal(h, d)
    if case["op"] == "prefill":
        x["q"] = normal(case["n"], h, d)
    if case["op"] == "evict" or case.get("mass"):
        x["mass"] = normal(g, rows).mul(1.5).exp()
    return x


def _quantise(x):
    """Codes and scales of rows [rows, kv_heads, dim], the last block padded with zero rows."""
    rows, g, d = x.shape
    x = torch.cat([x, x.new_zeros(-rows % BLOCK, g, d)]).reshape(-1, BLOCK, g, d)
    amax = x.abs().amax((1, 3))
    top = torch.full_like(amax, 127)  # a tensor: a quotient with a plain number is a product with its rounded reciprocal
    scale = amax / top
    inverse = torch.where(amax > 0, top / amax, torch.zeros_like(amax))
    codes = torch.round(x.double() * inverse.double()[:, None, :, None]).to(torch.int8)  # 64 bits: next to a border
    return codes.reshape(-1, g, d)[:rows], scale


def _values(codes, scale):
    rows = codes.shape[0]
    return codes.float() * scale.repeat_interleave(BLOCK, 0)[:rows, :, None]


def _cache(case, capacity):
    return _pkg.KvCache8(_ctx[torch.cuda.current_device()], capacity, case["heads"], case["kv_heads"], case["dim"])


def _fill(case, x, rows):
    cache = _cache(case, -(-x["k"].shape[0] // 64) * 64 if case["op"] != "append" else case["pos"] + case["n"])
    first = case["pos"] - case["pos"] % BLOCK if case["op"] == "append" else 0
    if rows:
        cache.append(x["k"].data_ptr(), x["v"].data_ptr(), first, rows)
    return cache


def prepare(case, seed):
    global _pkg
    x = _inputs(case, seed)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["op"] == "append":  # the open block's earlier rows are in the cache, the new ones in hand
        before = case["pos"] % BLOCK
        s |= {"k": x["k"][before:].contiguous(), "v": x["v"][before:].contiguous(), "rows": before + case["n"]}
        if not own:
            s |= {"k_open": x["k"][:before].clone(), "v_open": x["v"][:before].clone()}
    else:
        s |= {name: x[name] for name in ("q", "mass") if name in x}
        if not own:
            s["k"], s["k_scale"] = _quantise(x["k"])
            s["v"], s["v_scale"] = _quantise(x["v"])
    if own:
        if _pkg is None:
            import __graft_entry__
            _pkg = __graft_entry__.load_package()
        device = torch.cuda.current_device()
        if device not in _ctx:
            _ctx[device] = _pkg.Context(device, stream=torch.cuda.current_stream().cuda_stream)
        s["cache"] = _fill(case, x, {"append": case.get("pos", 0) % BLOCK}.get(case["op"], x["k"].shape[0]))
        new = lambda *shape, dtype=torch.float32: torch.empty(*shape, device="cuda", dtype=dtype)  # noqa: E731
        if case["op"] == "append":
            s |= {"k_out": new(s["rows"], g, d), "v_out": new(s["rows"], g, d)}
        elif case["op"] == "evict":
            keep = case["keep"]
            wide = torch.zeros(g, s["cache"].n_ctx, device="cuda")
            wide[:, :case["T"]] = s["mass"]
            s |= {"to": _cache(case, keep), "mass": wide, "mass_out": new(g, keep), "kept": new(g, keep, dtype=torch.int32), "k_out": new(keep, g, d), "v_out": new(keep, g, d)}
        else:
            s["out"] = torch.empty_like(s["q"])
            if case["mass"]:
                wide = torch.zeros(g, s["cache"].n_ctx, device="cuda")
                wide[:, :s["mass"].shape[1]] = s["mass"]
                s |= {"mass": wide, "mass_out": torch.zeros_like(wide)}
    return s


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    return {"append": _plain_append, "decode": _plain_attention, "prefill": _plain_attention, "evict": _plain_evict}[case["op"]](s, case)


def _run_own(s, case):
    cache = s["cache"]
    if case["op"] == "append":
        cache.append(s["k"].data_ptr(), s["v"].data_ptr(), case["pos"], case["n"])
        cache.read(case["pos"] - case["pos"] % BLOCK, s["rows"], s["k_out"].data_ptr(), s["v_out"].data_ptr())
        return {"k": s["k_out"], "v": s["v_out"]}
    if case["op"] == "evict":
        cache.evict(s["to"], case["T"], case["keep"], case["sink"], case["recent"], s["mass"].data_ptr(), s["mass_out"].data_ptr(), s["kept"].data_ptr())
        s["to"].read(0, case["keep"], s["k_out"].data_ptr(), s["v_out"].data_ptr())
        return {"kept": s["kept"], "mass": s["mass_out"], "k": s["k_out"], "v": s["v_out"]}
    mass = {"mass_in": s["mass"].data_ptr(), "mass_out": s["mass_out"].data_ptr()} if case["mass"] else {}
    if case["op"] == "decode":
        T = case["T"]
        cache.attn_decode(s["q"].data_ptr(), T, s["out"].data_ptr(), **mass)
    else:
        T = case["past"] + case["n"]
        cache.attn_prefill(s["q"].data_ptr(), case["past"], case["n"], s["out"].data_ptr(), **mass)
    return {"out": s["out"], "mass": s["mass_out"][:, :T]} if mass else {"out": s["out"]}


def _plain_append(s, case):
    k = _values(*_quantise(torch.cat([s["k_open"], s["k"]])))
    return {"k": k, "v": _values(*_quantise(torch.cat([s["v_open"], s["v"]])))}


def _plain_attention(s, case):
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    k, v = _values(s["k"], s["k_scale"]).permute(1, 2, 0), _values(s["v"], s["v_scale"]).permute(1, 0, 2)  # [g, d, T], [g, T, d]
    T = k.shape[2]
    q = s["q"].reshape(-1, g, h // g, d).permute(1, 0, 2, 3)  # [g, n, group, d]
    n = q.shape[1]
    scores = torch.matmul(q.reshape(g, -1, d), k).reshape(g, n, h // g, T) / math.sqrt(d)
    seen = torch.arange(T, device="cuda") <= torch.arange(T - n, T, device="cuda")[:, None]
    scores = scores.masked_fill(~seen[:, None, :], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(g, -1, T), v).reshape(g, n, h // g, d).permute(1, 0, 2, 3).reshape(s["q"].shape)
    return {"out": out, "mass": s["mass"] + p.sum((1, 2))} if case["mass"] else {"out": out}


def _plain_evict(s, case):
    T, keep, sink, recent = case["T"], case["keep"], case["sink"], case["recent"]
    g = case["kv_heads"]
    order = torch.sort(s["mass"][:, sink:T - recent], dim=1, descending=True, stable=True).indices[:, :keep - sink - recent] + sink
    always = torch.cat([torch.arange(sink, device="cuda"), torch.arange(T - recent, T, device="cuda")]).expand(g, -1)
    kept = torch.cat([always, order], 1).sort(1).values  # [g, keep]
    whole = torch.cat([kept, kept.new_full((g, -keep % BLOCK), -1)], 1).reshape(g, -1, BLOCK)
    whole = (whole[..., 0] % BLOCK == 0) & (whole[..., -1] == whole[..., 0] + BLOCK - 1)  # blocks that stay together keep their codes

    def moved(codes, scale):
        at = kept.T[:, :, None].expand(-1, -1, codes.shape[2])
        again, scale2 = _quantise(torch.gather(_values(codes, scale), 0, at))
        old = torch.gather(codes, 0, at).float() * torch.gather(scale, 0, kept.T // BLOCK)[:, :, None]
        return torch.where(whole.T.repeat_interleave(BLOCK, 0)[:keep, :, None], old, _values(again, scale2))

    return {"kept": kept.int(), "mass": torch.gather(s["mass"], 1, kept), "k": moved(s["k"], s["k_scale"]), "v": moved(s["v"], s["v_scale"])}


def _exact_block_codes(x64):
    """[blocks, BLOCK, g, d] in 64 bits -> codes and scales; the two factors are 32-bit numbers by definition."""
    amax = x64.abs().amax(3, keepdim=True).amax(1, keepdim=True)
    top = torch.full_like(amax, 127)
    scale = (amax / top).float().double()
    inverse = torch.where(amax > 0, top / torch.where(amax > 0, amax, top), torch.zeros_like(amax)).float().double()
    return torch.round(x64 * inverse), scale


def _exact_rows(x):
    """The values that rows [rows, g, d] stand for in the cache, their codes and their scales, in 64 bits."""
    rows, g, d = x.shape
    full = torch.zeros(-(-rows // BLOCK) * BLOCK, g, d, dtype=torch.float64, device=x.device)
    full[:rows] = x.double()
    codes, scale = _exact_block_codes(full.view(-1, BLOCK, g, d))
    scale = scale.expand(-1, BLOCK, g, 1).reshape(-1, g, 1)[:rows]
    codes = codes.reshape(-1, g, d)[:rows]
    return codes * scale, codes, scale


def exact(case, seed):
    x = _inputs(case, seed)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        return {"k": _exact_rows(x["k"])[0], "v": _exact_rows(x["v"])[0]}
    if case["op"] == "evict":
        return _exact_evict(case, x)
    k, v = _exact_rows(x["k"])[0], _exact_rows(x["v"])[0]
    rows, group = k.shape[0], h // g
    q = x["q"].double().reshape(-1, h, d)
    n = q.shape[0]
    out = torch.empty(n, h, d, dtype=torch.float64, device="cuda")
    mass = x["mass"].double() if case["mass"] else None
    limit = torch.arange(rows - n, rows, device="cuda")
    for head in range(h):
        s = q[:, head] @ k[:, head // group].T * d ** -0.5
        p = torch.softmax(torch.where(torch.arange(rows, device="cuda")[None, :] > limit[:, None], -math.inf, s), -1)
        out[:, head] = p @ v[:, head // group]
        if case["mass"]:
            mass[head // group] += p.sum(0)
    out = out.reshape(x["q"].shape)
    return {"out": out, "mass": mass} if case["mass"] else {"out": out}


def _exact_evict(case, x):
    T, keep, sink, recent, g, d = case["T"], case["keep"], case["sink"], case["recent"], case["kv_heads"], case["dim"]
    out = {"kept": torch.empty(g, keep, dtype=torch.int32, device="cuda"), "mass": torch.empty(g, keep, dtype=torch.float64, device="cuda")}
    for name in ("k", "v"):
        out[name] = torch.empty(keep, g, d, dtype=torch.float64, device="cuda")
    whole = {name: _exact_rows(x[name]) for name in ("k", "v")}
    for head in range(g):
        stays = torch.zeros(T, dtype=torch.bool, device="cuda")
        stays[:sink] = True
        stays[T - recent:] = True
        middle = x["mass"][head].double().clone()
        middle[stays] = -1.0
        stays[torch.argsort(-middle, stable=True)[:keep - sink - recent]] = True
        at = stays.nonzero()[:, 0]
        out["kept"][head], out["mass"][head] = at.int(), x["mass"][head].double()[at]
        run16 = torch.cat([at, at.new_full((-keep % BLOCK,), -1)]).view(-1, BLOCK)
        together = ((run16[:, 0] % BLOCK == 0) & (run16[:, 15] - run16[:, 0] == 15)).repeat_interleave(BLOCK)[:keep, None]
        for name in ("k", "v"):
            value, codes, scale = (t[at, head] for t in whole[name])
            stored = value.float().double()[:, None, :]  # what the cache stands for is a 32-bit number by definition
            out[name][:, head] = torch.where(together, codes * scale, _exact_rows(stored)[0][:, 0])
    return out
