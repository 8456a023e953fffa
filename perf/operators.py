"""Timed cases of the 4-bit operators: a key/value cache held in 4 bits (written,
read back and attended to) and the few-row linear with 4-bit weights.

Four kinds of call, each through ltx_amd.runtime:

  write      new rows of k and v are quantised into a paged cache; what the cache
             then holds of them is read back (the values the 4 bits stand for)
  read       rows of the cache come back in 16 bits
  attention  rows of q attend to the cache: single tokens of many sequences, the
             tokens of a latent frame of a streamed video, ragged prefills
  linear     y = a . (q s)^T (+ bias, GELU), 4-bit weights with a scale per 128

The cache's form: per row and head 32 consecutive values share a power of two
2^e and are held as e2m1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives). e is the one that takes the group's largest magnitude to at most 7
and above 3.5 (7 .. 6 rounds down), limited to what the 16-bit type holds; values
round to the nearest, ties to the even code.

Head and width sizes are the block's (32 heads x 128, d_model 4096, FFN 16,384),
with 32, 8 or 4 heads in the cache; lengths go from one token to the benchmark's
28,672. A case is a dict of plain values; listed() names the fixed ones, draw()
gives others of the same ranges.
"""
import math
import os
import sys

import torch

own = False

HD, PAGE, GROUP = 128, 64, 32  # head size, tokens a page, values that share a scale in the cache
WGROUP = 128                   # weights that share a scale in the linear
D, H, FF = 4096, 32, 16384
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EXPONENTS = {"f16": (-23, 13), "bf16": (-125, 125)}  # 0.5 * 2^e and 6 * 2^e are finite, non-zero numbers of the type
PROJ = ((4096, 4096), (8192, 4096), (12288, 4096), (16384, 4096), (4096, 16384))  # (n, k) of the block's projections


def listed():
    return [
        # one token of 32 sequences appended, a serving step; k and v are slices of fused q|k|v rows
        dict(name="write_bf16_step32", kind="write", mode="bf16", kv_heads=8, seqs=32, new=1, keys=8192, ragged=True),
        # the first frames of a clip enter the cache: 13 latent frames of 32 x 64
        dict(name="write_f16_t26624", kind="write", mode="f16", kv_heads=32, seqs=1, new=26624, keys=26624,
             ragged=False),
        # the last 250 tokens or so of five sequences, for a recomputation in 16 bits
        dict(name="read_bf16_ragged", kind="read", mode="bf16", kv_heads=8, seqs=5, new=251, keys=2970, ragged=True),
        # a whole clip's keys and values back in 16 bits
        dict(name="read_f16_t28672", kind="read", mode="f16", kv_heads=32, seqs=1, new=28672, keys=28672,
             ragged=False),
        # the smallest call: one token, one short sequence, as many cached heads as query heads
        dict(name="attention_f16_step1", kind="attention", mode="f16", heads=32, kv_heads=32, seqs=1, new=1, keys=1000,
             ragged=False, causal=True, gate=False),
        # a serving step: 32 ragged sequences, four query heads a cached head
        dict(name="attention_bf16_step32", kind="attention", mode="bf16", heads=32, kv_heads=8, seqs=32, new=1,
             keys=8192, ragged=True, causal=True, gate=False),
        # four long sequences, a token each, the block's own heads and gate
        dict(name="attention_f16_step4_long", kind="attention", mode="f16", heads=32, kv_heads=32, seqs=4, new=1,
             keys=28672, ragged=False, causal=True, gate=True),
        # a streamed video's next latent frame (32 x 64 tokens) against the 13 before it and itself
        dict(name="attention_f16_frame", kind="attention", mode="f16", heads=32, kv_heads=32, seqs=1, new=2048,
             keys=28672, ragged=False, causal=False, gate=True),
        # ragged prompts of three sequences enter at once
        dict(name="attention_bf16_prefill", kind="attention", mode="bf16", heads=32, kv_heads=8, seqs=3, new=2970,
             keys=2970, ragged=True, causal=True, gate=False),
        # one token's out projection
        dict(name="linear_f16_m1", kind="linear", mode="f16", m=1, n=4096, k=4096, scale="f16", bias=True, gelu=False,
             out_f32=False),
        # FFN up with GELU for a batch of single tokens, the blobs' f32 scales
        dict(name="linear_bf16_m32", kind="linear", mode="bf16", m=32, n=16384, k=4096, scale="f32", bias=False,
             gelu=True, out_f32=False),
        # FFN down in the parity mode, an odd count of rows
        dict(name="linear_f32_m5", kind="linear", mode="f32", m=5, n=4096, k=16384, scale="f32", bias=True, gelu=False,
             out_f32=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "attention", "attention", "attention", "linear", "linear"])
    mode = rng.choice(["f16", "bf16"])
    if kind == "linear":
        mode = rng.choice(["f16", "bf16", "f32"])
        n, k = rng.choice(PROJ)
        return dict(kind=kind, mode=mode, m=_log(rng, 1, 256), n=n, k=k, scale=rng.choice(["f16", "f32"]),
                    bias=rng.random() < 0.5, gelu=n == FF, out_f32=mode == "f32" or rng.random() < 0.3)
    kv_heads = rng.choice([32, 8, 4])
    if kind != "attention":
        seqs = _log(rng, 1, 32)
        new = _log(rng, 1, 26624 // seqs)
        return dict(kind=kind, mode=mode, kv_heads=kv_heads, seqs=seqs, new=new, keys=new + _log(rng, 1, 2048),
                    ragged=rng.random() < 0.5)
    seqs = _log(rng, 1, 64)
    keys = _log(rng, 1, min(28672, 114688 // seqs))
    new = 1 if rng.random() < 0.5 else min(keys, _log(rng, 1, max(1, 2048 // seqs)))
    return dict(kind=kind, mode=mode, heads=H, kv_heads=kv_heads, seqs=seqs, new=new, keys=keys,
                ragged=rng.random() < 0.5, causal=rng.random() < 0.7, gate=rng.random() < 0.3)


# ---- the shape of a batch ----------------------------------------------------

def _lengths(case):
    """New rows and keys of each sequence; ragged ones go down from the case's."""
    n, top, keys = case["seqs"], case["new"], case["keys"]
    if not case["ragged"]:
        return [top] * n, [keys] * n
    new = [max(1, top - top * b // (2 * n) - (b if top > n else 0)) for b in range(n)]
    return new, [max(new[b], keys - keys * b // n - (3 * b if keys > 4 * n else 0)) for b in range(n)]


def _pairs(case):
    """(row, key) pairs that the mask leaves."""
    return sum(n * L - (n * (n - 1) // 2 if case["causal"] else 0) for n, L in zip(*_lengths(case)))


def work(case):
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        a = 4 if case["mode"] == "f32" else 2
        s = 4 if case["scale"] == "f32" else 2
        return {"bytes": m * k * a + n * k // 2 + n * (k // WGROUP) * s + (4 * n if case["bias"] else 0)
                + m * n * (4 if case["out_f32"] else 2), "flops": 2 * m * n * k}
    new, keys = _lengths(case)
    row = case["kv_heads"] * (HD // 2 + HD // GROUP) * 2  # k and v of one cached token
    full = case["kv_heads"] * HD * 2 * 2
    if case["kind"] == "write":  # read, held, read back, returned
        return {"bytes": sum(new) * (2 * full + 2 * row), "flops": 0}
    if case["kind"] == "read":
        return {"bytes": sum(new) * (full + row), "flops": 0}
    width = case["heads"] * HD
    return {"bytes": sum(keys) * row + sum(new) * (2 * width * 2 + (4 * case["heads"] if case["gate"] else 0)),
            "flops": 4 * HD * case["heads"] * _pairs(case)}


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + 29)
    return g


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _weights(case, g):
    """Student-t(3) x 0.02 weights in -7 .. 7, two a byte (the even one low), a scale per 128 along k."""
    n, k = case["n"], case["k"]
    z = torch.randn(n, k // WGROUP, WGROUP, generator=g, device="cuda")
    chi = torch.zeros_like(z)
    for _ in range(3):
        chi += torch.randn(z.shape, generator=g, device="cuda").square_()
    w = 0.02 * z / torch.sqrt(chi / 3)
    s = (w.abs().amax(-1) / 7).clamp_min(1e-8)
    s = s.half() if case["scale"] == "f16" else s
    q = torch.round(w / s.float()[..., None]).clamp_(-8, 7).to(torch.int32).reshape(n, k // 2, 2) & 15
    return (q[..., 0] | (q[..., 1] << 4)).to(torch.uint8), s


def _kv(case, g, rows):
    """k with channels of unlike size, as norm weights leave it, and v, in the type."""
    h, dt = case["kv_heads"], DTYPES[case["mode"]]
    k = _normal(g, rows, h, HD) * torch.exp(_normal(g, h, HD, std=0.5))
    v = _normal(g, rows, h, HD, std=0.7)
    return k.to(dt).reshape(rows, h * HD), v.to(dt).reshape(rows, h * HD)


def _starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def _batch(case, g):
    """Row starts, lengths and the page table of the sequences: pages lie anywhere in the pool."""
    new, keys = _lengths(case)
    width = -(-max(keys) // PAGE)
    order = torch.randperm(len(keys) * width + 3, generator=g, device="cuda").to(torch.int32)
    ints = dict(dtype=torch.int32, device="cuda")
    return dict(new=new, keys=keys, pool=len(keys) * width + 3, starts=torch.tensor(_starts(new), **ints),
                lengths=torch.tensor(keys, **ints), pages=order[:len(keys) * width].reshape(len(keys), width).contiguous())


def _inputs(case, seed):
    """What both forms and the definition start from."""
    g = _gen(seed)
    dt = DTYPES[case["mode"]]
    if case["kind"] == "linear":
        q, s = _weights(case, g)
        return dict(a=_normal(g, case["m"], case["k"]).to(dt), q=q, s=s,
                    bias=_normal(g, case["n"], std=0.02) if case["bias"] else None)
    b = _batch(case, g)
    rows = sum(b["new"])
    if case["kind"] == "write":
        k, v = _kv(case, g, rows)
        fused = torch.cat([torch.zeros(rows, H * HD, dtype=dt, device="cuda"), k, v], 1)  # q | k | v
        b["k"], b["v"] = fused[:, H * HD:H * HD + k.shape[1]], fused[:, H * HD + k.shape[1]:]
        return b
    # what the cache holds before the call: every key of every sequence
    b["k"], b["v"] = _kv(case, g, sum(b["keys"]))
    if case["kind"] == "attention":
        width = case["heads"] * HD
        fused = _normal(g, rows, width + 2 * case["kv_heads"] * HD).to(dt)
        b["q"] = fused[:, :width]
        b["gate"] = _normal(g, rows, case["heads"]) if case["gate"] else None
    return b


_contexts = []


def _context():
    """The program's context."""
    if not _contexts:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ltx-zml_amd"))
        from ltx_amd import runtime as rt
        _contexts.append((rt, rt.Context(0)))
    return _contexts[0]


def prepare(case, seed):
    st = dict(_inputs(case, seed), case=case)
    dt = DTYPES[case["mode"]]
    if case["kind"] == "linear":
        if own:
            _context()
            st["y"] = torch.empty(case["m"], case["n"], dtype=torch.float32 if case["out_f32"] else dt, device="cuda")
        return st
    rows, heads = sum(st["new"]), case["kv_heads"]
    if own:
        rt, ctx = _context()
        mode = rt.MODES[case["mode"]]
        st["cache"] = ctx.kv_cache(heads, st["pool"], mode)
        st["batch"] = rt.KvBatch(st["lengths"], st["pages"], st["starts"], rows)
        if case["kind"] != "write":
            filled = _starts(st["keys"])
            whole = rt.KvBatch(st["lengths"], st["pages"],
                               torch.tensor(filled, dtype=torch.int32, device="cuda"), filled[-1])
            ctx.kv_write(st["cache"], whole, st.pop("k"), st.pop("v"))
        if case["kind"] == "attention":
            st["out"] = torch.empty(rows, case["heads"] * HD, dtype=dt, device="cuda")
            st["work"] = torch.empty(ctx.kv_attention_workspace(st["cache"], st["batch"], case["heads"]),
                                     dtype=torch.uint8, device="cuda")
        else:
            st["k_out"] = torch.empty(rows, heads * HD, dtype=dt, device="cuda")
            st["v_out"] = torch.empty_like(st["k_out"])
    else:
        # the plain cache: codes and exponents by page, and the places of the rows
        st["codes"] = torch.zeros(2, st["pool"] * PAGE, heads, HD // 2, dtype=torch.uint8, device="cuda")
        st["exps"] = torch.zeros(2, st["pool"] * PAGE, heads, HD // GROUP, dtype=torch.int8, device="cuda")
        st["places"] = _places(st, st["new"], st["keys"])
        if case["kind"] != "write":
            _plain_write(st, _places(st, st["keys"], st["keys"]), st.pop("k"), st.pop("v"))
    torch.cuda.synchronize()
    return st


def _places(st, counts, keys):
    """The pool's row of each of the last counts[b] positions of the sequences."""
    n = torch.tensor(counts, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), n)
    first = torch.tensor([k - c - s for k, c, s in zip(keys, counts, _starts(counts))], device="cuda")
    pos = torch.arange(seq.numel(), device="cuda") + first[seq]
    return st["pages"][seq, pos // PAGE].long() * PAGE + pos % PAGE


# ---- the plain forms ---------------------------------------------------------

def _plain_codes(x, mode, heads):
    """x [rows][heads * 128] -> packed e2m1 codes and exponents."""
    lo, hi = EXPONENTS[mode]
    x = x.float().reshape(x.shape[0], heads, HD // GROUP, GROUP)
    m, e = torch.frexp(x.abs().amax(-1))
    e = (e - 3 + (m > 0.875).int()).clamp(lo, hi)
    y = x * ((127 - e) << 23).view(torch.float32)[..., None]
    a = y.abs().clamp_max(6)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | ((y < 0).to(torch.uint8) << 3)
    code = code.reshape(x.shape[0], heads, HD // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), e.to(torch.int8)


def _plain_write(st, places, k, v):
    case = st["case"]
    for i, x in enumerate((k, v)):
        code, e = _plain_codes(x, case["mode"], case["kv_heads"])
        st["codes"][i].index_copy_(0, places, code)
        st["exps"][i].index_copy_(0, places, e)


def _plain_values(codes, exps):
    """The values that codes [..., 64] and exponents [..., 4] stand for, in 32 bits."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda")
    table = torch.cat([table, -table])
    both = torch.stack([codes & 15, codes >> 4], -1).int()
    x = table[both].reshape(*exps.shape, GROUP)
    return (x * ((exps.int() + 127) << 23).view(torch.float32)[..., None]).reshape(*exps.shape[:-1], HD)


def _plain_read(st):
    dt = DTYPES[st["case"]["mode"]]
    x = _plain_values(st["codes"][:, st["places"]], st["exps"][:, st["places"]])
    x = x.reshape(2, x.shape[1], -1).to(dt)
    return [x[0], x[1]]


def _plain_attention(st):
    case = st["case"]
    heads, kvh, new, keys = case["heads"], case["kv_heads"], st["new"], st["keys"]
    b, n, L, group = len(new), max(new), max(keys), case["heads"] // case["kv_heads"]
    at = torch.arange(L, device="cuda")
    place = st["pages"].long()[:, at // PAGE] * PAGE + at % PAGE
    kv = _plain_values(st["codes"][:, place], st["exps"][:, place])  # [2][b][L][kvh][128]
    k, v = kv.transpose(2, 3).contiguous()  # [b][kvh][L][128]
    # rows of each sequence, padded to the longest: [b][kvh][group * n][128]
    i = torch.arange(n, device="cuda")
    count = torch.tensor(new, device="cuda")
    row = torch.minimum(st["starts"][:-1].long()[:, None] + i, st["starts"][1:].long()[:, None] - 1)
    q = st["q"].float().reshape(-1, kvh, group, HD)[row]  # [b][n][kvh][group][128]
    q = q.permute(0, 2, 3, 1, 4).reshape(b, kvh, group * n, HD)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(b, kvh, group, n, L) / math.sqrt(HD)
    length = st["lengths"].long()[:, None, None]
    seen = at < length
    if case["causal"]:
        seen = seen & (at <= length - count[:, None, None] + i[:, None])
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.reshape(b, kvh, group * n, L), v).reshape(b, kvh, group, n, HD) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, heads, HD)[i < count[:, None]]  # [rows][heads][128]
    if st["gate"] is not None:
        o = o * (2 / (1 + torch.exp(-st["gate"])))[..., None]
    return o.reshape(-1, heads * HD).to(DTYPES[case["mode"]])


def _plain_linear(st):
    case, q = st["case"], st["q"]
    w = torch.stack([q & 15, q >> 4], -1).reshape(q.shape[0], -1, WGROUP).int()
    w = ((w ^ 8) - 8).float() * st["s"].float()[..., None]
    y = torch.matmul(st["a"].float(), w.reshape(q.shape[0], -1).T)
    if st["bias"] is not None:
        y = y + st["bias"]
    if case["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y if case["out_f32"] else y.to(st["a"].dtype)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "linear":
            return _plain_linear(state)
        if kind == "attention":
            return _plain_attention(state)
        if kind == "write":
            _plain_write(state, state["places"], state["k"], state["v"])
        return _plain_read(state)
    rt, ctx = _context()
    mode = rt.MODES[case["mode"]]
    if kind == "linear":
        return ctx.linear_q4(state["a"], state["q"], state["s"], state["bias"], state["y"], mode=mode,
                             gelu=case["gelu"])
    if kind == "attention":
        return ctx.kv_attention(state["cache"], state["batch"], state["q"], state["out"], case["heads"],
                                causal=case["causal"], glog=state["gate"], work=state["work"])
    if kind == "write":
        ctx.kv_write(state["cache"], state["batch"], state["k"], state["v"])
    ctx.kv_read(state["cache"], state["batch"], state["k_out"], state["v_out"])
    return [state["k_out"], state["v_out"]]


# ---- the definition in 64 bits -----------------------------------------------

def _exact_values(x, mode, heads):
    """What the cache makes of x [rows][heads * 128]: for each group the nearest
    of the sixteen numbers, found by bisection between their midpoints."""
    lo, hi = EXPONENTS[mode]
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    mid = (grid[1:] + grid[:-1]) / 2
    for r in range(0, x.shape[0], 8192):
        g = x[r:r + 8192].double().reshape(-1, GROUP)
        top = g.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(top.clamp_min(1e-300))) - 2
        e = torch.where(top > 7 * torch.exp2(e), e + 1, e).clamp(lo, hi)
        y = g.abs() / torch.exp2(e)
        below, above = torch.searchsorted(mid, y), torch.searchsorted(mid, y, right=True)
        index = torch.where((below != above) & (below % 2 == 1), above, below)  # a midpoint goes to the even code
        out[r:r + 8192] = (torch.copysign(grid[index], g) * torch.exp2(e)).reshape(-1, heads * HD)
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "linear":
        nibbles = torch.stack([x["q"] % 16, x["q"] // 16], 2).flatten(1).double()
        w = torch.where(nibbles > 7, nibbles - 16, nibbles)
        y = x["a"].double() @ (w * x["s"].double().repeat_interleave(WGROUP, 1)).T
        if x["bias"] is not None:
            y += x["bias"].double()
        if case["gelu"]:
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        return y
    kvh = case["kv_heads"]
    k, v = (_exact_values(t, case["mode"], kvh) for t in (x["k"], x["v"]))
    if case["kind"] == "write":
        return [k, v]
    new, keys = x["new"], x["keys"]
    ends = _starts(keys)[1:]
    if case["kind"] == "read":
        return [torch.cat([t[e - n:e] for e, n in zip(ends, new)]) for t in (k, v)]
    group = case["heads"] // kvh
    out = torch.empty(sum(new), case["heads"] * HD, dtype=torch.float64, device="cuda")
    for b, (n, L) in enumerate(zip(new, keys)):
        r = _starts(new)[b]
        for h in range(case["heads"]):
            cols, own_cols = slice(h // group * HD, (h // group + 1) * HD), slice(h * HD, (h + 1) * HD)
            s = x["q"][r:r + n, own_cols].double() @ k[ends[b] - L:ends[b], cols].T / HD ** 0.5
            if case["causal"]:
                s += torch.full((n, L), -math.inf, dtype=torch.float64, device="cuda").triu_(L - n + 1)
            p = torch.softmax(s, 1)
            out[r:r + n, own_cols] = p @ v[ends[b] - L:ends[b], cols]
    if x["gate"] is not None:
        out *= 2 * torch.sigmoid(x["gate"].double()).repeat_interleave(HD, 1)
    return out
