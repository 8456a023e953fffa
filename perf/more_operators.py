"""Timed cases of the operators between a block's hidden state and the 4-bit cache
in a streamed step: microscaled 4-bit linears, norm and rotary positions of q and k,
and attention with a sliding window and first tokens that stay visible.

Four kinds of call, each through ltx_amd.runtime:

  quantise   rows become 4-bit codes and scales; what these stand for is read back
  linear     y = a . w^T (+ bias, GELU), both operands in that form; few rows of a
             come in 16 bits and are quantised on the way, more in a call before it,
             or they are in the form already
  rope       RMS norm over the row (or none), then every pair (j, j + 64) of a head
             turned by freq * position + phase, each pair on one of several axes
  attention  rows of q attend to the last `window` keys that they could see and to
             the first `sinks`, in a paged cache of 4-bit keys and values

The 4-bit form: 32 consecutive values share a power of two 2^e and are held as e2m1
numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives). e is the one that takes the
group's largest magnitude to at most 7 and above 3.5 (7 .. 6 rounds down), limited to
what the type holds; values round to the nearest, ties to the even code.

Head and width sizes are the block's (32 heads x 128, d_model 4096, FFN 16,384), with
32, 8 or 4 heads in the cache; lengths go from one token to the benchmark's 28,672. A
case is a dict of plain values; listed() names the fixed ones, draw() gives others of
the same ranges.
"""
import math
import os
import sys

import torch

own = False

HD, PAGE, GROUP = 128, 64, 32  # head size, tokens a page, values that share a scale
D, H, FF = 4096, 32, 16384
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EXPONENTS = {"f16": (-23, 13), "bf16": (-125, 125), "f32": (-125, 125)}  # 0.5 * 2^e and 6 * 2^e are numbers of the type
PROJ = ((4096, 4096), (8192, 4096), (12288, 4096), (16384, 4096), (4096, 16384))  # (n, k) of the block's projections
FEW = 64   # up to this many rows a linear takes them in 16 bits
EPS = 1e-6
SECTIONS = (16, 24, 24)  # pairs on time, height and width where all heads turn alike


def listed():
    return [
        # the hidden state of 8 single tokens before their projections: slices of wider rows
        dict(name="quantise_bf16_step8", kind="quantise", mode="bf16", rows=8, k=4096, wide=True),
        # a whole clip's hidden state before q|k|v
        dict(name="quantise_f16_t28672", kind="quantise", mode="f16", rows=28672, k=4096, wide=False),
        # one token's out projection, from 16-bit rows
        dict(name="linear_f16_m1", kind="linear", mode="f16", m=1, n=4096, k=4096, a="rows", bias=True, gelu=False,
             out_f32=False),
        # FFN up with GELU for an odd batch of single tokens, from 16-bit rows
        dict(name="linear_bf16_m33", kind="linear", mode="bf16", m=33, n=16384, k=4096, a="rows", bias=False,
             gelu=True, out_f32=False),
        # q|k|v of a streamed latent frame (32 x 64 tokens), quantised and multiplied
        dict(name="linear_f16_frame_qkv", kind="linear", mode="f16", m=2048, n=12288, k=4096, a="rows", bias=True,
             gelu=False, out_f32=False),
        # FFN down of a whole clip, the hidden layer in 4 bits already, f32 residual
        dict(name="linear_bf16_t28672_down", kind="linear", mode="bf16", m=28672, n=4096, k=16384, a="mx4", bias=True,
             gelu=False, out_f32=True),
        # one token each of 32 sequences: 32 query heads on 8, all heads alike, no norm, q|k|v slices
        dict(name="rope_bf16_step32", kind="rope", mode="bf16", rows=32, heads=32, kv_heads=8, plan="alike", norm=False),
        # a whole clip with the block's own frequencies and qk norm
        dict(name="rope_f16_t28672", kind="rope", mode="f16", rows=28672, heads=32, kv_heads=32, plan="grid", norm=True),
        # one token far into a stream, a short window and four first tokens
        dict(name="attention_f16_step1", kind="attention", mode="f16", heads=32, kv_heads=32, seqs=1, new=1, keys=28672,
             ragged=False, causal=True, gate=False, window=1000, sinks=4),
        # a serving step: 32 ragged sequences, four query heads a cached head
        dict(name="attention_bf16_step32", kind="attention", mode="bf16", heads=32, kv_heads=8, seqs=32, new=1,
             keys=8192, ragged=True, causal=True, gate=False, window=4096, sinks=64),
        # a streamed video's next latent frame against the 4 before it, itself and the first
        dict(name="attention_f16_frame", kind="attention", mode="f16", heads=32, kv_heads=32, seqs=1, new=2048,
             keys=28672, ragged=False, causal=False, gate=True, window=10240, sinks=2048),
        # ragged prompts of three sequences enter at once, an odd window
        dict(name="attention_bf16_prefill", kind="attention", mode="bf16", heads=32, kv_heads=8, seqs=3, new=2970,
             keys=2970, ragged=True, causal=True, gate=False, window=701, sinks=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantise", "linear", "linear", "linear", "rope", "attention", "attention", "attention"])
    mode = rng.choice(["f16", "bf16"])
    if kind == "quantise":
        return dict(kind=kind, mode=rng.choice(["f16", "bf16", "f32"]), rows=_log(rng, 1, 14336),
                    k=128 * rng.randint(1, 32), wide=rng.random() < 0.5)
    if kind == "linear":
        n, k = rng.choice(PROJ)
        if rng.random() < 0.3:
            n, k = _log(rng, 1, 16384), 128 * _log(rng, 1, 128)
        m = _log(rng, 1, FEW) if rng.random() < 0.4 else _log(rng, FEW, min(28672, 28672 * D * FF // (n * k)))
        return dict(kind=kind, mode=mode, m=m, n=n, k=k, a=rng.choice(["rows", "mx4"]), bias=rng.random() < 0.5,
                    gelu=n == FF, out_f32=rng.random() < 0.3)
    if kind == "rope":
        plan = rng.choice(["alike", "grid"])
        return dict(kind=kind, mode=rng.choice(["f16", "bf16", "f32"]), rows=_log(rng, 1, 14336), heads=H,
                    kv_heads=H if plan == "grid" else rng.choice([32, 8, 4]), plan=plan, norm=rng.random() < 0.5)
    seqs = _log(rng, 1, 64)
    keys = _log(rng, 1, min(28672, 114688 // seqs))
    new = 1 if rng.random() < 0.5 else min(keys, _log(rng, 1, max(1, 2048 // seqs)))
    return dict(kind=kind, mode=mode, heads=H, kv_heads=rng.choice([32, 8, 4]), seqs=seqs, new=new, keys=keys,
                ragged=rng.random() < 0.5, causal=rng.random() < 0.7, gate=rng.random() < 0.3,
                window=_log(rng, 1, 10240), sinks=0 if rng.random() < 0.3 else _log(rng, 1, 2048))


# ---- the shape of a batch ----------------------------------------------------

def _lengths(case):
    """New rows and keys of each sequence; ragged ones go down from the case's."""
    n, top, keys = case["seqs"], case["new"], case["keys"]
    if not case["ragged"]:
        return [top] * n, [keys] * n
    new = [max(1, top - top * b // (2 * n) - (b if top > n else 0)) for b in range(n)]
    return new, [max(new[b], keys - keys * b // n - (3 * b if keys > 4 * n else 0)) for b in range(n)]


def _seen(case):
    """Of all sequences: (row, key) pairs, and keys that some row sees."""
    window, sinks = case["window"], case["sinks"]
    pairs = keys = 0
    for n, L in zip(*_lengths(case)):
        ends = [L - n + 1 + i for i in range(n)] if case["causal"] else [L] * n
        pairs += sum(min(e, min(window, e) + min(sinks, max(0, e - window))) for e in ends)
        low = max(0, ends[0] - window)
        keys += L - low + min(sinks, low)
    return pairs, keys


def work(case):
    kind, a = case["kind"], 4 if case["mode"] == "f32" else 2
    if kind == "quantise":  # read, held, read back, returned
        n = case["rows"] * case["k"]
        return {"bytes": 2 * n * a + 2 * (n // 2 + n // GROUP), "flops": 0}
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        held = k // 2 + k // GROUP
        return {"bytes": m * (k * a if case["a"] == "rows" else held) + n * held + (4 * n if case["bias"] else 0)
                + m * n * (4 if case["out_f32"] else 2), "flops": 2 * m * n * k}
    if kind == "rope":
        width = (case["heads"] + case["kv_heads"]) * HD
        return {"bytes": case["rows"] * (2 * width * a + 24) + (4 * width if case["norm"] else 0), "flops": 0}
    pairs, keys = _seen(case)
    rows, width = sum(_lengths(case)[0]), case["heads"] * HD
    return {"bytes": keys * case["kv_heads"] * (HD // 2 + HD // GROUP) * 2
            + rows * (2 * width * 2 + (4 * case["heads"] if case["gate"] else 0)),
            "flops": 4 * HD * case["heads"] * pairs}


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + 41)
    return g


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _hidden(g, rows, k, dt):
    """Rows as a norm leaves them: channels of unlike size, some far larger."""
    x = torch.empty(rows, k, dtype=dt, device="cuda")
    size = torch.exp(_normal(g, k, std=0.5))
    size[torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")] *= 20
    for r in range(0, rows, 4096):
        n = min(4096, rows - r)
        x[r:r + n] = (_normal(g, n, k) * size).to(dt)
    return x


def _weights(g, n, k):
    """Student-t(3) x 0.02, bf16, as the block's."""
    w = torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
    for r in range(0, n, 2048):
        m = min(2048, n - r)
        chi = sum(_normal(g, m, k).square_() for _ in range(3))
        w[r:r + m] = (0.02 * _normal(g, m, k) / torch.sqrt(chi / 3)).to(torch.bfloat16)
    return w


def _plan(case):
    """Frequency, phase and axis of each head's 64 pairs, f64 and int32 [heads][64]."""
    if case["plan"] == "alike":  # all heads alike: sections of pairs on time, height, width
        freq = 10000.0 ** -(torch.arange(64, dtype=torch.float64) / 64)
        axis = torch.repeat_interleave(torch.arange(3), torch.tensor(SECTIONS))
        return freq[None], torch.zeros(1, 64, dtype=torch.float64), axis[None].to(torch.int32)
    # the block's: 682 frequencies on three axes in turn over the heads' 2,048 pairs, two
    # pairs that do not turn; positions as fractions of (20, 2048, 2048) mapped to -1 .. 1
    f = (10000.0 ** torch.linspace(0, 1, 682, dtype=torch.float64) * (math.pi / 2)).float().double()
    j = torch.arange(32 * 64) - 2
    axis = torch.where(j < 0, 0, j % 3)
    f = torch.where(j < 0, 0.0, f[torch.div(j.clamp_min(0), 3, rounding_mode="floor")])
    top = torch.tensor([20.0, 2048.0, 2048.0], dtype=torch.float64)[axis]
    return (2 * f / top).reshape(32, 64), (-f).reshape(32, 64), axis.reshape(32, 64).to(torch.int32)


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
    g, kind, dt = _gen(seed), case["kind"], DTYPES[case["mode"]]
    if kind == "quantise":
        x = _hidden(g, case["rows"], 3 * case["k"] if case["wide"] else case["k"], dt)
        return dict(x=x[:, case["k"]:2 * case["k"]] if case["wide"] else x)
    if kind == "linear":
        return dict(a=_hidden(g, case["m"], case["k"], dt), w=_weights(g, case["n"], case["k"]),
                    bias=_normal(g, case["n"], std=0.02) if case["bias"] else None)
    if kind == "rope":
        rows, qw, kw = case["rows"], case["heads"] * HD, case["kv_heads"] * HD
        fused = torch.empty(rows, qw + 2 * kw, dtype=dt, device="cuda")  # q | k | v
        for r in range(0, rows, 4096):
            n = min(4096, rows - r)
            fused[r:r + n] = _normal(g, n, qw + 2 * kw).to(dt)
        at = torch.arange(rows, device="cuda")  # a grid of 32 x 64 places a frame, some way into the stream
        first = torch.randint(0, 12, (1,), generator=g, device="cuda")
        pos = torch.stack([(first + at // 2048).double() * 8 / 24, (at // 64 % 32).double() * 32, (at % 64).double() * 32], 1)
        norm = [1 + _normal(g, w, std=0.2) if case["norm"] else None for w in (qw, kw)]
        return dict(q=fused[:, :qw], k=fused[:, qw:qw + kw], pos=pos.contiguous(), wq=norm[0], wk=norm[1])
    b = _batch(case, g)
    rows, width, kw = sum(b["new"]), case["heads"] * HD, case["kv_heads"] * HD
    # what the cache holds before the call: every key of every sequence
    n = sum(b["keys"])
    scale = torch.exp(_normal(g, kw, std=0.5))
    b["k"], b["v"] = (_normal(g, n, kw) * scale).to(dt), _normal(g, n, kw, std=0.7).to(dt)
    b["q"] = _normal(g, rows, width + 2 * kw).to(dt)[:, :width]
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


def _held(rows, k):
    """Room for codes and scales of rows: two codes a byte; of 128 values four scales, of all rows in turn."""
    return (torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda"),
            torch.empty(k // 128, rows, 4, dtype=torch.uint8, device="cuda"))


def prepare(case, seed):
    kind, dt = case["kind"], DTYPES[case["mode"]]
    st = dict(_inputs(case, seed), case=case)
    if own:
        rt, ctx = _context()
        mode = rt.MODES[case["mode"]]
    if kind == "quantise":
        if own:
            st["held"] = _held(case["rows"], case["k"])
            st["y"] = torch.empty(case["rows"], case["k"], dtype=dt, device="cuda")
    elif kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        w = st.pop("w")
        if own:
            st["w"] = ctx.mx4_quantise(w, *_held(n, k), mode=rt.MODE_BF16)
            st["y"] = torch.empty(m, n, dtype=torch.float32 if case["out_f32"] else dt, device="cuda")
            if case["a"] == "mx4":
                st["a"] = ctx.mx4_quantise(st["a"], *_held(m, k), mode=mode)
            elif m > FEW:
                st["held"] = _held(m, k)
        else:
            st["w"] = _plain_codes(w, "bf16")
            if case["a"] == "mx4":
                st["a"] = _plain_codes(st["a"], case["mode"])
    elif kind == "rope":
        plan = _plan(case)
        if own:
            st["plan"] = ctx.rope(*plan, axes=3)
            st["out"] = (torch.empty(st["q"].shape, dtype=dt, device="cuda"),
                         torch.empty(st["k"].shape, dtype=dt, device="cuda"))
        else:
            st["plan"] = [t.cuda() for t in plan]
    else:
        rows, heads = sum(st["new"]), case["kv_heads"]
        if own:
            st["cache"] = ctx.kv_cache(heads, st["pool"], mode)
            st["batch"] = rt.KvBatch(st["lengths"], st["pages"], st["starts"], rows)
            filled = _starts(st["keys"])
            whole = rt.KvBatch(st["lengths"], st["pages"],
                               torch.tensor(filled, dtype=torch.int32, device="cuda"), filled[-1])
            ctx.kv_write(st["cache"], whole, st.pop("k"), st.pop("v"))
            st["out"] = torch.empty(rows, case["heads"] * HD, dtype=dt, device="cuda")
            st["work"] = torch.empty(ctx.kv_attention_window_workspace(st["cache"], st["batch"], case["heads"],
                                                                       case["window"], case["sinks"],
                                                                       causal=case["causal"]),
                                     dtype=torch.uint8, device="cuda")
        else:  # the plain cache: codes and exponents by page
            place = _places(st)
            for x in ("k", "v"):
                codes, e = _plain_codes(st.pop(x), case["mode"])
                held = [torch.zeros(st["pool"] * PAGE, heads, HD // 2, dtype=torch.uint8, device="cuda"),
                        torch.zeros(st["pool"] * PAGE, heads, HD // GROUP, dtype=torch.int8, device="cuda")]
                held[0][place] = codes.reshape(-1, heads, HD // 2)
                held[1][place] = e.reshape(-1, heads, HD // GROUP)
                st["held_" + x] = held
    torch.cuda.synchronize()
    return st


def _places(st):
    """The pool's row of every key of the sequences."""
    n = torch.tensor(st["keys"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(st["keys"]), device="cuda"), n)
    pos = torch.arange(seq.numel(), device="cuda") - torch.tensor(_starts(st["keys"])[:-1], device="cuda")[seq]
    return st["pages"][seq, pos // PAGE].long() * PAGE + pos % PAGE


# ---- the plain forms ---------------------------------------------------------

def _plain_codes(x, mode):
    """x [rows][k] -> packed e2m1 codes [rows][k / 2] and exponents [rows][k / 32]."""
    lo, hi = EXPONENTS[mode]
    rows, k = x.shape
    codes = torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda")
    exps = torch.empty(rows, k // GROUP, dtype=torch.int8, device="cuda")
    for r in range(0, rows, 8192):
        y = x[r:r + 8192].float().reshape(-1, k // GROUP, GROUP)
        m, e = torch.frexp(y.abs().amax(-1))
        e = (e - 3 + (m > 0.875).int()).clamp(lo, hi)
        y = y * ((127 - e) << 23).view(torch.float32)[..., None]
        a = y.abs().clamp_max(6)
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        a = torch.round(a / step) * step
        code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
        code = (code | ((y < 0).to(torch.uint8) << 3)).reshape(-1, k // 2, 2)
        codes[r:r + 8192] = code[..., 0] | (code[..., 1] << 4)
        exps[r:r + 8192] = e.to(torch.int8)
    return codes, exps


def _plain_values(codes, exps):
    """The values that codes [..., k / 2] and exponents [..., k / 32] stand for, in 32 bits."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda")
    table = torch.cat([table, -table])
    both = torch.stack([codes & 15, codes >> 4], -1).int()
    x = table[both].reshape(*exps.shape, GROUP)
    return (x * ((exps.int() + 127) << 23).view(torch.float32)[..., None]).flatten(-2)


def _plain_linear(st):
    case = st["case"]
    a = st["a"] if case["a"] == "mx4" else _plain_codes(st["a"], case["mode"])
    y = torch.matmul(_plain_values(*a), _plain_values(*st["w"]).T)
    if st["bias"] is not None:
        y = y + st["bias"]
    if case["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y if case["out_f32"] else y.to(DTYPES[case["mode"]])


def _plain_rope(st):
    freq, phase, axis = st["plan"]
    angle = st["pos"][:, axis.long()] * freq + phase  # f64: positions lie thousands of turns away
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    outs = []
    for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
        y = y.reshape(y.shape[0], -1, 2, 64)
        heads = y.shape[1] // cos.shape[1]  # heads that turn alike follow each other
        c, s = (t.repeat_interleave(heads, 1) for t in (cos, sin))
        y = torch.stack([y[:, :, 0] * c - y[:, :, 1] * s, y[:, :, 1] * c + y[:, :, 0] * s], 2)
        outs.append(y.reshape(x.shape).to(x.dtype))
    return outs


def _plain_attention(st):
    case = st["case"]
    heads, kvh, new, keys = case["heads"], case["kv_heads"], st["new"], st["keys"]
    b, n, L, group = len(new), max(new), max(keys), case["heads"] // case["kv_heads"]
    at = torch.arange(L, device="cuda")
    place = st["pages"].long()[:, at // PAGE] * PAGE + at % PAGE
    k, v = (_plain_values(*(t[place] for t in st[x])).transpose(1, 2).contiguous() for x in ("held_k", "held_v"))
    # rows of each sequence, padded to the longest: [b][kvh][group * n][128]
    i = torch.arange(n, device="cuda")
    count = torch.tensor(new, device="cuda")
    row = torch.minimum(st["starts"][:-1].long()[:, None] + i, st["starts"][1:].long()[:, None] - 1)
    q = st["q"].float().reshape(-1, kvh, group, HD)[row]  # [b][n][kvh][group][128]
    q = q.permute(0, 2, 3, 1, 4).reshape(b, kvh, group * n, HD)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(b, kvh, group, n, L) / math.sqrt(HD)
    length = st["lengths"].long()[:, None, None]
    end = length - count[:, None, None] + i[:, None] + 1 if case["causal"] else length
    seen = (at < end) & ((at >= end - case["window"]) | (at < case["sinks"]))
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.reshape(b, kvh, group * n, L), v).reshape(b, kvh, group, n, HD) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, heads, HD)[i < count[:, None]]  # [rows][heads][128]
    if st["gate"] is not None:
        o = o * (2 / (1 + torch.exp(-st["gate"])))[..., None]
    return o.reshape(-1, heads * HD).to(DTYPES[case["mode"]])


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "linear":
            return _plain_linear(state)
        if kind == "rope":
            return _plain_rope(state)
        if kind == "attention":
            return _plain_attention(state)
        return _plain_values(*_plain_codes(state["x"], case["mode"])).to(state["x"].dtype)
    rt, ctx = _context()
    mode = rt.MODES[case["mode"]]
    if kind == "quantise":
        q, s = ctx.mx4_quantise(state["x"], *state["held"], mode=mode)
        return ctx.mx4_values(q, s, state["y"], mode=mode)
    if kind == "linear":
        a, scales = state["a"] if case["a"] == "mx4" else (state["a"], None)
        if "held" in state:
            a, scales = ctx.mx4_quantise(a, *state["held"], mode=mode)
        return ctx.linear_mx4(a, scales, *state["w"], state["bias"], state["y"], mode=mode, gelu=case["gelu"])
    if kind == "rope":
        q, k = state["out"]
        ctx.qk_rope(state["plan"], state["pos"], state["q"], q, state["k"], k, state["wq"], state["wk"], eps=EPS,
                    mode=mode)
        return [q, k]
    return ctx.kv_attention_window(state["cache"], state["batch"], state["q"], state["out"], case["heads"],
                                   case["window"], case["sinks"], causal=case["causal"], glog=state["gate"],
                                   work=state["work"])


# ---- the definition in 64 bits -----------------------------------------------

def _exact_values(x, mode):
    """What the form makes of x [rows][k]: for each group the nearest of the sixteen
    numbers, found by bisection between their midpoints."""
    lo, hi = EXPONENTS[mode]
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    mid = (grid[1:] + grid[:-1]) / 2
    for r in range(0, x.shape[0], 4096):
        g = x[r:r + 4096].double().reshape(-1, GROUP)
        top = g.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(top.clamp_min(1e-300))) - 2
        e = torch.where(top > 7 * torch.exp2(e), e + 1, e).clamp(lo, hi)
        y = g.abs() / torch.exp2(e)
        below, above = torch.searchsorted(mid, y), torch.searchsorted(mid, y, right=True)
        index = torch.where((below != above) & (below % 2 == 1), above, below)  # a midpoint goes to the even code
        out[r:r + 4096] = (torch.copysign(grid[index], g) * torch.exp2(e)).reshape(-1, x.shape[1])
    return out


def _exact_attention(case, x):
    kvh, new, keys = case["kv_heads"], x["new"], x["keys"]
    k, v = (_exact_values(t, case["mode"]) for t in (x["k"], x["v"]))
    ends, group = _starts(keys)[1:], case["heads"] // kvh
    out = torch.empty(sum(new), case["heads"] * HD, dtype=torch.float64, device="cuda")
    for b, (n, L) in enumerate(zip(new, keys)):
        r, at = _starts(new)[b], torch.arange(L, device="cuda")
        last = torch.arange(L - n, L, device="cuda")[:, None] if case["causal"] else torch.full((n, 1), L - 1, device="cuda")
        hidden = (at > last) | ((last - at >= case["window"]) & (at >= case["sinks"]))
        for h in range(case["heads"]):
            cols, own_cols = slice(h // group * HD, (h // group + 1) * HD), slice(h * HD, (h + 1) * HD)
            s = x["q"][r:r + n, own_cols].double() @ k[ends[b] - L:ends[b], cols].T / HD ** 0.5
            p = torch.softmax(s.masked_fill_(hidden, -math.inf), 1)
            out[r:r + n, own_cols] = p @ v[ends[b] - L:ends[b], cols]
    if x["gate"] is not None:
        out *= 2 * torch.sigmoid(x["gate"].double()).repeat_interleave(HD, 1)
    return out


def exact(case, seed):
    x, kind = _inputs(case, seed), case["kind"]
    if kind == "quantise":
        return _exact_values(x["x"], case["mode"])
    if kind == "attention":
        return _exact_attention(case, x)
    if kind == "linear":
        y = _exact_values(x["a"], case["mode"]) @ _exact_values(x["w"], "bf16").T
        if x["bias"] is not None:
            y += x["bias"].double()
        if case["gelu"]:
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        return y
    freq, phase, axis = (t.cuda() for t in _plan(case))
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       x["pos"][:, axis.reshape(-1).long()] * freq.reshape(-1) + phase.reshape(-1))
    outs = []
    for t, w in ((x["q"], x["wq"]), (x["k"], x["wk"])):
        out = torch.empty(t.shape, dtype=torch.float64, device="cuda")
        for r in range(0, t.shape[0], 4096):
            y = t[r:r + 4096].double()
            if w is not None:
                y = y / torch.sqrt((y * y).sum(1, keepdim=True) / y.shape[1] + EPS) * w.double()
            y = y.reshape(y.shape[0], freq.shape[0], -1, 2, 64)
            z = torch.complex(y[..., 0, :].contiguous(), y[..., 1, :].contiguous())
            z = z * turn[r:r + 4096].reshape(y.shape[0], freq.shape[0], 1, 64)
            out[r:r + 4096] = torch.stack([z.real, z.imag], -2).reshape(y.shape[0], -1)
        outs.append(out)
    return outs
