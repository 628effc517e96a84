"""Cases and plain forms of the decayed linear attention operators.

Three operators of ``catfuse_b200.ops`` are measured here:

* ``qk_norm_rope``: per-head RMS norm of queries and keys with the position
  rotation (one to three position axes) in the same pass;
* ``decay_attention``: causal linear attention with a decay per head over whole
  prompts, dense or packed, with the state that it leaves behind;
* ``decay_attention_step``: the same recurrence for one token per sequence.

``run`` computes a case with elementary torch operations in 32 bits, or, where
``own`` is set, with the calls a user of the package makes.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One decoding step of a small spiking transformer's twelve heads of 32
        # (384 channels): what a stream pays before each token's attention.
        {"name": "rope token", "op": "rope", "dtype": "fp16", "tokens": 8, "heads": 12,
         "kv_heads": 12, "dim": 32, "rot": 32, "axes": 1, "order": "blocks", "pairing": "adjacent",
         "norm": True},
        # A text prompt with grouped heads, q and k taken out of the fused projection.
        {"name": "rope text", "op": "rope", "dtype": "bf16", "tokens": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "axes": 1, "order": "blocks", "pairing": "half",
         "norm": True},
        # A clip of 28x28 patch grids: time, height and width positions, heads
        # of 80 with a quarter of each left unrotated.
        {"name": "rope clip", "op": "rope", "dtype": "fp16", "tokens": 12544, "heads": 16,
         "kv_heads": 16, "dim": 80, "rot": 60, "axes": 3, "order": "cyclic", "pairing": "half",
         "norm": True},
        # Spikes of a 64-token patch grid, four time steps folded into the heads
        # (4 x 12 heads of 32): the smallest call, where latency counts.
        {"name": "prompt patches", "op": "prompt", "dtype": "fp16", "batch": 2, "length": 64,
         "heads": 48, "kv_heads": 48, "dk": 32, "dv": 32, "packed": False, "carry": False,
         "values": "spikes"},
        # One chat prompt: few sequences, so the token axis has to be split.
        {"name": "prompt chat", "op": "prompt", "dtype": "bf16", "batch": 1, "length": 4095,
         "heads": 32, "kv_heads": 32, "dk": 128, "dv": 128, "packed": False, "carry": False,
         "values": "normal"},
        # Prompts of very different lengths packed into one call, grouped heads.
        {"name": "prompt packed", "op": "prompt", "dtype": "bf16", "batch": 23, "length": 1111,
         "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128, "packed": True, "carry": False,
         "values": "normal"},
        # One long document with narrow heads, continued from a carried state.
        {"name": "prompt document", "op": "prompt", "dtype": "fp16", "batch": 1, "length": 65536,
         "heads": 16, "kv_heads": 16, "dk": 64, "dv": 64, "packed": False, "carry": True,
         "values": "normal"},
        # A large batch of equal prompts: the throughput case.
        {"name": "prompt batch", "op": "prompt", "dtype": "bf16", "batch": 16, "length": 4096,
         "heads": 16, "kv_heads": 16, "dk": 128, "dv": 128, "packed": False, "carry": True,
         "values": "normal"},
        # One stream, one token: pure latency.
        {"name": "token one", "op": "token", "dtype": "fp16", "batch": 1, "heads": 12,
         "kv_heads": 12, "dk": 32, "dv": 32, "slots": False},
        # A serving batch with grouped heads whose states lie in a pool.
        {"name": "token serving", "op": "token", "dtype": "bf16", "batch": 61, "heads": 32,
         "kv_heads": 8, "dk": 128, "dv": 128, "slots": True},
        # A full batch with a state for each head: the largest state traffic.
        {"name": "token full", "op": "token", "dtype": "bf16", "batch": 128, "heads": 32,
         "kv_heads": 32, "dk": 128, "dv": 128, "slots": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["fp16", "bf16"])
    op = rng.choice(["rope", "prompt", "prompt", "token"])
    kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    group = rng.choice([1, 1, 1, 2, 3, 4, 8])
    while kv * group > 48:
        group -= 1
    if op == "rope":
        dim = rng.choice([32, 64, 80, 96, 128, 160, 256])
        axes = rng.choice([1, 1, 2, 3])
        rot = rng.choice([dim, dim, dim // 2])
        limit = (600 << 20) // (4 * dim * kv * (group + 1))
        return {"op": op, "dtype": dtype, "tokens": _log_int(rng, 1, min(32768, limit)),
                "heads": kv * group, "kv_heads": kv, "dim": dim, "rot": rot, "axes": axes,
                "order": rng.choice(["blocks", "cyclic"]),
                "pairing": rng.choice(["half", "adjacent"]), "norm": rng.random() < 0.8}
    dk, dv = rng.choice([(32, 32), (64, 64), (128, 128), (128, 128), (48, 96), (64, 128),
                         (128, 64), (80, 80)])
    if op == "token":
        limit = max(1, (512 << 20) // (8 * kv * dk * dv))
        return {"op": op, "dtype": dtype, "batch": _log_int(rng, 1, min(256, limit)),
                "heads": kv * group, "kv_heads": kv, "dk": dk, "dv": dv,
                "slots": rng.random() < 0.5}
    tokens = _log_int(rng, 16, min(65536, (512 << 20) // (2 * kv * (group + 1) * (dk + dv))))
    packed = rng.random() < 0.5
    batch = min(tokens, _log_int(rng, 1, 64))
    return {"op": op, "dtype": dtype, "batch": batch, "length": max(1, tokens // batch),
            "heads": kv * group, "kv_heads": kv, "dk": dk, "dv": dv, "packed": packed,
            "carry": (not packed) and rng.random() < 0.5,
            "values": rng.choice(["normal", "normal", "spikes"])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _sections(c):
    """Rotated pairs of each position axis: the first axis (time) takes what
    does not divide evenly."""
    pairs, a = c["rot"] // 2, c["axes"]
    rest = [pairs // a] * (a - 1)
    return (pairs - sum(rest), *rest)


def _axis_of_pair(c):
    """Position axis of each rotated pair: whole blocks, or one pair of each
    axis in turn until an axis has used up its share."""
    left = list(_sections(c))
    if c["order"] == "blocks":
        return [a for a, n in enumerate(left) for _ in range(n)]
    got, a = [], 0
    while len(got) < c["rot"] // 2:
        if left[a]:
            left[a] -= 1
            got.append(a)
        a = (a + 1) % len(left)
    return got


def _log_decay(heads, device):
    """Decays from e^-1 down to e^-1/512 over the heads: short
    memories beside long ones."""
    return -torch.exp2(torch.linspace(0.0, -9.0, heads, device=device))


def _values(shape, kind, dtype, g, device):
    if kind == "spikes":
        return (torch.rand(shape, generator=g, device=device) < 0.2).to(dtype)
    return torch.randn(shape, generator=g, device=device).to(dtype)


def _lengths(total, n, seed):
    """n lengths of at least one token that sum to total, spread over their logarithm."""
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(4.0 * torch.rand(n, generator=g, dtype=torch.float64))
    cut = torch.floor(torch.cumsum(w, 0) / w.sum() * (total - n)).to(torch.int64)
    cut[-1] = total - n
    return torch.diff(cut, prepend=torch.zeros(1, dtype=torch.int64)) + 1


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    h, hk = c["heads"], c["kv_heads"]
    st = {"case": c}
    if c["op"] == "rope":
        n, d = c["tokens"], c["dim"]
        qkv = torch.randn(n, (h + 2 * hk) * d, generator=g, device=dev).mul_(2.0).to(dt)
        st["q"] = qkv[:, :h * d].unflatten(1, (h, d))
        st["k"] = qkv[:, h * d:(h + hk) * d].unflatten(1, (hk, d))
        if c["axes"] == 1:
            first = int(torch.randint(0, 4096, (1,), generator=g, device=dev))
            st["positions"] = torch.arange(first, first + n, device=dev, dtype=torch.int32)
        else:
            t = torch.arange(n, device=dev, dtype=torch.int32)
            grid = [t // 784, t // 28 % 28, t % 28]
            st["positions"] = torch.stack(grid[3 - c["axes"]:] if c["axes"] < 3 else grid)
        pairs = c["rot"] // 2
        st["inv_freq"] = 10000.0 ** (-torch.arange(pairs, device=dev, dtype=torch.float32) / pairs)
        st["axis"] = torch.tensor(_axis_of_pair(c), device=dev)
        for w in ("q_weight", "k_weight"):
            st[w] = 1.0 + 0.1 * torch.randn(d, generator=g, device=dev) if c["norm"] else None
        return st
    b, dk, dv = c["batch"], c["dk"], c["dv"]
    st["log_decay"] = _log_decay(hk, dev)
    if c["op"] == "token":
        rows = 2 * b if c["slots"] else b
        st["q"] = _values((b, h, dk), "normal", dt, g, dev)
        st["k"] = _values((b, hk, dk), "normal", dt, g, dev)
        st["v"] = _values((b, hk, dv), "normal", dt, g, dev)
        st["s_in"] = torch.randn(rows, hk, dk, dv, generator=g, device=dev)
        st["s_out"] = torch.zeros_like(st["s_in"])
        st["slots"] = torch.randperm(rows, generator=g, device=dev)[:b].to(torch.int32) if c["slots"] else None
        return st
    n = b * c["length"]
    lead = (n,) if c["packed"] else (b, c["length"])
    st["q"] = _values((*lead, h, dk), c["values"], dt, g, dev)
    st["k"] = _values((*lead, hk, dk), c["values"], dt, g, dev)
    st["v"] = _values((*lead, hk, dv), c["values"], dt, g, dev)
    st["cu_seqlens"] = None
    if c["packed"]:
        ends = torch.cumsum(_lengths(n, b, seed), 0)
        st["cu_seqlens"] = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(dev, torch.int32)
    st["s_in"] = torch.randn(b, hk, dk, dv, generator=g, device=dev) if c["carry"] else None
    st["s_out"] = torch.empty(b, hk, dk, dv, device=dev)
    return st


# ---------------------------------------------------------------------------
# plain forms, in 32 bits
# ---------------------------------------------------------------------------

def _plain_rope_one(x, weight, cos, sin, rot, pairing):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight
    r = y[..., :rot]
    if pairing == "half":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([r, y[..., rot:]], -1).to(x.dtype)


def _plain_rope(st):
    c = st["case"]
    pos = st["positions"].reshape(c["axes"], -1).float()
    angle = (pos[st["axis"]] * st["inv_freq"][:, None]).t()[:, None, :]
    cos, sin = torch.cos(angle), torch.sin(angle)
    return [_plain_rope_one(st["q"], st["q_weight"], cos, sin, c["rot"], c["pairing"]),
            _plain_rope_one(st["k"], st["k_weight"], cos, sin, c["rot"], c["pairing"])]


def _plain_token(st):
    c = st["case"]
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    b, h, dk = q.shape
    hk, dv = v.shape[1:]
    s = st["s_in"] if st["slots"] is None else st["s_in"][st["slots"].long()]
    s = torch.exp(st["log_decay"])[:, None, None] * s + k[..., :, None] * v[..., None, :]
    o = torch.matmul(q.view(b, hk, h // hk, dk), s) * c["dk"] ** -0.5
    if st["slots"] is None:
        st["s_out"].copy_(s)
    else:
        st["s_out"][st["slots"].long()] = s
    return [o.reshape(b, h, dv).to(st["q"].dtype), st["s_out"]]


def _plain_dense(q, k, v, ld, s_in, chunk=128):
    """Chunked form: products inside a chunk, one product with the state that
    enters it.  Zero tokens fill up the front, so the last chunk ends at the
    last token."""
    b, n, h, dk = q.shape
    hk, dv = v.shape[2:]
    g = h // hk
    chunk = min(chunk, n)
    front = -n % chunk
    nc = (n + front) // chunk

    def cut(x):  # [b, n, heads, d] -> [b, hk, chunks, group * chunk, d]
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, front, 0))
        x = x.view(b, nc, chunk, hk, x.shape[2] // hk, x.shape[3])
        return x.permute(0, 3, 1, 4, 2, 5).reshape(b, hk, nc, -1, x.shape[-1])

    q, k, v = cut(q), cut(k), cut(v)
    t = torch.arange(chunk, device=q.device)
    gap = t[:, None] - t[None, :]
    ld1, ld2 = ld[:, None], ld[:, None, None]
    within = torch.exp(ld2 * gap.clamp(min=0)) * (gap >= 0)
    att = torch.matmul(q, k.transpose(-1, -2)).view(b, hk, nc, g, chunk, chunk)
    att = att * within[:, None, None]
    o = torch.matmul(att.view(b, hk, nc, g * chunk, chunk), v)
    left = torch.matmul((k * torch.exp(ld1 * (chunk - 1 - t))[:, None, :, None]).transpose(-1, -2), v)
    c = torch.arange(nc + 1, device=q.device)
    back = c[:, None] - 1 - c[None, :nc]
    across = torch.exp(ld2 * chunk * back.clamp(min=0)) * (back >= 0)
    s = torch.matmul(across, left.view(b, hk, nc, dk * dv)).view(b, hk, nc + 1, dk, dv)
    grow = torch.exp(ld1 * (t + 1)).repeat(1, g)[:, None, :, None]
    o = o + torch.matmul(q, s[:, :, :nc]) * grow
    last = s[:, :, nc]
    o = o.view(b, hk, nc, g, chunk, dv).permute(0, 2, 4, 1, 3, 5).reshape(b, nc * chunk, h, dv)[:, front:]
    if s_in is not None:
        i = torch.arange(n, device=q.device)
        qr = q.view(b, hk, nc, g, chunk, dk).permute(0, 1, 3, 2, 4, 5).reshape(b, hk, g, nc * chunk, dk)[:, :, :, front:]
        add = torch.matmul(qr, s_in[:, :, None]) * torch.exp(ld1 * (i + 1))[:, None, :, None]
        o = o + add.permute(0, 3, 1, 2, 4).reshape(b, n, h, dv)
        last = last + torch.exp(ld * n)[:, None, None] * s_in
    return o, last


def _plain_packed(q, k, v, ld, cu, chunk=128):
    """The chunked form over packed sequences: chunks of the whole row of
    tokens, in which only tokens of the same sequence meet."""
    n, h, dk = q.shape
    hk, dv = v.shape[1:]
    g = h // hk
    ns = cu.numel() - 1
    nc = -(-n // chunk)
    i = torch.arange(nc * chunk, device=q.device)
    seq = torch.searchsorted(cu[1:].long(), i, right=True).view(nc, chunk)

    def cut(x):
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, nc * chunk - n))
        x = x.view(nc, chunk, hk, x.shape[1] // hk, x.shape[2])
        return x.permute(2, 0, 3, 1, 4).reshape(hk, nc, -1, x.shape[-1])

    q, k, v = cut(q), cut(k), cut(v)
    t = torch.arange(chunk, device=q.device)
    gap = t[:, None] - t[None, :]
    ld1, ld2 = ld[:, None], ld[:, None, None]
    same = (gap >= 0) & (seq[:, :, None] == seq[:, None, :])
    within = torch.exp(ld2 * gap.clamp(min=0))[:, None] * same
    att = torch.matmul(q, k.transpose(-1, -2)).view(hk, nc, g, chunk, chunk) * within[:, :, None]
    o = torch.matmul(att.view(hk, nc, g * chunk, chunk), v)
    tail = seq[:, -1]
    keep = torch.exp(ld1 * (chunk - 1 - t))[:, None] * (seq == tail[:, None])
    left = torch.matmul((k * keep[..., None]).transpose(-1, -2), v)
    c = torch.arange(nc, device=q.device)
    back = c[:, None] - 1 - c[None, :]
    before = torch.cat([torch.full_like(tail[:1], -1), tail[:-1]])
    across = torch.exp(ld2 * chunk * back.clamp(min=0)) * ((back >= 0) & (before[:, None] == tail[None, :]))
    s = torch.matmul(across, left.view(hk, nc, dk * dv)).view(hk, nc, dk, dv)
    grow = torch.exp(ld1 * (t + 1))[:, None] * (seq == before[:, None])
    o = o + torch.matmul(q, s) * grow.repeat(1, 1, g)[..., None]
    o = o.view(hk, nc, g, chunk, dv).permute(1, 3, 0, 2, 4).reshape(nc * chunk, h, dv)[:n]
    end = cu[1:].long() - 1
    ce, off = end // chunk, end % chunk
    me = torch.arange(ns, device=q.device)
    mine = (t[None] <= off[:, None]) & (seq[ce] == me[:, None])
    w = torch.exp(ld2 * (off[:, None] - t[None]).clamp(min=0)) * mine
    last = torch.matmul((k[:, ce] * w[..., None]).transpose(-1, -2), v[:, ce])
    last = last + (torch.exp(ld1 * (off + 1)) * (before[ce] == me))[..., None, None] * s[:, ce]
    return o, last.transpose(0, 1)


def run(state):
    st, c = state, state["case"]
    if own:
        from catfuse_b200 import ops
        if c["op"] == "rope":
            return list(ops.qk_norm_rope(
                st["q"], st["k"], st["positions"], st["inv_freq"], q_weight=st["q_weight"],
                k_weight=st["k_weight"], norm=c["norm"], eps=1e-6, sections=_sections(c),
                axis_order=c["order"], pairing=c["pairing"]))
        if c["op"] == "token":
            o = ops.decay_attention_step(st["q"], st["k"], st["v"], st["log_decay"], st["s_in"],
                                         s_out=st["s_out"], slots=st["slots"])
        else:
            o = ops.decay_attention(st["q"], st["k"], st["v"], st["log_decay"], s_in=st["s_in"],
                                    s_out=st["s_out"], cu_seqlens=st["cu_seqlens"])
        return [o, st["s_out"]]
    if c["op"] == "rope":
        return _plain_rope(st)
    if c["op"] == "token":
        return _plain_token(st)
    if c["packed"]:
        o, s = _plain_packed(st["q"], st["k"], st["v"], st["log_decay"], st["cu_seqlens"])
    else:
        o, s = _plain_dense(st["q"], st["k"], st["v"], st["log_decay"], st["s_in"])
    st["s_out"].copy_(s)
    return [(o * c["dk"] ** -0.5).to(st["q"].dtype), st["s_out"]]


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its result from the definition in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    c = case
    h, hk = c["heads"], c["kv_heads"]
    if c["op"] == "rope":
        n, rows = c["tokens"], c["tokens"] * (h + hk)
        flops = rows * (3 * c["rot"] + (4 * c["dim"] if c["norm"] else 0))
        return {"bytes": rows * c["dim"] * 4 + 4 * n * c["axes"] + 2 * c["rot"] + (8 * c["dim"] if c["norm"] else 0),
                "flops": flops}
    b, dk, dv = c["batch"], c["dk"], c["dv"]
    n = b if c["op"] == "token" else b * c["length"]
    states = 2 if c["op"] == "token" or c["carry"] else 1
    data = 2 * n * (h * (dk + dv) + hk * (dk + dv)) + 4 * hk
    # each token: its key-value product joins the state, its queries read it
    return {"bytes": data + states * 4 * b * hk * dk * dv + (4 * (b + 1) if c.get("packed") else 0),
            "flops": n * (3 * hk + 2 * h) * dk * dv}


def _exact_sequence(q, k, v, ld, s0):
    """[n, h, d] of one sequence: every earlier token, weighted by its decay."""
    n, h, dk = q.shape
    hk = v.shape[1]
    at = torch.arange(n, device=q.device, dtype=torch.float64)
    out = torch.empty(n, h, v.shape[2], device=q.device, dtype=torch.float64)
    last = torch.empty(hk, dk, v.shape[2], device=q.device, dtype=torch.float64)
    for x in range(hk):
        a = ld[x]
        for lo in range(0, n, 2048):
            hi = min(n, lo + 2048)
            age = at[lo:hi, None] - at[None, :hi]
            w = torch.where(age >= 0, torch.exp(a * age.clamp(min=0)), 0.0)
            for y in range(x * (h // hk), (x + 1) * (h // hk)):
                row = ((q[lo:hi, y] @ k[:hi, x].T) * w) @ v[:hi, x]
                if s0 is not None:
                    row = row + torch.exp(a * (at[lo:hi, None] + 1)) * (q[lo:hi, y] @ s0[x])
                out[lo:hi, y] = row
        last[x] = (k[:, x] * torch.exp(a * (n - 1 - at))[:, None]).T @ v[:, x]
        if s0 is not None:
            last[x] += torch.exp(a * n) * s0[x]
    return out * dk ** -0.5, last


def exact(case, seed):
    c, st = case, prepare(case, seed)
    f = torch.float64
    q, k = st["q"].to(f), st["k"].to(f)
    if c["op"] == "rope":
        pos = st["positions"].reshape(c["axes"], -1).to(f)
        axis = _axis_of_pair(c)
        z = torch.polar(torch.ones((), device=q.device, dtype=f),
                        torch.stack([pos[a] * st["inv_freq"][p].to(f) for p, a in enumerate(axis)], -1))
        got = []
        for x, w in ((q, st["q_weight"]), (k, st["k_weight"])):
            if w is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + 1e-6) * w.to(f)
            half = c["rot"] // 2
            first = torch.arange(half, device=x.device) * (1 if c["pairing"] == "half" else 2)
            second = first + (half if c["pairing"] == "half" else 1)
            y = torch.complex(x[..., first], x[..., second]) * z[:, None]
            x = x.clone()
            x[..., first], x[..., second] = y.real, y.imag
            got.append(x)
        return got
    v, ld = st["v"].to(f), st["log_decay"].to(f)
    s_in = None if st["s_in"] is None else st["s_in"].to(f)
    if c["op"] == "token":
        at = torch.arange(c["batch"], device=q.device) if st["slots"] is None else st["slots"].long()
        s = torch.exp(ld).view(-1, 1, 1) * s_in[at] + torch.einsum("bhe,bhd->bhed", k, v)
        o = torch.einsum("bhge,bhed->bhgd", q.unflatten(1, (c["kv_heads"], -1)), s).flatten(1, 2)
        all_states = torch.zeros_like(s_in)
        all_states[at] = s
        return [o * c["dk"] ** -0.5, all_states]
    if c["packed"]:
        cu = st["cu_seqlens"].tolist()
        parts = [_exact_sequence(q[a:b], k[a:b], v[a:b], ld, None) for a, b in zip(cu, cu[1:])]
        return [torch.cat([p[0] for p in parts]), torch.stack([p[1] for p in parts])]
    parts = [_exact_sequence(q[b], k[b], v[b], ld, None if s_in is None else s_in[b])
             for b in range(c["batch"])]
    return [torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])]
