"""The operators of the 4-bit KV cache, as their speed is measured.

The cache holds keys and values as 4-bit floats (e2m1: magnitudes 0, 0.5, 1,
1.5, 2, 3, 4, 6 and a sign) in groups of 32 consecutive dimensions of a head
(16 where the head has 16) that share a power of two:

- the group's scale s is the smallest power of two with max|x| <= 7 s, within
  [2^-100, 2^125], stored as the byte log2(s) + 127; 255 marks a group that
  holds an infinity or a NaN, and all of it reads back as NaN;
- a code is x / s rounded to the nearest magnitude, halves to the even code,
  magnitudes above 6 to 6; the even dimension of a pair is the low half byte.

One sequence's rows are a slab of four planes: key codes [nkv][cap][hd / 2],
value codes, key scales [nkv][cap][groups], value scales; a batch is slabs at
a common stride.  Four kinds of pass:

- "write": f32 key and value rows are quantised into the cache; what the rows
  now stand for is read back;
- "read": a range of the cache as f32 rows;
- "attn": causal attention of `rows` query rows a sequence, the first at
  position pos, over the cache, which holds the rows' keys already; a slot
  with pos -1 is idle, its output is zeros;
- "step": the rows' keys and values are appended first, as a decode step does,
  and what they stand for is returned beside the attention's output.
"""
from __future__ import annotations

import math

import torch

own = False

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# head layouts: query heads, KV heads, head dim
HEADS = {
    "1b": (16, 8, 128),
    "4b": (32, 8, 128),
    "tiny": (4, 2, 16),
    "h32": (6, 6, 32),
    "h64": (16, 2, 64),
    "h256": (8, 4, 256),
}


def _case(name, kind, heads, cap, pos, rows):
    return {"name": name, "kind": kind, "heads": heads, "cap": cap, "pos": pos, "rows": rows}


def listed():
    return [
        # one token of the benchmark's 64-token prompt + 256 steps: latency
        _case("attn_1b_ctx320", "attn", "1b", 512, "319", 1),
        # a decode step behind the benchmark's longest prompt
        _case("step_1b_ctx8k", "step", "1b", 8448, "8299", 1),
        # drafts for a queue of requests of mixed lengths, two slots idle
        _case("attn_4b_batch14", "attn", "4b", 1024, "64,17,160,-1,90,33,210,48,75,120,-1,29,1003,140", 1),
        # long documents, one of them just begun
        _case("attn_1b_long4", "attn", "1b", 131072, "100000,65,131070,40001", 1),
        # a serving batch in the middle of its requests
        _case("step_4b_batch48", "step", "4b", 4096, ",".join(str(37 + (i * 1117) % 4011) for i in range(48)), 1),
        # a turn of a conversation over a document
        _case("attn_1b_turn45", "attn", "1b", 2112, "1630", 45),
        # prompts: a page or two, and the benchmark's longest
        _case("attn_1b_prompt1000", "attn", "1b", 1024, "0", 1000),
        _case("attn_1b_prompt8192", "attn", "1b", 8192, "0", 8192),
        # the rows of a serving batch's step, and of the longest prompt
        _case("write_4b_batch48", "write", "4b", 4096, ",".join(str(37 + (i * 1117) % 4011) for i in range(48)), 1),
        _case("write_1b_prompt8192", "write", "1b", 8448, "0", 8192),
        # a kept prefix for a program that works on f32 rows, and a piece of
        # the smallest model's cache
        _case("read_1b_ctx8k", "read", "1b", 8448, "0", 8191),
        _case("read_tiny_301", "read", "tiny", 512, "17", 301),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "step", "step", "write", "read"])
    heads = rng.choice(["1b", "1b", "4b", "4b", "tiny", "h32", "h64", "h256"])
    nq, nkv, hd = HEADS[heads]
    if kind in ("write", "read"):
        seqs = _log(rng, 1, 64)
        rows = _log(rng, 1, max(1, 8192 * 1024 // (seqs * nkv * hd)))
    elif rng.random() < 0.6:
        seqs, rows = _log(rng, 1, 64), 1
    else:
        seqs, rows = rng.choice([1, 1, 1, 2, 3]), _log(rng, 2, 2500)
    # contexts as long as the largest listed case's bytes and products allow
    most = min(131072, 2 ** 28 // (seqs * nkv * hd), 2 ** 36 // (seqs * rows * nq * hd))
    pos = [_log(rng, 1, max(1, most)) - 1 for _ in range(seqs)]
    if kind == "attn" and seqs > 2:
        pos[rng.randrange(seqs)] = -1
    cap = max(pos) + rows + rng.choice([0, 1, 13, 64, 500])
    c = _case("", kind, heads, cap, ",".join(map(str, pos)), rows)
    del c["name"]
    return c


def _shape(case):
    nq, nkv, hd = HEADS[case["heads"]]
    pos = [int(x) for x in case["pos"].split(",")]
    return nq, nkv, hd, max(1, hd // 32), case["cap"], pos, case["rows"]


# ---- the cache in torch --------------------------------------------------------

def _quantise(x, groups):
    """Codes [..., hd / 2] and scale bytes [..., groups] of x [..., hd]."""
    g = x.unflatten(-1, (groups, -1))
    bits = g.abs().amax(-1).view(torch.int32)
    # the exponent that puts the maximum into (3.5, 7]
    e = (bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x600000).int()
    e = e.clamp(27, 252)
    bad = ~torch.isfinite(g).all(-1)
    r = torch.where(bad[..., None], torch.zeros_like(g), g) / (e << 23).view(torch.float32)[..., None]
    a = r.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (r < 0)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.where(bad, torch.full_like(e, 255), e).to(torch.uint8)


def _planes(slab, case):
    """Codes [seq, 2, nkv, cap, hd / 2] and scales [seq, 2, nkv, cap, groups]."""
    _, nkv, hd, groups, cap, _, _ = _shape(case)
    n = nkv * cap * hd
    return (slab[:, :n].unflatten(1, (2, nkv, cap, hd // 2)),
            slab[:, n:n + 2 * nkv * cap * groups].unflatten(1, (2, nkv, cap, groups)))


def _values(codes, scales):
    """What codes [..., hd / 2] with scale bytes [..., groups] stand for."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2)
    s = (scales.int() << 23).view(torch.float32).masked_fill(scales == 255, math.nan)
    return (v.unflatten(-1, (scales.shape[-1], -1)) * s[..., None]).flatten(-2)


# ---- inputs ----------------------------------------------------------------------

def _rows(gen, shape, hd, keys):
    """Key or value rows [..., nkv, hd]: a few key channels are some times
    larger than the rest, and values differ in size by token."""
    x = torch.randn(shape + (hd,), generator=gen, device="cuda")
    if keys:
        wide = torch.rand(hd, generator=gen, device="cuda") < 0.05
        return x * torch.where(wide, 6.0, 1.0)
    return x * torch.exp(0.5 * torch.randn(shape + (1,), generator=gen, device="cuda"))


def prepare(case, seed):
    nq, nkv, hd, groups, cap, pos, rows = _shape(case)
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    seqs = len(pos)
    size = (nkv * cap * (hd + 2 * groups) + 15) // 16 * 16
    slab = torch.zeros(seqs, size, dtype=torch.uint8, device="cuda")
    codes, scales = _planes(slab, case)
    if case["kind"] != "write":
        for b in range(seqs):
            for i in range(2):
                codes[b, i], scales[b, i] = _quantise(_rows(gen, (nkv, cap), hd, i == 0), groups)
    s = {"case": case, "slab": slab, "pos": torch.tensor(pos, dtype=torch.int32, device="cuda")}
    if case["kind"] in ("write", "step"):
        for i, name in enumerate(("k", "v")):
            s[name] = _rows(gen, (seqs, rows, nkv), hd, i == 0).flatten(-2)
    if case["kind"] in ("attn", "step"):
        s["q"] = torch.randn(seqs, rows, nq * hd, generator=gen, device="cuda")
        s["out"] = torch.empty_like(s["q"])
    if case["kind"] != "attn":
        s["k_read"] = torch.empty(seqs, rows, nkv * hd, device="cuda")
        s["v_read"] = torch.empty_like(s["k_read"])
    return s


# ---- one pass ----------------------------------------------------------------------

def _write(s):
    _, _, hd, groups, _, pos, rows = _shape(s["case"])
    codes, scales = _planes(s["slab"], s["case"])
    new = torch.stack((s["k"], s["v"]), 2).unflatten(-1, (-1, hd))
    c, e = _quantise(new, groups)
    at = s["pos"].long()[:, None] + torch.arange(rows, device="cuda")
    seq = torch.arange(len(pos), device="cuda")[:, None]
    codes[seq, :, :, at] = c
    scales[seq, :, :, at] = e


def _read(s):
    _, _, _, _, _, pos, rows = _shape(s["case"])
    codes, scales = _planes(s["slab"], s["case"])
    at = s["pos"].long()[:, None] + torch.arange(rows, device="cuda")
    seq = torch.arange(len(pos), device="cuda")[:, None]
    v = _values(codes[seq, :, :, at], scales[seq, :, :, at])
    return v[:, :, 0].flatten(2), v[:, :, 1].flatten(2)


def _attend(s):
    nq, nkv, hd, _, _, pos, rows = _shape(s["case"])
    codes, scales = _planes(s["slab"], s["case"])
    n = max(1, max(pos) + rows)
    kv = _values(codes[:, :, :, :n], scales[:, :, :, :n])
    q = s["q"].unflatten(-1, (nkv, nq // nkv, hd)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    a = torch.matmul(q, kv[:, 0].transpose(-1, -2).contiguous()) / math.sqrt(hd)
    last = s["pos"][:, None] + torch.arange(rows, device="cuda")
    hidden = (torch.arange(n, device="cuda") > last[..., None]) | (s["pos"] < 0)[:, None, None]
    a = a.unflatten(2, (nq // nkv, rows)).masked_fill_(hidden[:, None, None], -math.inf)
    top = a.amax(-1, keepdim=True)
    p = torch.exp(a - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), kv[:, 1].contiguous()).unflatten(2, (nq // nkv, rows))
    o = torch.where(total == 0, torch.zeros_like(o), o / total)
    return o.permute(0, 3, 1, 2, 4).flatten(2)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        return _own(s)
    if kind in ("write", "step"):
        _write(s)
    out = [_attend(s)] if kind in ("attn", "step") else []
    return out + (list(_read(s)) if kind != "attn" else [])


def _own(s):
    import tinyminigo_amd as T

    nq, nkv, hd, _, cap, pos, rows = _shape(s["case"])
    kind, stream = s["case"]["kind"], torch.cuda.current_stream().cuda_stream
    if "kv" not in s:
        # the cache's description and the attention's workspace, kept by a program
        s["kv"] = T.Kv4(s["slab"].data_ptr(), cap=cap, nkv=nkv, hd=hd, n_seq=len(pos), seq_stride=s["slab"].shape[1])
        if kind in ("attn", "step"):
            s["ws"] = torch.zeros(T.kv4_attn_workspace(s["kv"], rows, nq), dtype=torch.uint8, device="cuda")
    kv = s["kv"]
    # one sequence's position is known to the program, a batch's are on the device
    at = {"pos": pos[0]} if len(pos) == 1 else {"pos_dev": s["pos"].data_ptr()}
    new = (s["k"].data_ptr(), s["v"].data_ptr()) if kind in ("write", "step") else (0, 0)
    out = []
    if kind == "write":
        T.kv4_write(kv, new[0], new[1], rows, stream=stream, **at)
    elif kind in ("attn", "step"):
        T.kv4_attn(kv, s["q"].data_ptr(), s["out"].data_ptr(), rows, nq, k_dev=new[0], v_dev=new[1],
                   ws_dev=s["ws"].data_ptr(), ws_bytes=s["ws"].numel(), stream=stream, **at)
        out.append(s["out"])
    if kind != "attn":
        T.kv4_read(kv, s["k_read"].data_ptr(), s["v_read"].data_ptr(), rows, stream=stream, **at)
        out += [s["k_read"], s["v_read"]]
    return out


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    nq, nkv, hd, groups, _, pos, rows = _shape(case)
    live = [p for p in pos if p >= 0]
    row4 = 2 * nkv * (hd // 2 + groups)  # a cached position
    row32 = 2 * nkv * hd * 4             # the same as f32 rows
    nbytes, flops = 0, 0
    if case["kind"] in ("write", "step"):
        nbytes += len(live) * rows * (row32 + row4)
    if case["kind"] in ("attn", "step"):
        nbytes += len(pos) * rows * 2 * nq * hd * 4
        nbytes += sum((p + (rows if case["kind"] == "attn" else 0)) * row4 for p in live)
        flops += sum(4 * nq * hd * (rows * p + rows * (rows + 1) // 2) for p in live)
    if case["kind"] != "attn":
        nbytes += len(live) * rows * (row32 + (row4 if case["kind"] == "read" else 0))
    return {"bytes": nbytes, "flops": flops}


# ---- the same in 64 bits -----------------------------------------------------------

def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest64(x, groups):
    """The values that x's codes and scales stand for, from the definition."""
    g = x.double().unflatten(-1, (groups, -1))
    top = g.abs().amax(-1, keepdim=True)
    frac, e = torch.frexp(top / 7)
    e = torch.where(frac == 0.5, e - 1, e).clamp(-100, 125)
    s = _power64(e)
    out = torch.zeros_like(g)
    a = g.abs() / s
    near = torch.full_like(a, math.inf)
    # even codes first, so that a half stays with them
    for m in MAGNITUDES[0::2] + MAGNITUDES[1::2]:
        d = (a - m).abs()
        out = torch.where(d < near, torch.full_like(out, m), out)
        near = torch.minimum(near, d)
    return (torch.copysign(out, g) * s).flatten(-2)


def _decoded64(slab, case, b, i, upto):
    """Keys (i = 0) or values of one sequence's first positions [nkv, upto, hd]."""
    _, nkv, hd, groups, cap, _, _ = _shape(case)
    n = nkv * cap * hd // 2
    c = slab[b, i * n:(i + 1) * n].view(nkv, cap, hd // 2)[:, :upto].long()
    at = 2 * n + i * nkv * cap * groups
    e = slab[b, at:at + nkv * cap * groups].view(nkv, cap, groups)[:, :upto]
    v = torch.empty(nkv, upto, hd, dtype=torch.float64, device=slab.device)
    for half in range(2):
        code = (c >> (4 * half)) & 15
        m = code & 7
        # subnormal codes 0 and 1 are 0 and 0.5; the others (1 + m / 2) 2^(e - 1)
        mag = torch.where(m < 2, 0.5 * m, (1 + 0.5 * (m & 1)) * _power64((m >> 1) - 1))
        v[..., half::2] = torch.where(code >= 8, -mag, mag)
    return v * _power64(e.long() - 127).repeat_interleave(hd // groups, -1)


def exact(case, seed):
    s = prepare(case, seed)
    nq, nkv, hd, groups, cap, pos, rows = _shape(case)
    seqs, group = len(pos), nq // nkv
    new = None
    if case["kind"] in ("write", "step"):
        new = [_nearest64(s[n].unflatten(-1, (nkv, hd)), groups) for n in ("k", "v")]  # [seq, rows, nkv, hd]
    out = []
    if case["kind"] in ("attn", "step"):
        o = torch.zeros(seqs, rows, nkv, group, hd, dtype=torch.float64, device="cuda")
        for b, p in enumerate(pos):
            if p < 0:
                continue
            k, v = (_decoded64(s["slab"], case, b, i, p + rows) for i in range(2))
            if new is not None:
                k[:, p:], v[:, p:] = new[0][b].transpose(0, 1), new[1][b].transpose(0, 1)
            q = s["q"][b].double().view(rows, nkv, group, hd)
            late = torch.arange(p + rows, device="cuda")[None] > p + torch.arange(rows, device="cuda")[:, None]
            for g in range(nkv):
                kt = k[g].t().contiguous()
                for h in range(group):
                    w = (q[:, g, h] @ kt / math.sqrt(hd)).masked_fill(late, -math.inf).softmax(-1)
                    o[b, :, g, h] = w @ v[g]
        out.append(o.view(seqs, rows, nq * hd))
    if new is not None:
        out += [x.flatten(2) for x in new]
    elif case["kind"] == "read":
        for i in range(2):
            rows_of = [_decoded64(s["slab"], case, b, i, p + rows)[:, p:] for b, p in enumerate(pos)]
            out.append(torch.stack([r.transpose(0, 1).flatten(1) for r in rows_of]))
    return out
