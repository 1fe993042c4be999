"""Timing cases of the operators for serving many sequences out of a paged cache, and of the head norms of queries and keys.

A case is one pass through one operator:

  norm      RMS norm of every head of the queries and keys of a layer with its rotation (``CudaDnn.QkNormRopeForward``)
  norm_bwd  the gradient of that: of queries, keys and both weights (``QkNormRopeBackward``)
  append    new tokens into the cache: rows of the q | k | v projection normalised, rotated, keys and values stored in the pages
            that a block table names (``PagedAppend``)
  paged     attention of the new tokens of every sequence over its pages, one token or a chunk each (``AttnPagedForward``)

The plain forms are written with elementary torch operations in 32 bits; angles are taken in 64.
"""
import ctypes
import math
import random  # noqa: F401  (draw takes a random.Random)

import numpy as np
import torch

own = False

EPS = 1e-5
THETA = 10000.0


def listed():
    return [
        # a prompt of five tokens through a narrow model's layer: nothing but the call
        dict(name="norm_f32_small", kind="norm", act="f32", B=1, T=5, H=6, kvH=6, hs=48),
        # a training step's queries and keys of a 768-wide layer, 16-bit storage
        dict(name="norm_bf16_train", kind="norm", act="bf16", B=8, T=1024, H=12, kvH=12, hs=64),
        # gradients in a 288-wide model's training step, sequences that are no power of two
        dict(name="norm_bwd_f32", kind="norm_bwd", act="f32", B=4, T=700, H=6, kvH=6, hs=48),
        # gradients at the width of a large model, four query heads to a key head
        dict(name="norm_bwd_bf16", kind="norm_bwd", act="bf16", B=4, T=2048, H=32, kvH=8, hs=128),
        # a decoding step: one new token of each of sixteen sequences
        dict(name="append_bf16_step", kind="append", act="bf16", cache="bf16", norm=True, B=16, new=1, len=900, ragged=True, pad=0, page=16, order="head",
             dropped=0, H=12, kvH=12, hs=64),
        # chunks of six prompts, activations in 32 bits over a 16-bit cache, a padded batch, no norms
        dict(name="append_f32_chunk", kind="append", act="f32", cache="bf16", norm=False, B=6, new=400, len=2500, ragged=True, pad=37, page=32, order="pos",
             dropped=0, H=12, kvH=4, hs=64),
        # a scheduler's full step of prompt tokens in 16-bit storage
        dict(name="append_bf16_chunk", kind="append", act="bf16", cache="bf16", norm=True, B=8, new=1024, len=4096, ragged=False, pad=0, page=16,
             order="head", dropped=0, H=32, kvH=8, hs=128),
        # one user's next token over a short history
        dict(name="paged_f32_one", kind="paged", act="f32", cache="f32", B=1, new=1, len=100, ragged=False, pad=0, page=16, order="head", dropped=0, H=12,
             kvH=12, hs=64),
        # a decoding step of many users, lengths of all kinds
        dict(name="paged_bf16_step", kind="paged", act="bf16", cache="bf16", B=64, new=1, len=4096, ragged=True, pad=0, page=16, order="head", dropped=0,
             H=32, kvH=8, hs=128),
        # one token over a very long history
        dict(name="paged_bf16_long", kind="paged", act="bf16", cache="bf16", B=1, new=1, len=131000, ragged=False, pad=0, page=64, order="pos", dropped=0,
             H=32, kvH=8, hs=128),
        # chunks of prompts over what is cached of them
        dict(name="paged_bf16_chunk", kind="paged", act="bf16", cache="bf16", B=4, new=1024, len=8192, ragged=False, pad=0, page=32, order="head", dropped=0,
             H=32, kvH=8, hs=128),
        # chunks and single tokens side by side in 32 bits, the oldest pages given up
        dict(name="paged_f32_mixed", kind="paged", act="f32", cache="f32", B=12, new=300, len=1500, ragged=True, pad=5, page=16, order="pos", dropped=3, H=12,
             kvH=12, hs=64),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_bwd", "append", "paged", "paged", "paged"])
    hs = rng.choice([32, 48, 64, 64, 96, 128, 128])
    kvH = rng.randint(1, 12)
    H = kvH * rng.choice([1, 1, 2, 4, 7, 8])
    if H > 40:
        H = kvH
    if kind in ("norm", "norm_bwd"):
        T = _log(rng, 1, 2048)
        return dict(kind=kind, act=rng.choice(["f32", "bf16"]), B=_log(rng, 1, max(1, min(32, 8192 // T))), T=T, H=H, kvH=kvH, hs=hs)
    act, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "bf16")])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    new = rng.choice([1, 1, _log(rng, 2, 1024), _log(rng, 2, 1024)])
    room = 262144 if kind == "paged" and new == 1 and act == "bf16" else 32768
    length = _log(rng, new, 8192 if new > 1 else 65536 if room > 65536 else 16384)
    # no more cache than the largest listed case reads
    values = 4 * kvH * hs * (2 if cache == "f32" else 1)
    B = _log(rng, 1, max(1, min(128, room // length, 4096 // new, 500_000_000 // (values * length))))
    return dict(kind=kind, act=act, cache=cache, B=B, new=new, len=length, ragged=rng.random() < 0.7, pad=rng.choice([0, 0, rng.randint(1, 40)]), page=page,
                order=rng.choice(["head", "pos"]), dropped=rng.choice([0, 0, 0, rng.randint(1, 4)]), H=H, kvH=kvH, hs=hs,
                **({"norm": rng.random() < 0.6} if kind == "append" else {}))


# ---- what the sizes of a case say ----------------------------------------------------------------------------------------
def _sequences(c):
    """New tokens and cached positions (the new ones among them) of every sequence."""
    new, lens = [], []
    for b in range(c["B"]):
        f = (0.37 + 0.6180339887 * b) % 1.0 if c["ragged"] else 1.0
        # ragged: every third sequence of a step with chunks has a single new token, the others up to a whole chunk
        n = c["new"] if not c["ragged"] else 1 if b % 3 == 2 else max(1, int(c["new"] * (0.3 + 0.7 * f)))
        new.append(n)
        lens.append(max(n, int(c["len"] * (0.05 + 0.95 * f))) if c["ragged"] else max(n, c["len"]))
    return new, lens


def _dropped(c, length, n):
    """Positions of a sequence's oldest pages that are given up: whole pages, none that a new token is in."""
    return min(c["dropped"], (length - n) // c["page"]) * c["page"]


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)

    act, H, kvH, hs = _type(c["act"]), c["H"], c["kvH"], c["hs"]
    i = {}
    if c["kind"] in ("norm", "norm_bwd"):
        B, T = c["B"], c["T"]
        i["q"], i["k"] = normal(B, H, T, hs, std=1.5, dtype=act), normal(B, kvH, T, hs, std=1.5, dtype=act)
        i["wq"], i["wk"] = normal(hs, std=0.2, mean=1.0, dtype=act), normal(hs, std=0.2, mean=1.0, dtype=act)
        if c["kind"] == "norm_bwd":
            i["dq"], i["dk"] = normal(B, H, T, hs, dtype=act), normal(B, kvH, T, hs, dtype=act)
        return i
    new, lens = _sequences(c)
    page, cache = c["page"], _type(c["cache"])
    width = max(-(-n // page) for n in lens) + 1
    need = sum(-(-n // page) for n in lens)
    pages = need + 3
    # where the pages lie is what earlier requests left: any order; entries past a sequence's end name no page
    order = torch.randperm(pages, generator=g, device="cuda")[:need].cpu().numpy()
    table, at = np.full((c["B"], width), -1.0, np.float32), 0
    for b, n in enumerate(lens):
        count = -(-n // page)
        table[b, :count] = order[at:at + count]
        table[b, :_dropped(c, n, new[b]) // page] = -1.0
        at += count
    i["table"] = torch.from_numpy(table).cuda()
    i["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.float32, device="cuda")
    i["lens"] = torch.tensor(lens, dtype=torch.float32, device="cuda")
    tokens = sum(new) + c["pad"]
    shape = (pages, kvH, page, hs) if c["order"] == "head" else (pages, page, kvH, hs)
    i["kp"], i["vp"] = normal(*shape, dtype=cache), normal(*shape, dtype=cache)
    if c["kind"] == "append":
        i["qkv"] = normal(tokens, (H + 2 * kvH) * hs, dtype=act)
        if c["norm"]:
            i["wq"], i["wk"] = normal(hs, std=0.2, mean=1.0, dtype=act), normal(hs, std=0.2, mean=1.0, dtype=act)
    else:
        i["q"] = normal(tokens, H, hs, dtype=act)
    return i


def _tokens(c):
    return sum(_sequences(c)[0]) + c["pad"]


def _strides(c):
    """Elements from page to page, head to head, position to position."""
    whole = c["kvH"] * c["page"] * c["hs"]
    return (whole, c["page"] * c["hs"], c["hs"]) if c["order"] == "head" else (whole, c["hs"], c["kvH"] * c["hs"])


def _by_head(c, pages):
    """A view (pages, heads, positions, values) of the cache."""
    return pages if c["order"] == "head" else pages.permute(0, 2, 1, 3)


# ---- the framework's side: one device context, memory behind handles ---------------------------------------------------------
_context = []


def _cuda():
    if not _context:
        from mycaffe_amd.cudadnn import CudaDnn
        _context.append(CudaDnn(0))
    return _context[0]


class _Handles:
    """Device memory of the framework; freed once neither the state nor a view of it is left."""

    def __init__(self, cuda):
        self.cuda, self.memory, self.ropes = cuda, [], []

    def __del__(self):
        try:
            for h in self.memory:
                self.cuda.FreeMemory(h)
            for h in self.ropes:
                self.cuda.FreeRope(h)
        except Exception:
            pass


class _Memory:
    """Memory behind a handle, for torch (no copy)."""

    def __init__(self, owner, handle, shape, half):
        get = owner.cuda._lib.Internal_GetPointerFloat
        get.argtypes = [ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.POINTER(ctypes.c_void_p)]
        p = ctypes.c_void_p()
        if get(0, owner.cuda.m_hKernel, int(handle), ctypes.byref(p)) != 0 or not p.value:
            raise RuntimeError("no address behind memory handle %d" % handle)
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<i2" if half else "<f4", "data": (p.value, False), "version": 2}


def _empty(owner, shape, dtype):
    half = dtype == torch.bfloat16
    h = owner.cuda.AllocMemory(int(math.prod(shape)), bHalfSize=half)
    owner.memory.append(h)
    v = torch.as_tensor(_Memory(owner, h, shape, half), device="cuda")
    return h, v.view(torch.bfloat16) if half else v


def prepare(case, seed):
    c, i = dict(case), _inputs(case, seed)
    act, H, kvH, hs = _type(c["act"]), c["H"], c["kvH"], c["hs"]
    # outputs that a program keeps room for (the cache is both)
    out = {}
    if c["kind"] in ("norm", "norm_bwd"):
        out = {"yq": tuple(i["q"].shape), "yk": tuple(i["k"].shape)}
        if c["kind"] == "norm_bwd":
            out = {"xq": out["yq"], "xk": out["yk"], "gq": (hs,), "gk": (hs,)}
    else:
        out = {"y": (_tokens(c), H, hs)}
    if not own:
        s = dict(case=c, **i)
        if "y" in out:
            s["y"] = torch.zeros(out["y"], dtype=act, device="cuda")
        return s
    cuda = _cuda()
    owner = _Handles(cuda)
    s = dict(case=c, cuda=cuda, owner=owner, h={}, v={})
    for name, t in i.items():
        s["h"][name], s["v"][name] = _empty(owner, tuple(t.shape), t.dtype)
        s["v"][name].copy_(t)
    for name, shape in out.items():
        s["h"][name], s["v"][name] = _empty(owner, shape, act)
        s["v"][name].zero_()
    # the rotation's handle, of as many positions as a sequence can have
    positions = c["T"] if "T" in c else i["table"].shape[1] * c["page"]
    if c["kind"] != "paged":
        s["rope"] = cuda.CreateRope(0, 0, positions * H * hs, 1, positions, H, hs, THETA)
        owner.ropes.append(s["rope"])
    if "table" in i:
        s["pages"], s["width"], s["tokens"] = i["kp"].shape[0], i["table"].shape[1], _tokens(c)
    torch.cuda.synchronize()
    return s


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


# ---- the framework's calls ---------------------------------------------------------------------------------------------------
def _own_norm(s):
    c, h = s["case"], s["h"]
    s["cuda"].QkNormRopeForward(c["B"], c["T"], c["H"], c["kvH"], c["hs"], h["q"], h["k"], h["wq"], h["wk"], h["yq"], h["yk"], s["rope"], EPS)
    return [s["v"]["yq"], s["v"]["yk"]]


def _own_norm_bwd(s):
    c, h = s["case"], s["h"]
    s["cuda"].QkNormRopeBackward(c["B"], c["T"], c["H"], c["kvH"], c["hs"], h["q"], h["k"], h["wq"], h["wk"], h["dq"], h["dk"], h["xq"], h["xk"], h["gq"],
                                 h["gk"], s["rope"], EPS)
    return [s["v"][n] for n in ("xq", "xk", "gq", "gk")]


def _own_append(s):
    c, h = s["case"], s["h"]
    s["cuda"].PagedAppend(c["B"], s["tokens"], c["H"], c["kvH"], c["hs"], s["pages"], c["page"], s["width"], h["qkv"], h["y"], h["kp"], h["vp"], h["table"],
                          h["starts"], h["lens"], *_strides(c), s["rope"], c["norm"], h.get("wq", 0), h.get("wk", 0), EPS)
    return [s["v"]["y"], s["v"]["kp"], s["v"]["vp"]]


def _own_paged(s):
    c, h = s["case"], s["h"]
    s["cuda"].AttnPagedForward(c["B"], s["tokens"], c["H"], c["kvH"], c["hs"], s["pages"], c["page"], s["width"], h["q"], h["kp"], h["vp"], h["table"],
                               h["starts"], h["lens"], h["y"], *_strides(c))
    return s["v"]["y"]


# ---- plain forms: elementary operations in 32 bits ----------------------------------------------------------------------------
def _turns(positions, hs):
    """Cosines and sines of a list of positions, (n, hs / 2); angles in 64 bits."""
    f = THETA ** (-torch.arange(0, hs, 2, dtype=torch.float64, device="cuda") / hs)
    a = positions.double()[:, None] * f
    return torch.cos(a).float(), torch.sin(a).float()


def _rotate(x, cos, sin):
    """Adjacent pairs of the last axis by the angles whose cosines and sines broadcast against them."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(x.shape)


def _normalise(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_norm(s):
    c = s["case"]
    cos, sin = _turns(torch.arange(c["T"], device="cuda"), c["hs"])
    return [_rotate(_normalise(s[x].float(), s[w].float()), cos, sin).to(s[x].dtype) for x, w in (("q", "wq"), ("k", "wk"))]


def _plain_norm_bwd(s):
    c = s["case"]
    cos, sin = _turns(torch.arange(c["T"], device="cuda"), c["hs"])
    dx, dw = [], []
    for n in "qk":
        x, w, g = s[n].float(), s["w" + n].float(), _rotate(s["d" + n].float(), cos, -sin)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xr, gw = x * r, g * w
        dx.append((r * (gw - xr * (gw * xr).mean(-1, keepdim=True))).to(s[n].dtype))
        # a long sum: in 64 bits
        dw.append((g * xr).sum((0, 1, 2), dtype=torch.float64).to(s[n].dtype))
    return dx + dw


def _plain_append(s):
    c = s["case"]
    H, kvH, hs, page = c["H"], c["kvH"], c["hs"], c["page"]
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1]
    total = int(_tokens(c)) - c["pad"]
    seq = torch.repeat_interleave(torch.arange(c["B"], device="cuda"), new, output_size=total)
    pos = torch.arange(total, device="cuda") - starts[seq] + (lens - new)[seq]
    x = s["qkv"][:total].float().reshape(total, H + 2 * kvH, hs)
    q, k, v = x[:, :H], x[:, H:H + kvH], x[:, H + kvH:]
    if c["norm"]:
        q, k = _normalise(q, s["wq"].float()), _normalise(k, s["wk"].float())
    cos, sin = (t[:, None] for t in _turns(pos, hs))
    s["y"][:total] = _rotate(q, cos, sin).to(s["y"].dtype)
    at, slot = s["table"][seq, pos // page].long(), pos % page
    _by_head(c, s["kp"])[at, :, slot] = _rotate(k, cos, sin).to(s["kp"].dtype)
    _by_head(c, s["vp"])[at, :, slot] = v.to(s["vp"].dtype)
    return [s["y"], s["kp"], s["vp"]]


def _plain_paged(s):
    c = s["case"]
    H, kvH, hs, page = c["H"], c["kvH"], c["hs"], c["page"]
    G, scale = H // kvH, 1.0 / math.sqrt(hs)
    kp, vp = _by_head(c, s["kp"]), _by_head(c, s["vp"])
    at = 0
    for b, (n, length) in enumerate(zip(*_sequences(c))):
        gone = _dropped(c, length, n)
        pages = s["table"][b, gone // page:-(-length // page)].long()
        have = length - gone
        k = kp[pages].permute(1, 3, 0, 2).reshape(kvH, hs, -1)[:, :, :have].float()     # (heads, values, positions)
        v = vp[pages].permute(1, 0, 2, 3).reshape(kvH, -1, hs)[:, :have].float()
        q = s["q"][at:at + n].float().reshape(n, kvH, G, hs).permute(1, 0, 2, 3).reshape(kvH, n * G, hs) * scale
        scores = torch.matmul(q.contiguous(), k.contiguous())
        if n > 1:
            last = torch.arange(have - n, have, device="cuda").repeat_interleave(G)
            scores = scores.masked_fill(torch.arange(have, device="cuda")[None, :] > last[:, None], float("-inf"))
        w = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.matmul(w, v.contiguous()) / w.sum(-1, keepdim=True)
        s["y"][at:at + n] = o.reshape(kvH, n, G, hs).permute(1, 0, 2, 3).reshape(n, H, hs).to(s["y"].dtype)
        at += n
    return s["y"]


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------
def _turned(x, pos, back=False):
    """exp(i angle) times the pairs of x as complex numbers; pos broadcasts against x without its last axis."""
    hs = x.shape[-1]
    z = torch.view_as_complex(x.double().contiguous().reshape(*x.shape[:-1], hs // 2, 2))
    inverse = torch.tensor([THETA ** (-2.0 * j / hs) for j in range(hs // 2)], dtype=torch.float64, device=x.device)
    angle = pos.double().unsqueeze(-1) * inverse
    z = z * torch.polar(torch.ones_like(angle), -angle if back else angle)
    return torch.view_as_real(z).reshape(x.shape)


def _exact_head_norm(x, w):
    x = x.double()
    return w.double() * x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS)


def exact(case, seed):
    c, i = dict(case), _inputs(case, seed)
    if c["kind"] == "norm":
        t = torch.arange(c["T"], device="cuda")
        return [_turned(_exact_head_norm(i[n], i["w" + n]), t) for n in "qk"]
    if c["kind"] == "norm_bwd":
        t = torch.arange(c["T"], device="cuda")
        dx, dw = [], []
        for n in "qk":
            x, w, g = i[n].double(), i["w" + n].double(), _turned(i["d" + n], t, back=True)
            ms = x.pow(2).sum(-1, keepdim=True) / c["hs"] + EPS
            # y_j = w_j x_j ms^(-1/2): dy_j / dx_l = w_j (delta_jl ms^(-1/2) - x_j x_l ms^(-3/2) / hs)
            dx.append(g * w * ms.pow(-0.5) - x * (g * w * x).sum(-1, keepdim=True) * ms.pow(-1.5) / c["hs"])
            dw.append((g * x * ms.pow(-0.5)).reshape(-1, c["hs"]).sum(0))
        return dx + dw
    new, lens = _sequences(c)
    H, kvH, hs, page = c["H"], c["kvH"], c["hs"], c["page"]
    table = i["table"].cpu().numpy().astype(np.int64)
    if c["kind"] == "append":
        total = sum(new)
        pos = torch.tensor([p for n, m in zip(new, lens) for p in range(m - n, m)], device="cuda")
        where = torch.tensor([[table[b, p // page], p % page] for b, (n, m) in enumerate(zip(new, lens)) for p in range(m - n, m)], device="cuda")
        x = i["qkv"][:total].reshape(total, H + 2 * kvH, hs).double()
        q, k, v = x.split([H, kvH, kvH], 1)
        if c["norm"]:
            q, k = _exact_head_norm(q, i["wq"]), _exact_head_norm(k, i["wk"])
        y = torch.zeros(total + c["pad"], H, hs, dtype=torch.float64, device="cuda")
        y[:total] = _turned(q, pos[:, None])
        stored = []
        for pages, rows in ((i["kp"], _turned(k, pos[:, None])), (i["vp"], v)):
            full = pages.double()
            flat = full if c["order"] == "pos" else full.transpose(1, 2).contiguous()
            flat[where[:, 0], where[:, 1]] = rows
            stored.append(flat if c["order"] == "pos" else flat.transpose(1, 2).contiguous())
        return [y] + stored
    y = torch.zeros(sum(new) + c["pad"], H, hs, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        where = np.arange(_dropped(c, m, n), m)
        p, o = torch.from_numpy(table[b, where // page]).cuda(), torch.from_numpy(where % page).cuda()
        seen = torch.from_numpy(where).cuda()[None, :] <= torch.arange(m - n, m, device="cuda")[:, None]
        for j in range(kvH):
            if c["order"] == "head":
                k, v = i["kp"][p, j, o].double(), i["vp"][p, j, o].double()
            else:
                k, v = i["kp"][p, o, j].double(), i["vp"][p, o, j].double()
            kt = k.t().contiguous()
            for h in range(j * H // kvH, (j + 1) * H // kvH):
                e = (i["q"][at:at + n, h].double() @ kt) / hs ** 0.5
                e = torch.where(seen, e, torch.full_like(e, -math.inf))
                y[at:at + n, h] = torch.exp(e - torch.logsumexp(e, 1, keepdim=True)) @ v
        at += n
    return y


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------
def work(case):
    c = case
    ea, H, kvH, hs = (4 if c["act"] == "f32" else 2), c["H"], c["kvH"], c["hs"]
    if c["kind"] in ("norm", "norm_bwd"):
        n = c["B"] * c["T"] * (H + kvH) * hs
        if c["kind"] == "norm":
            return dict(bytes=float(ea * (2 * n + 2 * hs)), flops=7.0 * n)
        return dict(bytes=float(ea * (3 * n + 4 * hs)), flops=14.0 * n)
    new, lens = _sequences(c)
    ec, total = (4 if c["cache"] == "f32" else 2), sum(new)
    if c["kind"] == "append":
        return dict(bytes=float(total * hs * (ea * (2 * H + 2 * kvH) + ec * 2 * kvH)), flops=7.0 * total * (H + kvH) * hs)
    have = [m - _dropped(c, m, n) for n, m in zip(new, lens)]
    # token j of n sees all but the n - 1 - j positions behind it
    pairs = sum(n * m - n * (n - 1) // 2 for n, m in zip(new, have))
    return dict(bytes=float(2 * ea * total * H * hs + 2 * ec * kvH * hs * sum(have)), flops=4.0 * pairs * H * hs)
