"""Timing cases of what a server does around a paged cache: room for a step's tokens, attention behind a prefix that many sequences share, and
the draw of their next tokens.

A case is one pass through one operator:

  plan    a step's new tokens get pages: block table, free pages, starts, lengths, positions and slots (``CudaDnn.PagedPlan``)
  prefix  attention of the new tokens of every sequence over its pages, the prefix of a group of sequences read once for all of them
          (``AttnPagedPrefixForward``)
  sample  the next token of every sequence by temperature, top-k, top-p and min-p from given random numbers (``SampleForward``)

The plain forms are written with elementary torch operations: attention in 32 bits, weights of tokens and their sums in 64 (a draw lies next to a border of
a sum over the whole vocabulary), whole numbers as whole numbers.
"""
import ctypes
import math
import random  # noqa: F401  (draw takes a random.Random)

import numpy as np
import torch

own = False


def listed():
    return [
        # four conversations, one new token each: nothing but the call
        dict(name="plan_step_small", kind="plan", B=4, page=16, width=64, fill=0.5, step="decode", short=False),
        # a decoding step of a busy server: some sequences end, some begin behind a shared prompt
        dict(name="plan_step", kind="plan", B=512, page=16, width=512, fill=0.5, step="mixed", short=False),
        # prompts come in, more of them than there are pages: the last ones wait
        dict(name="plan_prompts", kind="plan", B=256, page=32, width=1024, fill=0.1, step="prompts", short=True),
        # a few short chats behind one short system prompt in 32 bits
        dict(name="prefix_f32_small", kind="prefix", act="f32", cache="f32", B=4, groups=1, new=1, shared=96, own=40, page=16, order="head", pad=0, H=6, kvH=6, hs=48),
        # a decoding step of 64 sequences behind one long document, four query heads to a key head
        dict(name="prefix_bf16_step", kind="prefix", act="bf16", cache="bf16", B=64, groups=1, new=1, shared=8192, own=512, page=16, order="head", pad=0, H=32, kvH=8,
             hs=128),
        # many users of three assistants, each assistant with its own prompt; heads of 64, none shared
        dict(name="prefix_bf16_many", kind="prefix", act="bf16", cache="bf16", B=192, groups=3, new=1, shared=2048, own=700, page=16, order="pos", pad=3, H=12, kvH=12,
             hs=64),
        # questions of some hundred tokens to one long document
        dict(name="prefix_bf16_chunk", kind="prefix", act="bf16", cache="bf16", B=16, groups=1, new=256, shared=16384, own=600, page=32, order="head", pad=0, H=32, kvH=8,
             hs=128),
        # a few tokens each in 32 bits over a 16-bit cache, two prompts
        dict(name="prefix_f32_mixed", kind="prefix", act="f32", cache="bf16", B=24, groups=2, new=5, shared=3000, own=300, page=24, order="pos", pad=7, H=12, kvH=4, hs=64),
        # one user's next token out of the vocabulary of the 110M configuration
        dict(name="sample_f32_one", kind="sample", act="f32", rows=1, vocab=32000, k=False, p=True, m=False),
        # a step of 64 users who all draw from the 50 likeliest tokens, a vocabulary that is no power of two
        dict(name="sample_f32_topk", kind="sample", act="f32", rows=64, vocab=50261, k=True, p=False, m=False),
        # a large step over a large vocabulary in 16 bits, every user with settings of their own
        dict(name="sample_bf16_mixed", kind="sample", act="bf16", rows=256, vocab=131072, k=True, p=True, m=True),
        # temperature alone: the whole vocabulary stays
        dict(name="sample_bf16_temp", kind="sample", act="bf16", rows=48, vocab=200003, k=False, p=False, m=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "prefix", "prefix", "sample", "sample"])
    if kind == "plan":
        width, page = _log(rng, 8, 1024), rng.choice([8, 16, 16, 24, 32, 64, 128])
        # slots are whole numbers below 2^24
        return dict(kind=kind, B=_log(rng, 1, min(1024, 262144 // width, 12_000_000 // (width * page))), page=page, width=width,
                    fill=rng.choice([0.1, 0.3, 0.5, 0.8]), step=rng.choice(["decode", "mixed", "prompts"]), short=rng.random() < 0.3)
    if kind == "sample":
        vocab = _log(rng, 500, 262144)
        return dict(kind=kind, act=rng.choice(["f32", "bf16"]), rows=_log(rng, 1, max(1, min(512, 16_000_000 // vocab))), vocab=vocab, k=rng.random() < 0.5,
                    p=rng.random() < 0.6, m=rng.random() < 0.3)
    hs = rng.choice([32, 48, 64, 64, 96, 128, 128])
    kvH = rng.randint(1, 12)
    H = kvH * rng.choice([1, 1, 2, 4, 7, 8])
    if H > 40:
        H = kvH
    act, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "bf16")])
    shared = _log(rng, 64, 16384)
    new = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 2, 256)])
    rest = _log(rng, new, max(new, 1024))
    # no more products, and of them in 32 bits a fifth, than the largest listed case has
    most = 1.05e12 * (0.2 if act == "f32" else 1.0) / (4.0 * H * hs * new * (shared + rest))
    B = _log(rng, 2, max(2, min(256, int(most), 4096 // new)))
    return dict(kind=kind, act=act, cache=cache, B=B, groups=rng.randint(1, min(4, B)), new=new, shared=shared, own=rest, page=rng.choice([8, 16, 16, 24, 32, 64, 128]),
                order=rng.choice(["head", "pos"]), pad=rng.choice([0, 0, rng.randint(1, 40)]), H=H, kvH=kvH, hs=hs)


# ---- what the sizes of a case say ----------------------------------------------------------------------------------------
def _part(b):
    return (0.37 + 0.6180339887 * b) % 1.0


def _prefixes(c):
    """First sequences of the groups (and the end of the last), shared positions of each: the first has c["shared"], the others less."""
    firsts = [g * c["B"] // c["groups"] for g in range(c["groups"])] + [c["B"]]
    return firsts, [max(1, c["shared"] - g * c["shared"] // 5) for g in range(c["groups"])]


def _sequences(c):
    """New tokens and positions (the new ones among them) of every sequence, the group that each is in."""
    firsts, shared = _prefixes(c)
    new, lens, group = [], [], []
    for g in range(c["groups"]):
        for b in range(firsts[g], firsts[g + 1]):
            n = max(1, int(c["new"] * (0.3 + 0.7 * _part(b + 1))))
            new.append(n)
            lens.append(shared[g] + max(n, int(c["own"] * (0.1 + 0.9 * _part(b)))))
            group.append(g)
    return new, lens, group


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _strides(c):
    """Elements from page to page, head to head, position to position."""
    whole = c["kvH"] * c["page"] * c["hs"]
    return (whole, c["page"] * c["hs"], c["hs"]) if c["order"] == "head" else (whole, c["hs"], c["kvH"] * c["hs"])


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def _plan_inputs(c, seed):
    """A server's state before a step: sequences of all lengths, in pages that earlier requests left in any order."""
    r = np.random.default_rng(seed)
    B, W, page = c["B"], c["width"], c["page"]
    lens = np.maximum(1, (W * page * c["fill"] * r.random(B) * 1.2).astype(np.int64).clip(0, W * page - page))
    new, source, shared = np.ones(B, np.int64), np.full(B, -1, np.int64), np.zeros(B, np.int64)
    if c["step"] != "decode":
        kind = r.random(B)
        # places without a sequence, of which some begin, most of them behind the prompt of the first one; sequences that end; some that rest
        idle = (kind < (0.15 if c["step"] == "mixed" else 0.7)) & (np.arange(B) > 0)
        lens[idle], new[idle] = 0, 0
        begin = idle & (r.random(B) < 0.7)
        most = min(2048, max(1, W * page // 4))
        new[begin] = 1 + (most * r.random(int(begin.sum())) ** 2).astype(np.int64)
        behind = begin & (r.random(B) < 0.6)
        source[behind], shared[behind] = 0, int(lens[0]) // page // 2 * page
        ends = ~idle & (kind > 0.94) & (np.arange(B) > 0)
        new[ends] = -1
        new[~idle & ~ends & (r.random(B) < 0.05)] = 0
    held = -(-lens // page)
    need = np.where(new > 0, -(-(lens + np.maximum(new, 0)) // page) - held, 0).sum()
    spare = int(need * 0.6) if c["short"] else int(need) + 8 + B
    # a cache that could hold every table, and a step's budget of rows
    pages, tokens = B * W, B if c["step"] == "decode" else min(65536, B * max(1, W * page // 8))
    spare = min(spare, pages - int(held.sum()))
    order = r.permutation(pages)
    table = np.full((B, W), -1.0, np.float32)
    mask = np.arange(W)[None, :] < held[:, None]
    table[mask] = order[:int(held.sum())]
    free = np.full(pages + 1, -1.0, np.float32)
    free[0] = spare
    free[1:1 + spare] = order[int(held.sum()):int(held.sum()) + spare]
    f = {"new": new, "lens": lens, "from": source, "shared": shared}
    return {**{n: torch.from_numpy(v.astype(np.float32)).cuda() for n, v in f.items()}, "table": torch.from_numpy(table).cuda(), "free": torch.from_numpy(free).cuda()}, pages, tokens


def _sample_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rows, vocab = c["rows"], c["vocab"]

    def uniform(n=rows):
        return torch.rand(n, generator=g, device="cuda")

    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
    # a model's next token: a handful of candidates above the rest
    best = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    x.scatter_add_(1, best, 3 + 7 * torch.rand(rows, 24, generator=g, device="cuda"))
    i = {"x": x.to(_type(c["act"])), "u": uniform()}
    mixed = c["k"] and c["p"] and c["m"]
    # a server's mixture: one user in eight wants the likeliest token
    i["temperature"] = torch.where(uniform() < (0.125 if mixed else 0.0), torch.zeros(rows, device="cuda"), 0.4 + 0.9 * uniform())
    if c["k"]:
        i["k"] = torch.where(uniform() < 0.5, torch.floor(1 + 2000 * uniform() ** 2), torch.zeros(rows, device="cuda")) if mixed else torch.full((rows,), 50.0, device="cuda")
    if c["p"]:
        i["p"] = torch.where(uniform() < 0.3, torch.ones(rows, device="cuda"), 0.5 + 0.49 * uniform()) if mixed else torch.full((rows,), 0.9, device="cuda")
    if c["m"]:
        i["m"] = torch.where(uniform() < 0.5, torch.zeros(rows, device="cuda"), 0.01 + 0.2 * uniform())
    return i


def _prefix_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    new, lens, group = _sequences(c)
    firsts, shared = _prefixes(c)
    page, kvH, hs = c["page"], c["kvH"], c["hs"]
    width = max(-(-n // page) for n in lens) + 1
    # whole pages of the prefix are one copy for the group; what is left of it is each sequence's own
    common = [s // page for s in shared]
    count = [-(-n // page) - common[j] for n, j in zip(lens, group)]
    need = sum(common) + sum(count)
    pages = need + 3
    order = torch.randperm(pages, generator=g, device="cuda")[:need].cpu().numpy()
    table, at, prefix = np.full((c["B"], width), -1.0, np.float32), 0, []
    for n in common:
        prefix.append(order[at:at + n])
        at += n
    for b, (n, j) in enumerate(zip(count, group)):
        table[b, :common[j]] = prefix[j]
        table[b, common[j]:common[j] + n] = order[at:at + n]
        at += n
    i = {"table": torch.from_numpy(table).cuda()}
    for name, v in (("starts", np.concatenate([[0], np.cumsum(new)])), ("lens", lens), ("groups", firsts), ("shared", shared)):
        i[name] = torch.tensor(np.asarray(v), dtype=torch.float32, device="cuda")
    shape = (pages, kvH, page, hs) if c["order"] == "head" else (pages, page, kvH, hs)
    i["kp"], i["vp"] = normal(*shape, dtype=_type(c["cache"])), normal(*shape, dtype=_type(c["cache"]))
    # the part of a prefix behind its whole pages is the same in every sequence of the group
    for j in range(c["groups"]):
        rest = shared[j] - common[j] * page
        if rest:
            mine = torch.from_numpy(table[firsts[j]:firsts[j + 1], common[j]].astype(np.int64)).cuda()
            for t in ("kp", "vp"):
                if c["order"] == "head":
                    i[t][mine, :, :rest] = i[t][mine[0], :, :rest].clone()
                else:
                    i[t][mine, :rest] = i[t][mine[0], :rest].clone()
    i["q"] = normal(sum(new) + c["pad"], c["H"], hs, dtype=_type(c["act"]))
    return i


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
        self.cuda, self.memory = cuda, []

    def __del__(self):
        try:
            for h in self.memory:
                self.cuda.FreeMemory(h)
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
    c = dict(case)
    s = dict(case=c)
    # outputs that a program keeps room for
    if c["kind"] == "plan":
        i, s["pages"], s["tokens"] = _plan_inputs(c, seed)
        out = {"lens_out": i["lens"].shape, "table_out": i["table"].shape, "free_out": i["free"].shape, "shared_out": i["shared"].shape, "starts": (c["B"] + 1,),
               "positions": (s["tokens"],), "slots": (s["tokens"],), "last": (c["B"],)}
    elif c["kind"] == "sample":
        i, out = _sample_inputs(c, seed), {"ids": (c["rows"],), "logs": (c["rows"],)}
    else:
        i = _prefix_inputs(c, seed)
        s["pages"], s["width"], s["tokens"], out = i["kp"].shape[0], i["table"].shape[1], i["q"].shape[0], {"y": i["q"].shape}
    kinds = {n: _type(c["act"]) if n == "y" else torch.float32 for n in out}
    if not own:
        return {**s, **i, **{n: torch.zeros(tuple(shape), dtype=kinds[n], device="cuda") for n, shape in out.items()}}
    s.update(cuda=_cuda(), h={}, v={})
    s["owner"] = _Handles(s["cuda"])
    for name, t in i.items():
        s["h"][name], s["v"][name] = _empty(s["owner"], tuple(t.shape), t.dtype)
        s["v"][name].copy_(t)
    for name, shape in out.items():
        s["h"][name], s["v"][name] = _empty(s["owner"], tuple(shape), kinds[name])
        s["v"][name].zero_()
    torch.cuda.synchronize()
    return s


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


PLAN = ("lens_out", "table_out", "free_out", "shared_out", "starts", "positions", "slots", "last")


# ---- the framework's calls ---------------------------------------------------------------------------------------------------
def _own_plan(s):
    c, h = s["case"], s["h"]
    s["cuda"].PagedPlan(c["B"], s["tokens"], s["pages"], c["page"], c["width"], h["new"], h["lens"], h["table"], h["free"], h["lens_out"], h["table_out"], h["free_out"],
                        h["starts"], h["positions"], h["slots"], h["last"], h["from"], h["shared"], h["shared_out"])
    return [s["v"][n] for n in PLAN]


def _own_prefix(s):
    c, h = s["case"], s["h"]
    s["cuda"].AttnPagedPrefixForward(c["B"], s["tokens"], c["H"], c["kvH"], c["hs"], s["pages"], c["page"], s["width"], h["q"], h["kp"], h["vp"], h["table"], h["starts"],
                                     h["lens"], h["y"], *_strides(c), c["groups"], h["groups"], h["shared"])
    return s["v"]["y"]


def _own_sample(s):
    c, h = s["case"], s["h"]
    s["cuda"].SampleForward(c["rows"], c["vocab"], h["x"], h["u"], h["ids"], h["temperature"], h.get("k", 0), h.get("p", 0), h.get("m", 0), hLogProb=h["logs"])
    return [s["v"]["ids"], s["v"]["logs"]]


# ---- plain forms ----------------------------------------------------------------------------------------------------------------
def _plain_plan(s):
    c, pages, tokens = s["case"], s["pages"], s["tokens"]
    B, W, page = c["B"], c["width"], c["page"]
    new, lens, source, shared, table = (s[n].long() for n in ("new", "lens", "from", "shared", "table"))
    entry = torch.arange(W, device="cuda")[None, :]
    # pages of the sequences that end, behind those that are free (what does not go there: to a place behind the list)
    ends = new < 0
    back = ends[:, None] & (entry >= (shared // page)[:, None]) & (entry < (-(-lens // page))[:, None]) & (table >= 0) & (table < pages)
    place = torch.cumsum(back.reshape(-1), 0).reshape(B, W)
    count = s["free"][0].long()
    free = torch.cat([s["free"][1:].long(), torch.zeros(1, dtype=torch.long, device="cuda")])
    free.scatter_(0, torch.where(back, count + place - 1, torch.full_like(place, pages)).reshape(-1), table.reshape(-1))
    count = count + place[-1, -1]
    # sequences that begin behind the whole pages of another one
    lender = source.clamp(0, B - 1)
    begins = (lens == 0) & (new > 0) & (source >= 0) & (source < B) & (source != torch.arange(B, device="cuda")) & ~ends[lender]
    take = torch.where(begins, torch.minimum(shared // page, lens[lender] // page), torch.zeros_like(lens))
    before = lens + take * page
    able = (new > 0) & (before + new <= W * page)
    grow = torch.where(able, new, torch.zeros_like(new))
    first = -(-before // page)
    need = torch.where(able, -(-(before + grow) // page) - first, torch.zeros_like(grow))
    sums = torch.cumsum(need, 0)
    granted = able & (sums <= count) & (torch.cumsum(grow, 0) <= tokens)
    grow = torch.where(granted, grow, torch.zeros_like(grow))
    after = torch.where(ends, torch.zeros_like(lens), torch.where(granted, before + grow, lens))
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), torch.cumsum(grow, 0)])
    mine = granted[:, None] & (entry >= first[:, None]) & (entry < (first + need)[:, None])
    at = (count - 1 - ((sums - need)[:, None] + entry - first[:, None])).clamp(0, pages - 1)
    result = torch.where(mine, free[at], table)
    result = torch.where((granted & begins)[:, None] & (entry < take[:, None]), table[lender], result)
    result = torch.where(ends[:, None], torch.full_like(result, -1), result)
    left = count - torch.where(granted, need, torch.zeros_like(need)).sum()
    i = torch.arange(pages, device="cuda")
    s["free_out"][1:] = torch.where(i < left, free[:pages].float(), s["free_out"][1:])
    s["free_out"][0] = left.float()
    i = torch.arange(tokens, device="cuda")
    b = (torch.searchsorted(starts, i, right=True) - 1).clamp(0, B - 1)
    live = i < starts[-1]
    position = torch.where(live, after[b] - grow[b] + i - starts[b], torch.zeros_like(i))
    where = result[b, position // page]
    slot = torch.where((where >= 0) & (where < pages), where * page + position % page, torch.full_like(where, -1))
    s["positions"].copy_(torch.where(live, position.float(), s["positions"]))
    s["slots"].copy_(torch.where(live, slot.float(), s["slots"]))
    s["last"].copy_(torch.where(grow > 0, starts[1:] - 1, torch.full_like(grow, -1)))
    s["shared_out"].copy_(torch.where(ends, torch.zeros_like(shared), torch.where(granted & (lens == 0), take * page, shared)))
    s["starts"].copy_(starts)
    s["lens_out"].copy_(after)
    s["table_out"].copy_(result)
    return [s[n] for n in PLAN]


def _by_head(c, pages):
    """A view (pages, heads, positions, values) of the cache."""
    return pages if c["order"] == "head" else pages.permute(0, 2, 1, 3)


def _plain_prefix(s):
    c = s["case"]
    H, kvH, hs, page = c["H"], c["kvH"], c["hs"], c["page"]
    G, scale = H // kvH, 1.0 / math.sqrt(hs)
    kp, vp = _by_head(c, s["kp"]), _by_head(c, s["vp"])
    new, lens, _ = _sequences(c)
    firsts, shared = _prefixes(c)
    for g in range(c["groups"]):
        b0, b1 = firsts[g], firsts[g + 1]
        n, N, common = b1 - b0, max(new[b0:b1]), shared[g] // page
        # rows (n, N) of the group's tokens, short chunks filled up with their last token
        count, length = s["starts"][b0 + 1:b1 + 1] - s["starts"][b0:b1], s["lens"][b0:b1]
        j = torch.minimum(torch.arange(N, device="cuda")[None, :], count[:, None] - 1)
        row = (s["starts"][b0:b1, None] + j).long()
        q = s["q"][row].float().reshape(n, N, kvH, G, hs).permute(2, 0, 1, 3, 4) * scale          # (kvH, n, N, G, hs)
        # the prefix: one product for all rows of the group
        table = s["table"][b0:b1].long()
        scores = []
        if common:
            k = kp[table[0, :common]].permute(1, 3, 0, 2).reshape(kvH, hs, common * page).float()
            scores.append(torch.matmul(q.reshape(kvH, n * N * G, hs), k).reshape(kvH, n, N * G, common * page).transpose(0, 1))
        # what is behind it: a batch of all sequences, positions filled up to the longest
        width = -(-max(lens[b0:b1]) // page)
        own_pages = table[:, common:width].clamp(min=0)
        k = kp[own_pages].permute(0, 2, 4, 1, 3).reshape(n * kvH, hs, -1).float()
        e = torch.matmul(q.permute(1, 0, 2, 3, 4).reshape(n * kvH, N * G, hs), k.contiguous()).reshape(n, kvH, N, G, -1)
        t = common * page + torch.arange(e.shape[-1], device="cuda")
        seen = t[None, None, :] <= ((length - count)[:, None] + j)[:, :, None]
        scores.append(e.masked_fill(~seen[:, None, :, None, :], float("-inf")).reshape(n, kvH, N * G, -1))
        top = torch.stack([e.amax(-1, keepdim=True) for e in scores]).amax(0)
        w = [torch.exp(e - top) for e in scores]
        total = sum(e.sum(-1, keepdim=True) for e in w)
        v = vp[own_pages].permute(0, 2, 1, 3, 4).reshape(n * kvH, -1, hs).float()
        o = torch.matmul(w[-1].reshape(n * kvH, N * G, -1), v.contiguous()).reshape(n, kvH, N * G, hs)
        if common:
            v = vp[table[0, :common]].permute(1, 0, 2, 3).reshape(kvH, common * page, hs).float()
            o = o + torch.matmul(w[0].transpose(0, 1).reshape(kvH, n * N * G, -1), v).reshape(kvH, n, N * G, hs).transpose(0, 1)
        o = (o / total).reshape(n, kvH, N, G, hs).permute(0, 2, 1, 3, 4).reshape(n, N, H, hs)
        s["y"][row.reshape(-1)] = o.reshape(n * N, H, hs).to(s["y"].dtype)
    return s["y"]


def _plain_sample(s):
    x = s["x"].double()
    rows, vocab = x.shape
    greedy = s["temperature"] <= 0
    heat = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    ordered, index = torch.sort(x, dim=1, descending=True, stable=True)       # equal ones: the lowest index first
    w = torch.exp((ordered - ordered[:, :1]) / heat)
    rank = torch.arange(vocab, device="cuda")[None, :]
    keep = torch.ones_like(w, dtype=torch.bool)
    if "k" in s:
        k = s["k"].long()[:, None]
        keep = (rank < k) | (k <= 0)
    if "p" in s:
        sums = torch.cumsum(torch.where(keep, w, torch.zeros_like(w)), 1)
        p = s["p"].double()[:, None]
        before = torch.cat([torch.zeros(rows, 1, dtype=torch.float64, device="cuda"), sums[:, :-1]], 1)
        keep = keep & ((before < p * sums[:, -1:]) | (p >= 1) | (rank == 0))
    if "m" in s:
        keep = keep & ((w >= s["m"].double()[:, None]) | (rank == 0))
    weight = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, torch.zeros_like(w)))
    sums = torch.cumsum(weight, 1)
    drawn = (sums <= s["u"].double()[:, None] * sums[:, -1:]).sum(1)
    drawn = torch.where(greedy, index[:, 0], drawn)
    s["ids"].copy_(drawn)
    logs = torch.log(weight.gather(1, drawn[:, None]) / sums[:, -1:])[:, 0]
    s["logs"].copy_(torch.where(greedy, torch.zeros_like(logs), logs))
    return [s["ids"], s["logs"]]


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------
def _exact_plan(c, i, pages, tokens):
    """Sequence after sequence."""
    page, W = c["page"], c["width"]
    new, lens, source, shared = (i[n].cpu().numpy().astype(int).tolist() for n in ("new", "lens", "from", "shared"))
    old, free = i["table"].cpu().numpy().astype(int), i["free"].cpu().numpy().astype(int)
    stack, table, after, borrowed = free[1:1 + free[0]].tolist(), old.copy(), list(lens), list(shared)
    for b, n in enumerate(new):
        if n < 0:
            stack += [p for p in old[b, shared[b] // page:-(-lens[b] // page)].tolist() if 0 <= p < pages]
            table[b], after[b], borrowed[b] = -1, 0, 0
    starts, positions, slots, last = [0], [], [], []
    wait, asked = False, 0
    for b, n in enumerate(new):
        begin = lens[b]
        lender = source[b] if lens[b] == 0 and n > 0 and 0 <= source[b] < len(new) and source[b] != b and new[source[b]] >= 0 else -1
        if lender >= 0:
            begin = min(shared[b] // page, lens[lender] // page) * page
        if n > 0 and begin + n <= W * page:
            first, end = -(-begin // page), -(-(begin + n) // page)
            asked += n
            wait = wait or end - first > len(stack) or asked > tokens
            if not wait:
                if lender >= 0:
                    table[b, :first] = old[lender, :first]
                for e in range(first, end):
                    table[b, e] = stack.pop()
                if lens[b] == 0:
                    borrowed[b] = begin if lender >= 0 else 0
                after[b] = begin + n
                places = np.arange(begin, begin + n)
                positions.append(places)
                slots.append(np.where(table[b, places // page] >= 0, table[b, places // page] * page + places % page, -1))
        starts.append(starts[-1] + (after[b] - begin if after[b] > lens[b] else 0))
        last.append(starts[-1] - 1 if starts[-1] > starts[-2] else -1)
    full = np.zeros(pages + 1)
    full[0], full[1:1 + len(stack)] = len(stack), stack
    rows = [np.zeros(tokens) for _ in range(2)]
    for r, parts in zip(rows, (positions, slots)):
        if parts:
            r[:starts[-1]] = np.concatenate(parts)
    return [np.asarray(v, np.float64) for v in (after, table, full, borrowed, starts, *rows, last)]


def _exact_sample(c, i):
    ids, logs = [], []
    given = {n: v.cpu().double().numpy() for n, v in i.items() if n != "x"}
    for r in range(c["rows"]):
        x = i["x"][r].cpu().double().numpy()
        heat, u = given["temperature"][r], given["u"][r]
        if heat <= 0:
            ids.append(int(np.argmax(x)))
            logs.append(0.0)
            continue
        order = np.argsort(-x, kind="stable")
        if c["k"] and given["k"][r] > 0:
            order = order[:int(given["k"][r])]
        w = np.exp(x[order] / heat - x[order[0]] / heat)
        if c["p"] and given["p"][r] < 1:
            order = order[:1 + int(np.searchsorted(np.cumsum(w), given["p"][r] * w.sum(), side="left"))]
        if c["m"]:
            order = order[np.exp((x[order] - x[order[0]]) / heat) >= given["m"][r]]
        order = np.sort(order)
        w = np.exp((x[order] - x[order].max()) / heat)
        total = np.cumsum(w)
        at = int(np.searchsorted(total, u * total[-1], side="right"))
        ids.append(int(order[at]))
        logs.append(math.log(w[at]) - math.log(math.fsum(w)))
    return [np.asarray(ids, np.float64), np.asarray(logs)]


def exact(case, seed):
    c = dict(case)
    if c["kind"] == "plan":
        return _exact_plan(c, *_plan_inputs(c, seed))
    if c["kind"] == "sample":
        return _exact_sample(c, _sample_inputs(c, seed))
    i = _prefix_inputs(c, seed)
    new, lens, _ = _sequences(c)
    H, kvH, hs, page = c["H"], c["kvH"], c["hs"], c["page"]
    table = i["table"].cpu().numpy().astype(np.int64)
    y = torch.zeros(i["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    # every sequence over all of its own pages: who shares what does not show in the result
    for b, (n, m) in enumerate(zip(new, lens)):
        where = np.arange(m)
        p, o = torch.from_numpy(table[b, where // page]).cuda(), torch.from_numpy(where % page).cuda()
        seen = torch.from_numpy(where).cuda()[None, :] <= torch.arange(m - n, m, device="cuda")[:, None]
        for j in range(kvH):
            k, v = ((t[p, j, o] if c["order"] == "head" else t[p, o, j]).double() for t in (i["kp"], i["vp"]))
            q = i["q"][at:at + n, j * H // kvH:(j + 1) * H // kvH].double()
            e = (q.reshape(-1, hs) @ k.t().contiguous()).reshape(n, -1, m) / hs ** 0.5
            e = torch.where(seen[:, None, :], e, torch.full_like(e, -math.inf))
            a = torch.exp(e - torch.logsumexp(e, 2, keepdim=True))
            y[at:at + n, j * H // kvH:(j + 1) * H // kvH] = (a.reshape(-1, m) @ v).reshape(n, -1, hs)
        at += n
    return y


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "plan":
        # the block table and the list of free pages, about half of it in use, read and written once
        return dict(bytes=12.0 * c["B"] * c["width"] + 40.0 * c["B"], flops=10.0 * c["B"])
    if c["kind"] == "sample":
        n = float(c["rows"] * c["vocab"])
        return dict(bytes=n * (4 if c["act"] == "f32" else 2) + 28.0 * c["rows"], flops=10.0 * n)
    new, lens, group = _sequences(c)
    ea, ec, H, kvH, hs = (4 if c["act"] == "f32" else 2), (4 if c["cache"] == "f32" else 2), c["H"], c["kvH"], c["hs"]
    _, shared = _prefixes(c)
    whole = [n // c["page"] * c["page"] for n in shared]
    positions = sum(whole) + sum(m - whole[g] for m, g in zip(lens, group))
    pairs = sum(n * m - n * (n - 1) // 2 for n, m in zip(new, lens))
    return dict(bytes=float(2 * ea * sum(new) * H * hs + 2 * ec * kvH * hs * positions), flops=4.0 * pairs * H * hs)
