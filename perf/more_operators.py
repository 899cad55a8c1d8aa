"""The 4-bit cache and the operators beside it: what they compute, on which sizes, and what each has to move.

Three operators of a decoder layer that keeps its keys and values in 4 bits:

  turn       RMS norm of each query and key head, and rotary positions, whose pairs may belong to several axes (time,
             height, width), in one pass.
  append     the same on the way into the pages of a cache that holds a head's vector as 4-bit codes and four scales,
             one for each quarter of the head; values beside it.
  attention  attention of one or more new tokens of each sequence over these pages.

Element e of a head of D elements belongs to quarter c = e // (D / 4), at place r = e % (D / 4) in it.  A vector's code
for it, an unsigned number n, is bits 4 c .. 4 c + 3 of the vector's 16-bit word r (low byte first), and stands for
(n - 8) * scale[c].  scale[c] is max|x| / 7.5 of the quarter, rounded to bf16 and at least 2^-126; n - 8 is x / scale[c],
rounded to the nearest whole number (ties to even) and limited to -8 .. 7.

``run`` computes them in plain torch operations, or, with ``own`` set, through the public functions of siliconfer_b200.
``exact`` gives the same outputs from the definitions in 64 bits.  Codes have to be equal, so they are returned as they
lie, two to a byte; that is why keys are normed and turned in 64 bits on their way to them.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
ROPE_BASE = 10000.0


# ---------------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # One token of a 14-head decoder with normed heads: launch latency.
        dict(name="turn_1x14h", op="turn", T=1, H=14, Hkv=2, D=64, rot=64, axes=1, interleaved=False, norm=True, x="bf16"),
        # A prompt of 4096 text and image tokens: 64 query and 8 kv heads, positions in time, height and width.
        dict(name="turn_4096x64h", op="turn", T=4096, H=64, Hkv=8, D=128, rot=128, axes=3, interleaved=False, norm=True,
             x="bf16"),
        # The patches of an image in its encoder: 16 heads of 80, height and width, neighbouring pairs, no norm.
        dict(name="turn_1369x16h_d80", op="turn", T=1369, H=16, Hkv=16, D=80, rot=80, axes=2, interleaved=True, norm=False,
             x="f16"),
        # A decode step of 8 sequences with 32 heads: one token each.
        dict(name="append4_8x1_32h", op="append", B=8, n=1, S=1500, H=32, Hkv=32, D=128, page=64, rot=128, axes=1,
             interleaved=False, norm=False, x="bf16", ragged=True),
        # A prompt chunk of 4096 tokens in 4 sequences with normed heads, 64 query and 8 kv heads, three axes.
        dict(name="append4_4x1024_64h", op="append", B=4, n=1024, S=2000, H=64, Hkv=8, D=128, page=64, rot=128, axes=3,
             interleaved=False, norm=True, x="bf16", ragged=False),
        # Prompts of up to 333 tokens beside decoding sequences, half of each head turned, 32-bit activations.
        dict(name="append4_9x333_20h", op="append", B=9, n=333, S=900, H=20, Hkv=20, D=96, page=16, rot=48, axes=1,
             interleaved=True, norm=True, x="f32", ragged=True),
        # One short conversation of the 14-head decoder: launch latency.
        dict(name="attention4_1x1000_14h", op="attention", B=1, n=1, S=1000, H=14, Hkv=2, D=64, page=16, window=0,
             x="bf16", ragged=False, lse=False),
        # A decode step of 16 sequences of 8192 tokens, 64 query and 8 kv heads: the cache read.
        dict(name="attention4_16x8192_64h", op="attention", B=16, n=1, S=8192, H=64, Hkv=8, D=128, page=64, window=0,
             x="bf16", ragged=False, lse=False),
        # One sequence of 131072 tokens: the work has to be split over the keys.
        dict(name="attention4_1x131072_32h", op="attention", B=1, n=1, S=131072, H=32, Hkv=8, D=128, page=64, window=0,
             x="bf16", ragged=False, lse=True),
        # A served batch of 64 sequences of 0 to 4096 tokens with 32 heads of their own, 16-bit floating point.
        dict(name="attention4_64x4096_32h", op="attention", B=64, n=1, S=4096, H=32, Hkv=32, D=128, page=32, window=0,
             x="f16", ragged=True, lse=False),
        # Guesses of up to 5 tokens checked at once, a window of 1000 keys, 32-bit queries, heads of 256.
        dict(name="attention4_13x5_8h_f32", op="attention", B=13, n=5, S=2500, H=8, Hkv=1, D=256, page=128, window=1000,
             x="f32", ragged=True, lse=True),
        # Prompt chunks of up to 256 tokens beside decoding sequences, 64 query and 8 kv heads.
        dict(name="attention4_8x256_64h", op="attention", B=8, n=256, S=4000, H=64, Hkv=8, D=128, page=64, window=0,
             x="bf16", ragged=True, lse=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["turn", "append", "attention"])
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    H, Hkv = rng.choice([(14, 2), (32, 32), (64, 8), (8, 1), (20, 20)])
    if op == "turn":
        D = rng.choice([64, 72, 80, 96, 128, 128, 256])
        T = _log(rng, 1, min(4096, 4096 * 72 * 128 // ((H + Hkv) * D)))
        return dict(op=op, T=T, H=H, Hkv=Hkv, D=D, rot=rng.choice([D, D, D // 2]), axes=rng.choice([1, 2, 3, 4]),
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.7, x=x)
    D = rng.choice([64, 128, 128, 256] + ([96] if H != 32 else []))
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        B = _log(rng, 1, 64)
        n = _log(rng, 1, min(1024, 16384 * 128 // (B * H * D)) or 1)
        return dict(op=op, B=B, n=n, S=n + _log(rng, 1, 2000), H=H, Hkv=Hkv, D=D, page=page, rot=rng.choice([D, D, D // 2]),
                    axes=rng.choice([1, 1, 3]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.5, x=x,
                    ragged=rng.random() < 0.5)
    B = _log(rng, 1, 64)
    S = _log(rng, 16, min(131072, 100_000_000 // (B * Hkv * D)))
    n = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, min(256, S, 16_000_000 // (B * H * S))))
    return dict(op=op, B=B, n=n, S=max(S, n), H=H, Hkv=Hkv, D=D, page=page, window=rng.choice([0, 0, _log(rng, 8, 4096)]),
                x=x, ragged=rng.random() < 0.5, lse=rng.random() < 0.5)


def _counts(case):
    """(tokens after the call, new tokens) of each sequence, from the case alone.  Ragged batches hold an empty
    sequence (a batch slot in waiting) and, where several new tokens are allowed, single-token ones beside long ones."""
    B, S, n = case["B"], case["S"], case["n"]
    if not case["ragged"]:
        return [S] * B, [n] * B
    rng = random.Random(B * 7919 + S * 31 + n)
    news = [n if n == 1 or b == 0 else rng.choice([1, rng.randint(1, n), n]) for b in range(B)]
    lens = [S if b == 0 else rng.randint(c, S) for b, c in enumerate(news)]
    if B > 2:
        news[B // 2], lens[B // 2] = 0, 0
    return lens, news


# ---------------------------------------------------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    H, Hkv, D, e = case["H"], case["Hkv"], case["D"], SIZE[case["x"]]
    if case["op"] == "attention":
        lens, news = _counts(case)
        T, w = sum(news), case["window"]
        keys = sum(min(l, w + c - 1) if w else l for l, c in zip(lens, news) if c)
        pairs = sum(min(p + 1, w) if w else p + 1 for l, c in zip(lens, news) for p in range(l - c, l))
        return {"bytes": keys * Hkv * (D + 16) + 2 * T * H * D * e + (4 * T * H if case["lse"] else 0),
                "flops": 4 * pairs * H * D}
    T = case["T"] if case["op"] == "turn" else sum(_counts(case)[1])
    angles = T * (case["rot"] * 4 + 4 * case["axes"]) + 2 * D * e
    each = 6 + (4 if case["norm"] else 0)
    if case["op"] == "turn":
        return {"bytes": 2 * T * (H + Hkv) * D * e + angles, "flops": T * (H + Hkv) * D * each}
    return {"bytes": T * D * e * (2 * H + 2 * Hkv) + T * Hkv * (D + 16) + angles,
            "flops": T * D * ((H + Hkv) * each + 8 * Hkv)}


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.g = torch.Generator(device=self.dev).manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device=self.dev)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=self.dev)

    def integers(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device=self.dev)


def _angles(case, r, most):
    """A table of cosines and sines for positions below `most`, and the axis of each pair: the axes take turns until
    their pairs are used up, the first one has what is left over."""
    half, A = case["rot"] // 2, case["axes"]
    freq = ROPE_BASE ** (-torch.arange(half, device=r.dev, dtype=torch.float64) / half)
    angle = torch.arange(most, device=r.dev, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float(), [half - half // A * (A - 1)] + [half // A] * (A - 1)


def _axis_of_pairs(sections, interleaved):
    """What the sections say: pair j's axis, in runs, or the axes in turn."""
    if not interleaved:
        return [a for a, s in enumerate(sections) for _ in range(s)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def _heads(case, r, T):
    """What a fused projection gives: queries, keys and values side by side in each token's row; the norms' weights."""
    H, Hkv, D, dt = case["H"], case["Hkv"], case["D"], TYPES[case["x"]]
    # keys have a few channels that are far larger than the others
    size = torch.ones(H + 2 * Hkv, D, device=r.dev)
    size[H:H + Hkv] = torch.where(r.uniform(Hkv, D) < 0.05, 8.0, 1.0)
    qkv = (r.normal(T, H + 2 * Hkv, D) * size).to(dt)
    weight = lambda: (1 + 0.1 * r.normal(D)).to(dt) if case["norm"] else None
    return {"q": qkv[:, :H], "kn": qkv[:, H:H + Hkv], "vn": qkv[:, H + Hkv:], "wq": weight(), "wk": weight(),
            "eps": EPS if case["norm"] else None}


def _prepare_turn(case, r):
    T, A = case["T"], case["axes"]
    s = _heads(case, r, T)
    s["positions"] = r.integers(0, 4096, T, A).int()
    s["table"], sections = _angles(case, r, 4096)
    pairs = _axis_of_pairs(sections, True)
    s["axes"] = torch.tensor(pairs, dtype=torch.uint8, device=r.dev) if A > 1 else None
    if A == 1:
        s["positions"] = s["positions"][:, 0].contiguous()
    return s


def _prepare_cache(case, r):
    """Pages in random order, with the codes and scales that normal vectors of some spread have."""
    B, S, Hkv, D, page = case["B"], case["S"], case["Hkv"], case["D"], case["page"]
    per = -(-S // page)
    P = B * per + 3
    table = torch.randperm(P, generator=r.g, device=r.dev)[: B * per].view(B, per).to(torch.int32)
    lens, news = _counts(case)
    starts = torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32, device=r.dev)
    caches = []
    for _ in range(2):
        codes = torch.empty(P, Hkv, page, D // 2, dtype=torch.uint8, device=r.dev)
        for p in range(0, P, 64):
            part = codes[p:p + 64]
            n = (2.8 * r.normal(2, *part.shape) + 8).round_().clamp_(0, 15).to(torch.uint8)
            part.copy_(n[0] | n[1] << 4)
        caches += [codes, (0.3 * torch.exp2(r.uniform(P, Hkv, page, 4) * 2 - 1)).bfloat16()]
    return {"k": caches[0], "ks": caches[1], "v": caches[2], "vs": caches[3], "pages": table,
            "lens": torch.tensor(lens, dtype=torch.int32, device=r.dev), "starts": starts if case["ragged"] else None,
            "most": max(news), "T": sum(news)}


def _prepare_append(case, r):
    s = _prepare_cache(case, r)
    s.update(_heads(case, r, s["T"]))
    s["table"], sections = _angles(case, r, max(case["S"], 2048))
    s["axes"] = s["positions"] = None
    if case["axes"] > 1:
        s["axes"] = torch.tensor(_axis_of_pairs(sections, True), dtype=torch.uint8, device=r.dev)
        s["positions"] = r.integers(0, 2048, s["T"], case["axes"])
    return s


def _prepare_attention(case, r):
    s = _prepare_cache(case, r)
    s.update(q=(1.5 * r.normal(s["T"], case["H"], case["D"])).to(TYPES[case["x"]]), scale=case["D"] ** -0.5,
             window=case["window"], lse=case["lse"])
    return s


_PREPARE = {"turn": _prepare_turn, "append": _prepare_append, "attention": _prepare_attention}


def prepare(case, seed):
    s = _PREPARE[case["op"]](case, _Rand(seed))
    s["op"], s["interleaved"] = case["op"], case.get("interleaved", False)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _token_rows(s):
    """Sequence, place among its new tokens and position of each new token."""
    B, T, lens = s["lens"].numel(), s["T"], s["lens"].long()
    starts = torch.arange(B + 1, device=lens.device) * (T // B) if s["starts"] is None else s["starts"].long()
    t = torch.arange(T, device=lens.device)
    b = torch.searchsorted(starts, t, right=True) - 1
    i = t - starts[b]
    return starts, b, i, (lens - (starts[1:] - starts[:-1]))[b] + i


def _normed_turned(x, weight, eps, cos, sin, interleaved):
    """x [T, heads, D], normed for each head and turned, in x's type."""
    if eps is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(x.dtype)
    half = cos.shape[-1]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, rest], -1)


def _cos_sin(s, positions):
    """[T, 1, rot / 2] cosines and sines: pair j's from the position of its axis."""
    half = s["table"].shape[1] // 2
    j = torch.arange(half, device=positions.device)
    at = positions.long()[:, None] if s["axes"] is None else positions.long()[:, s["axes"].long()]
    return s["table"][at, j][:, None], s["table"][at, half + j][:, None]


def _plain_turn(s):
    cos, sin = _cos_sin(s, s["positions"])
    turned = lambda x, w: _normed_turned(x.float(), w, s["eps"], cos, sin, s["interleaved"]).to(x.dtype)
    return turned(s["q"], s["wq"]), turned(s["kn"], s["wk"])


def _plain_codes(x):
    """x [T, Hkv, D] -> bytes [T, Hkv, D / 2], scales [T, Hkv, 4]."""
    T, Hkv, D = x.shape
    quarters = x.view(T, Hkv, 4, D // 4)
    scale = (quarters.abs().amax(-1).double() / 7.5).bfloat16().clamp_min(2.0 ** -126)
    n = (quarters / scale.to(x.dtype)[..., None]).round().clamp(-8, 7).to(torch.int16) + 8
    words = torch.stack([n[:, :, 0] | n[:, :, 1] << 4, n[:, :, 2] | n[:, :, 3] << 4], -1)
    return words.to(torch.uint8).view(T, Hkv, D // 2), scale


def _plain_append(s):
    size = s["k"].shape[2]
    _, b, _, pos = _token_rows(s)
    cos, sin = _cos_sin(s, pos if s["positions"] is None else s["positions"])
    key = _normed_turned(s["kn"].double(), s["wk"], s["eps"], cos.double(), sin.double(), s["interleaved"])
    page_of, slot = s["pages"][b, pos // size].long(), pos % size
    s["k"][page_of, :, slot], s["ks"][page_of, :, slot] = _plain_codes(key)
    s["v"][page_of, :, slot], s["vs"][page_of, :, slot] = _plain_codes(s["vn"].float())
    q = _normed_turned(s["q"].float(), s["wq"], s["eps"], cos, sin, s["interleaved"]).to(s["q"].dtype)
    return q, s["k"], s["ks"], s["v"], s["vs"]


def _plain_values(codes, scales):
    """[..., D / 2] bytes and [..., 4] scales -> [..., D] in 32 bits."""
    w = codes.unflatten(-1, (-1, 2))
    n = torch.stack([w[..., 0] & 15, w[..., 0] >> 4, w[..., 1] & 15, w[..., 1] >> 4], -2)
    return ((n.float() - 8) * scales.float()[..., None]).flatten(-2)


def _plain_attention(s):
    q, pages, lens = s["q"], s["pages"].long(), s["lens"].long()
    (B, per), (P, Hkv, size, half) = pages.shape, s["k"].shape
    T, H, n, D = q.shape[0], q.shape[1], s["most"], 2 * half
    starts, b, i, _ = _token_rows(s)

    def values(codes, scales):
        return _plain_values(codes[pages], scales[pages]).transpose(1, 2).reshape(B, Hkv, per * size, D)

    rows = torch.zeros(B, n, H, D, device=q.device)
    rows[b, i] = q.float()
    rows = rows.view(B, n, Hkv, H // Hkv, D).transpose(1, 2).reshape(B, Hkv, -1, D)
    w = (rows @ values(s["k"], s["ks"]).transpose(2, 3)).mul_(s["scale"]).view(B, Hkv, n, H // Hkv, -1)
    pos = (lens - (starts[1:] - starts[:-1]))[:, None] + torch.arange(n, device=q.device)
    key = torch.arange(per * size, device=q.device)
    seen = key <= pos[:, :, None]
    if s["window"]:
        seen &= key > pos[:, :, None] - s["window"]
    w.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    w.sub_(top).exp_()
    total = w.sum(-1, keepdim=True)
    out = (w.view(B, Hkv, -1, per * size) @ values(s["v"], s["vs"])).view(B, Hkv, n, H // Hkv, D)
    out = torch.where(total > 0, out / total, 0.0)
    pick = lambda y: y.transpose(1, 2).reshape(B, n, H, -1)[b, i]
    out = pick(out).to(q.dtype)
    return (out, pick(top + total.log())[:, :, 0]) if s["lse"] else out


_PLAIN = {"turn": _plain_turn, "append": _plain_append, "attention": _plain_attention}


# ---------------------------------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def _own(s):
    op = s["op"]
    if op == "turn":
        from siliconfer_b200.rotary import qk_norm_rotary
        return qk_norm_rotary(s["q"], s["kn"], s["positions"], s["table"], q_weight=s["wq"], k_weight=s["wk"], eps=s["eps"],
                              interleaved=s["interleaved"], axes=s["axes"])
    if op == "append":
        from siliconfer_b200.paged_kv4 import paged4_append
        q = paged4_append(s["kn"], s["vn"], s["k"], s["ks"], s["v"], s["vs"], s["pages"], s["lens"], starts=s["starts"],
                          q=s["q"], table=s["table"], interleaved=s["interleaved"], positions=s["positions"],
                          axes=s["axes"], q_weight=s["wq"], k_weight=s["wk"], eps=s["eps"])
        return q, s["k"], s["ks"], s["v"], s["vs"]
    from siliconfer_b200.paged_kv4 import paged4_attention
    return paged4_attention(s["q"], s["k"], s["ks"], s["v"], s["vs"], s["pages"], s["lens"], starts=s["starts"],
                            scale=s["scale"], window=s["window"], return_lse=s["lse"])


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_heads(case, s, x, weight, places):
    """x [T, heads, D] normed and turned: places [T, axes] are the tokens' positions."""
    y = x.double()
    if case["norm"]:
        y = weight.double() * y / ((y ** 2).sum(-1, keepdim=True) / case["D"] + EPS).sqrt()
    half = case["rot"] // 2
    _, sections = _angles(case, _Rand(0), 1)
    axis = torch.tensor(_axis_of_pairs(sections, True), device=x.device)
    freq = ROPE_BASE ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = places.double()[:, axis] * freq
    z = torch.complex(angle.cos().float().double(), angle.sin().float().double())[:, None]
    if case["interleaved"]:
        lo, hi = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    else:
        lo, hi = slice(0, half), slice(half, 2 * half)
    y = y.clone()
    turned = torch.complex(y[..., lo].contiguous(), y[..., hi].contiguous()) * z
    y[..., lo], y[..., hi] = turned.real, turned.imag
    return y


def _exact_turn(case, s):
    places = s["positions"].view(case["T"], -1)
    return _exact_heads(case, s, s["q"], s["wq"], places), _exact_heads(case, s, s["kn"], s["wk"], places)


def _nearest_bf16(x):
    """8 significant bits, ties to even (no value here is subnormal)."""
    step = torch.exp2(torch.floor(torch.log2(x.clamp_min(2.0 ** -126))) - 7)
    return torch.round(x / step) * step


def _exact_append(case, s):
    lens, news = _counts(case)
    size, pages, D = case["page"], s["pages"].cpu().tolist(), case["D"]
    at = torch.cat([torch.arange(l - c, l) for l, c in zip(lens, news)]).to(s["k"].device)
    places = at[:, None] if s["positions"] is None else s["positions"]
    q = _exact_heads(case, s, s["q"], s["wq"], places)
    new = _exact_heads(case, s, s["kn"], s["wk"], places), s["vn"].double()
    slots = [(pages[b][p // size], p % size) for b, (l, c) in enumerate(zip(lens, news)) for p in range(l - c, l)]
    page_of, slot = torch.tensor(slots, device=q.device).view(-1, 2).T
    out = [q]
    for x, codes, scales in ((new[0], s["k"], s["ks"]), (new[1], s["v"], s["vs"])):
        codes, scales = codes.int(), scales.double()
        total = torch.zeros(x.shape[:2] + (D // 4,), dtype=torch.int32, device=x.device)
        quarter_scales = []
        for c in range(4):
            part = x[:, :, c * (D // 4):(c + 1) * (D // 4)]
            scale = _nearest_bf16(part.abs().max(-1).values / 7.5).clamp_min(2.0 ** -126)
            quarter_scales.append(scale)
            total += (torch.round(part / scale[..., None]).clamp(-8, 7).int() + 8) * 16 ** c
        codes[page_of, :, slot] = torch.stack([total % 256, total // 256], -1).flatten(-2)
        scales[page_of, :, slot] = torch.stack(quarter_scales, -1)
        out += [codes.to(torch.uint8), scales]
    return tuple(out)


def _exact_attention(case, s):
    lens, news = _counts(case)
    Hkv, D, G = case["Hkv"], case["D"], case["H"] // case["Hkv"]

    def take(codes, scales, p, l):
        word = codes[p].int()
        word = word[..., 0::2] + 256 * word[..., 1::2]
        parts = [((word // 16 ** c) % 16 - 8).double() * scales[p][..., c:c + 1].double() for c in range(4)]
        return torch.cat(parts, -1).permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :l]

    outs, lses, at = [], [], 0
    for b, (l, c) in enumerate(zip(lens, news)):
        if not c:
            continue
        p = s["pages"][b, :-(-l // case["page"])].long()
        k, v = take(s["k"], s["ks"], p, l), take(s["v"], s["vs"], p, l)
        q = s["q"][at:at + c].double().view(c, Hkv, G, D).permute(1, 2, 0, 3)
        at += c
        logits = torch.einsum("hgid,hjd->hgij", q, k) * case["D"] ** -0.5
        far = torch.arange(l - c, l, device=q.device)[:, None] - torch.arange(l, device=q.device)
        hidden = (far < 0) | (far >= case["window"]) if case["window"] else far < 0
        logits = logits.masked_fill(hidden, -math.inf)
        lses.append(torch.logsumexp(logits, -1).permute(2, 0, 1).reshape(c, -1))
        outs.append(torch.einsum("hgij,hjd->ihgd", torch.softmax(logits, -1), v).reshape(c, -1, D))
    out = torch.cat(outs)
    return (out, torch.cat(lses)) if case["lse"] else out


def exact(case, seed):
    s = prepare(case, seed)
    return {"turn": _exact_turn, "append": _exact_append, "attention": _exact_attention}[case["op"]](case, s)
