"""The 8-bit decoder operators: what they compute, on which sizes, and what each has to move.

Four operators of a decoder layer that keeps its activations and its cache in e4m3 (8-bit floating point):

  norm       root-mean-square norm with the residual's addition; the output in the input's type, or in e4m3 with one
             scale for each row and 128 columns.
  linear     product of such rows with an e4m3 weight that has one scale for each 128 x 128 block.
  append     rotary positions on queries and keys, and keys and values written into the e4m3 pages of a cache with one
             power-of-two scale for each page and kv head.
  attention  attention of one or more new tokens of each sequence over these pages.

``run`` computes them in plain torch operations in 32 bits, or, with ``own`` set, through the public functions of
siliconfer_b200.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
ROPE_BASE = 10000.0


# ---------------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # One token of a 4096-wide decoder on its way to the query, key and value projections: launch latency.
        dict(name="norm_1x4096", op="norm", T=1, K=4096, x="bf16", residual=True, quant=True),
        # A prompt chunk of 4096 tokens at the 8192-wide shape: memory traffic.
        dict(name="norm_4096x8192", op="norm", T=4096, K=8192, x="bf16", residual=True, quant=True),
        # One token through a 4096 x 4096 projection (the weight read is all there is).
        dict(name="linear_1x4096x4096", op="linear", T=1, K=4096, N=4096, out="bf16", bias=False),
        # A short prompt through the gate projection of the 896-wide decoder, ragged in tokens, biased, 32-bit output.
        dict(name="linear_77x896x4864", op="linear", T=77, K=896, N=4864, out="f32", bias=True),
        # A batch of 16 decoding sequences through the gate projection of the 8192-wide decoder.
        dict(name="linear_16x8192x28672", op="linear", T=16, K=8192, N=28672, out="bf16", bias=False),
        # A prompt of 2048 tokens through the 4096 -> 11008 projection: tensor cores.
        dict(name="linear_2048x4096x11008", op="linear", T=2048, K=4096, N=11008, out="bf16", bias=False),
        # A decode step of 8 sequences with 32 heads: one token each, pages partly filled.
        dict(name="append_8x1_32h", op="append", B=8, n=1, S=1500, H=32, Hkv=32, D=128, page=64, rot=128,
             interleaved=False, x="bf16", ragged=True),
        # A prompt chunk of 4096 tokens in 4 sequences with 64 query and 8 kv heads.
        dict(name="append_4x1024_64h", op="append", B=4, n=1024, S=2000, H=64, Hkv=8, D=128, page=64, rot=128,
             interleaved=False, x="bf16", ragged=False),
        # One short conversation of the 896-wide decoder (14 query and 2 kv heads of 64): launch latency.
        dict(name="attention_1x1000_14h", op="attention", B=1, n=1, S=1000, H=14, Hkv=2, D=64, page=16, window=0,
             x="bf16", ragged=False, lse=False),
        # A decode step of 16 sequences of 8192 tokens, 64 query and 8 kv heads: the cache read.
        dict(name="attention_16x8192_64h", op="attention", B=16, n=1, S=8192, H=64, Hkv=8, D=128, page=64, window=0,
             x="bf16", ragged=False, lse=False),
        # A served batch of 64 sequences of 0 to 4096 tokens with 32 heads of their own, 16-bit floating point.
        dict(name="attention_64x4096_32h", op="attention", B=64, n=1, S=4096, H=32, Hkv=32, D=128, page=32, window=0,
             x="f16", ragged=True, lse=False),
        # Prompt chunks of up to 256 tokens beside decoding sequences, 64 query and 8 kv heads.
        dict(name="attention_8x256_64h", op="attention", B=8, n=256, S=4000, H=64, Hkv=8, D=128, page=64, window=0,
             x="bf16", ragged=True, lse=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width of this repository's decoders, or any odd one."""
    known = [w for w in (128, 896, 1024, 4096, 4864, 8192, 11008, 28672) if lo <= w <= hi]
    return rng.choice(known) if known and rng.random() < 0.5 else max(lo, min(hi - 1, _log(rng, lo, hi)) | 1)


def draw(rng):
    op = rng.choice(["norm", "linear", "append", "attention"])
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        return dict(op=op, T=_log(rng, 1, 4096), K=_width(rng, 64, 8192), x=x, residual=rng.random() < 0.7,
                    quant=rng.random() < 0.6)
    if op == "linear":
        T = _log(rng, 1, 2048)
        K = _width(rng, 64, 8192)
        most = min(28672, 235_000_000 // K, 2048 * 4096 * 11008 // (T * K))
        return dict(op=op, T=T, K=K, N=_width(rng, 64, max(128, most)), out=x, bias=rng.random() < 0.5)
    H, Hkv = rng.choice([(14, 2), (32, 32), (64, 8), (8, 1), (20, 20)])
    D = rng.choice([64, 128, 128, 256] + ([96] if H != 32 else []))
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        B = _log(rng, 1, 64)
        n = _log(rng, 1, min(1024, 16384 * 128 // (B * H * D)) or 1)
        return dict(op=op, B=B, n=n, S=n + _log(rng, 1, 2000), H=H, Hkv=Hkv, D=D, page=page,
                    rot=rng.choice([D, D, D // 2]), interleaved=rng.random() < 0.5, x=x, ragged=rng.random() < 0.5)
    B = _log(rng, 1, 64)
    S = _log(rng, 16, min(32768, 100_000_000 // (B * Hkv * D)))
    n = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, min(128, S, 16_000_000 // (B * H * S))))
    return dict(op=op, B=B, n=n, S=max(S, n), H=H, Hkv=Hkv, D=D, page=page,
                window=rng.choice([0, 0, _log(rng, 8, 4096)]), x=x, ragged=rng.random() < 0.5, lse=rng.random() < 0.5)


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
    op = case["op"]
    if op == "norm":
        T, K, e = case["T"], case["K"], SIZE[case["x"]]
        out = T * K + 4 * T * (-(-K // 128)) if case["quant"] else T * K * e
        return {"bytes": T * K * e * (3 if case["residual"] else 1) + K * e + out, "flops": 6 * T * K}
    if op == "linear":
        T, K, N = case["T"], case["K"], case["N"]
        kb, nb = -(-K // 128), -(-N // 128)
        return {"bytes": T * K + N * K + 4 * kb * (T + nb) + T * N * SIZE[case["out"]] + (4 * N if case["bias"] else 0),
                "flops": 2 * T * N * K}
    H, Hkv, D, e = case["H"], case["Hkv"], case["D"], SIZE[case["x"]]
    lens, news = _counts(case)
    T = sum(news)
    if op == "append":
        pages = sum((l - 1) // case["page"] - (l - c) // case["page"] + 1 for l, c in zip(lens, news) if c)
        return {"bytes": T * D * (e * (2 * H + 2 * Hkv) + 2 * Hkv) + T * case["rot"] * 4 + 12 * Hkv * pages,
                "flops": T * D * (6 * (H + Hkv) + 4 * Hkv)}
    w = case["window"]
    keys = sum(min(l, w + c - 1) if w else l for l, c in zip(lens, news) if c)
    pairs = 0
    for l, c in zip(lens, news):
        for p in range(l - c, l):
            pairs += min(p + 1, w) if w else p + 1
    return {"bytes": keys * Hkv * D * 2 + 8 * Hkv * (keys // case["page"]) + 2 * T * H * D * e, "flops": 4 * pairs * H * D}


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

    def activations(self, T, K):
        """A residual stream: most channels near one, about one in a hundred twenty times as large."""
        big = torch.where(self.uniform(K) < 0.01, 20.0, 1.0)
        return self.normal(T, K) * big


def _padded_codes(values):
    """e4m3 codes whose rows start at multiples of 16 bytes."""
    T, K = values.shape
    store = torch.zeros(T, (K + 15) // 16 * 16, dtype=torch.uint8, device=values.device)
    store[:, :K] = values.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    return store.view(torch.float8_e4m3fn)[:, :K]


def _prepare_norm(case, r):
    T, K, dt = case["T"], case["K"], TYPES[case["x"]]
    return {"x": r.activations(T, K).to(dt), "weight": (1 + 0.1 * r.normal(K)).to(dt),
            "residual": r.activations(T, K).to(dt) if case["residual"] else None}


def _prepare_linear(case, r):
    T, K, N = case["T"], case["K"], case["N"]
    kb, nb = -(-K // 128), -(-N // 128)
    pad = torch.nn.functional.pad
    x = pad(r.activations(T, K), (0, kb * 128 - K)).view(T, kb, 128)
    sx = (x.abs().amax(2) / E4M3_MAX).clamp_min(1e-12)
    w = pad(0.02 * r.normal(N, K), (0, kb * 128 - K, 0, nb * 128 - N)).view(nb, 128, kb, 128)
    sw = (w.abs().amax((1, 3)) / E4M3_MAX).clamp_min(1e-12)
    return {"x": _padded_codes((x / sx[:, :, None]).view(T, -1)[:, :K]), "sx": sx,
            "w": _padded_codes((w / sw[:, None, :, None]).view(nb * 128, -1)[:N, :K]), "sw": sw,
            "bias": r.normal(N) if case["bias"] else None, "out": TYPES[case["out"]]}


def _prepare_cache(case, r):
    """Pages in random order; the contents of a cache whose pages were scaled by their largest values."""
    B, S, Hkv, D, page = case["B"], case["S"], case["Hkv"], case["D"], case["page"]
    per = -(-S // page)
    P = B * per + 3
    table = torch.randperm(P, generator=r.g, device=r.dev)[: B * per].view(B, per).to(torch.int32)
    lens, news = _counts(case)
    starts = torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32, device=r.dev)
    codes, scales = [], []
    for _ in range(2):
        codes.append((r.normal(P, Hkv, page, D) * 80).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn))
        scales.append(torch.exp2(r.integers(-7, -4, P, Hkv).float()))
    return {"k": codes[0], "ks": scales[0], "v": codes[1], "vs": scales[1], "pages": table,
            "lens": torch.tensor(lens, dtype=torch.int32, device=r.dev), "starts": starts if case["ragged"] else None,
            "most": max(news), "T": sum(news)}


def _prepare_append(case, r):
    s = _prepare_cache(case, r)
    H, Hkv, D, dt = case["H"], case["Hkv"], case["D"], TYPES[case["x"]]
    # what a fused projection gives: queries, keys and values side by side in each token's row
    qkv = r.normal(s["T"], (H + 2 * Hkv) * D).to(dt)
    part = lambda a, h: qkv[:, a * D:(a + h) * D].view(s["T"], h, D)
    half = case["rot"] // 2
    freq = ROPE_BASE ** (-torch.arange(half, device=r.dev, dtype=torch.float64) / half)
    angle = torch.arange(case["S"], device=r.dev, dtype=torch.float64)[:, None] * freq
    s.update(q=part(0, H), kn=part(H, Hkv), vn=part(H + Hkv, Hkv),
             table=torch.cat([angle.cos(), angle.sin()], 1).float(), interleaved=case["interleaved"])
    return s


def _prepare_attention(case, r):
    s = _prepare_cache(case, r)
    s.update(q=(2 * r.normal(s["T"], case["H"], case["D"])).to(TYPES[case["x"]]), scale=case["D"] ** -0.5,
             window=case["window"], lse=case["lse"])
    return s


_PREPARE = {"norm": _prepare_norm, "linear": _prepare_linear, "append": _prepare_append, "attention": _prepare_attention}


def prepare(case, seed):
    s = _PREPARE[case["op"]](case, _Rand(seed))
    s["op"], s["quant"] = case["op"], case.get("quant", False)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _plain_norm(s):
    x, w = s["x"], s["weight"]
    h = x.float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * w.float()
    more = () if s["residual"] is None else (h.to(x.dtype),)
    if not s["quant"]:
        return (y.to(x.dtype),) + more
    T, K = y.shape
    kb = -(-K // 128)
    y = torch.nn.functional.pad(y, (0, kb * 128 - K)).view(T, kb, 128)
    amax = y.abs().amax(2)
    scale = torch.where(amax == 0, 1.0, amax / E4M3_MAX)
    codes = (y / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return (codes.view(T, -1)[:, :K], scale) + more


def _plain_linear(s):
    x, w = s["x"], s["w"]
    N, K = w.shape
    xf = x.float() * s["sx"].repeat_interleave(128, 1)[:, :K]
    wf = w.float() * s["sw"].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = xf @ wf.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["out"])


def _token_rows(s):
    """Sequence, place among its new tokens and position of each new token."""
    B, T, lens = s["lens"].numel(), s["T"], s["lens"].long()
    starts = torch.arange(B + 1, device=lens.device) * (T // B) if s["starts"] is None else s["starts"].long()
    t = torch.arange(T, device=lens.device)
    b = torch.searchsorted(starts, t, right=True) - 1
    i = t - starts[b]
    return starts, b, i, (lens - (starts[1:] - starts[:-1]))[b] + i


def _rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, rest], -1)


def _plain_write(new, codes, scales, page_of, slot):
    """Writes the rows `new` [T, Hkv, D] into their pages; a page's scale grows where the new rows need it."""
    P, Hkv = scales.shape
    finite = torch.where(torch.isfinite(new), new.abs(), 0.0).amax(2)
    amax = torch.zeros_like(scales).scatter_reduce(0, page_of[:, None].expand(-1, Hkv), finite, "amax")
    mant, ex = torch.frexp(amax)
    need = torch.exp2(torch.where(amax == 0, -64, torch.where(mant <= 0.875, ex - 9, ex - 8)).clamp_min(-64).float())
    touched = torch.zeros(P, dtype=torch.bool, device=new.device).index_fill(0, page_of, True)
    first = torch.full((P,), 1 << 20, device=new.device).scatter_reduce(0, page_of, slot, "amin")
    fresh = touched & (first == 0)
    grown = torch.where(fresh[:, None], need, torch.where(touched[:, None], torch.maximum(scales, need), scales))
    raw = codes.view(torch.uint8)
    # pages that held tokens before: at most one for each run of new tokens, where that run starts
    head = page_of[(slot == first[page_of]) & (slot > 0)]
    old = codes[head].float() * (scales[head] / grown[head])[:, :, None, None]
    keep = torch.arange(codes.shape[2], device=new.device) < first[head][:, None]
    raw[head] = torch.where(keep[:, None, :, None], old.to(torch.float8_e4m3fn).view(torch.uint8), raw[head])
    put = (new / grown[page_of][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    raw[page_of, :, slot] = put.view(torch.uint8)
    scales.copy_(grown)


def _plain_append(s):
    q, table, size = s["q"], s["table"], s["k"].shape[2]
    _, b, _, pos = _token_rows(s)
    cos, sin = table[pos].chunk(2, 1)
    turn = lambda x: _rotate(x.float(), cos[:, None], sin[:, None], s["interleaved"])
    page_of, slot = s["pages"][b, pos // size].long(), pos % size
    _plain_write(turn(s["kn"]), s["k"], s["ks"], page_of, slot)
    _plain_write(s["vn"].float(), s["v"], s["vs"], page_of, slot)
    return turn(q).to(q.dtype), s["k"], s["ks"], s["v"], s["vs"]


def _plain_attention(s):
    q, pages, lens = s["q"], s["pages"].long(), s["lens"].long()
    (B, per), (P, Hkv, size, D) = pages.shape, s["k"].shape
    T, H, n = q.shape[0], q.shape[1], s["most"]
    starts, b, i, _ = _token_rows(s)

    def values(codes, scales):
        x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * scales[pages][..., None, None]
        return x.transpose(1, 2).reshape(B, Hkv, per * size, D)

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


_PLAIN = {"norm": _plain_norm, "linear": _plain_linear, "append": _plain_append, "attention": _plain_attention}


# ---------------------------------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def _own(s):
    op = s["op"]
    if op == "norm":
        from siliconfer_b200.norm import rms_norm, rms_norm_e4m3
        y = (rms_norm_e4m3 if s["quant"] else rms_norm)(s["x"], s["weight"], eps=EPS, residual=s["residual"])
        return y if isinstance(y, tuple) else (y,)
    if op == "linear":
        from siliconfer_b200.fp8_linear import fp8_linear
        return fp8_linear(s["x"], s["sx"], s["w"], s["sw"], bias=s["bias"], out_dtype=s["out"])
    if op == "append":
        from siliconfer_b200.paged_kv import paged_append
        q = paged_append(s["kn"], s["vn"], s["k"], s["ks"], s["v"], s["vs"], s["pages"], s["lens"], starts=s["starts"],
                         q=s["q"], table=s["table"], interleaved=s["interleaved"])
        return q, s["k"], s["ks"], s["v"], s["vs"]
    from siliconfer_b200.paged_kv import paged_attention
    return paged_attention(s["q"], s["k"], s["ks"], s["v"], s["vs"], s["pages"], s["lens"], starts=s["starts"],
                           scale=s["scale"], window=s["window"], return_lse=s["lse"])


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _nearest_e4m3(x):
    """The e4m3 value nearest to x (ties to the even significand), saturated at 448: 3 bits after the leading one, and
    steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))).clamp_min(-6) - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_norm(case, s):
    h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
    y = s["weight"].double() * h / ((h ** 2).sum(1, keepdim=True) / case["K"] + EPS).sqrt()
    more = [] if s["residual"] is None else [h]
    if not case["quant"]:
        return tuple([y] + more)
    codes, scales = torch.empty_like(y), []
    for c in range(0, case["K"], 128):
        g = y[:, c:c + 128]
        scale = g.abs().max(1).values / E4M3_MAX
        scales.append(torch.where(scale > 0, scale, torch.ones_like(scale)))
        codes[:, c:c + 128] = _nearest_e4m3(g / scales[-1][:, None])
    return tuple([codes, torch.stack(scales, 1)] + more)


def _exact_linear(case, s):
    x, w, K = s["x"].double(), s["w"].double(), case["K"]
    col = torch.arange(K, device=x.device) // 128
    row = torch.arange(case["N"], device=x.device) // 128
    y = (x * s["sx"].double()[:, col]) @ (w * s["sw"].double()[row][:, col]).T
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_turn(case, x, first):
    """Rotary positions of `x` [n, heads, D], whose first row has position `first`, from the table's 32-bit values."""
    half = case["rot"] // 2
    freq = ROPE_BASE ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = torch.arange(first, first + x.shape[0], device=x.device, dtype=torch.float64)[:, None] * freq
    z = torch.complex(angle.cos().float().double(), angle.sin().float().double())[:, None]
    y = x.double()
    lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
    turned = torch.complex(y[..., lo].contiguous(), y[..., hi].contiguous()) * z
    y = y.clone()
    y[..., lo], y[..., hi] = turned.real, turned.imag
    return y


def _exact_append(case, s):
    lens, news = _counts(case)
    size, pages = case["page"], s["pages"].cpu().tolist()
    kd, vd, ks, vs = s["k"].double(), s["v"].double(), s["ks"].double(), s["vs"].double()
    queries, at = [], 0
    for b, (l, c) in enumerate(zip(lens, news)):
        if not c:
            continue
        queries.append(_exact_turn(case, s["q"][at:at + c], l - c))
        new = {0: _exact_turn(case, s["kn"][at:at + c], l - c), 1: s["vn"][at:at + c].double()}
        at += c
        for j in range((l - c) // size, (l - 1) // size + 1):
            lo, hi, p = max(l - c, j * size), min(l, (j + 1) * size), pages[b][j]
            for which, (cache, scales) in enumerate(((kd, ks), (vd, vs))):
                rows = new[which][lo - (l - c):hi - (l - c)].transpose(0, 1)
                amax = rows.abs().amax((1, 2))
                scale = torch.exp2(torch.ceil(torch.log2((amax / E4M3_MAX).clamp_min(2.0 ** -64))))
                if lo > j * size:
                    scale = torch.maximum(scale, scales[p])
                    before = slice(0, lo - j * size)
                    cache[p][:, before] = _nearest_e4m3(cache[p][:, before] * (scales[p] / scale)[:, None, None])
                cache[p][:, lo - j * size:hi - j * size] = _nearest_e4m3(rows / scale[:, None, None])
                scales[p] = scale
    return torch.cat(queries), kd, ks, vd, vs


def _exact_attention(case, s):
    lens, news = _counts(case)
    Hkv, D, G = case["Hkv"], case["D"], case["H"] // case["Hkv"]
    outs, lses, at = [], [], 0
    for b, (l, c) in enumerate(zip(lens, news)):
        if not c:
            continue
        p = s["pages"][b, :-(-l // case["page"])].long()
        take = lambda codes, scales: ((codes[p].double() * scales[p].double()[:, :, None, None])
                                      .permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :l])
        k, v = take(s["k"], s["ks"]), take(s["v"], s["vs"])
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
    return {"norm": _exact_norm, "linear": _exact_linear, "append": _exact_append,
            "attention": _exact_attention}[case["op"]](case, s)
