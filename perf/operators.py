"""Cases of the operators around a quantised, paged KV cache.

One decoder layer of a served model, next to the residual norm and the block
selection (``dsa_topk_page_table_transform``) that the framework has:

* ``rope``:  per-head RMSNorm of queries and keys and the rotation by position, one pass;
* ``write``: the new tokens' keys and values, quantised with one scale per token and head, into their pages;
* ``read``:  a sequence's keys and values, back from their pages as dense 16-bit tensors;
* ``chunk``: both, as chunked prefill does (its chunk is written, then the whole context read);
* ``attn``:  attention of each query row over the pages that were selected for it.

Shapes: q [B, Q, Hq, D]; k, v [B, Q, H, D]; caches [P, H, bs, D] with scales
[P, H, bs]; page_table [B, NB]; q_pos [B, Q]; kv_lens [B]; a selection
(blocks, pages) [B, H, Q, K] as the block selection writes it.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_QT = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_QMAX = {"e4m3": 448.0, "int8": 127.0}
_MIN_SCALE = 1e-12
_EPS = 1e-6


# ---------------------------------------------------------------- the cases
def _rope(B, Q, Hq, H, D, rot, dtype, interleaved=False, pad=0):
    return {"op": "rope", "B": B, "Q": Q, "Hq": Hq, "H": H, "D": D, "rot": rot, "dtype": dtype,
            "interleaved": interleaved, "pad": pad, "max_pos": 16384}


def _write(B, Q, H, D, bs, ctx, dtype, qt, pad=0):
    return {"op": "write", "B": B, "Q": Q, "H": H, "D": D, "bs": bs, "ctx": ctx, "dtype": dtype, "qt": qt,
            "pad": pad}


def _read(B, H, D, bs, ctx, dtype, qt):
    return {"op": "read", "B": B, "H": H, "D": D, "bs": bs, "ctx": ctx, "dtype": dtype, "qt": qt}


def _chunk(B, Q, H, D, bs, ctx, dtype, qt):
    return {"op": "chunk", "B": B, "Q": Q, "H": H, "D": D, "bs": bs, "ctx": ctx, "dtype": dtype, "qt": qt, "pad": 0}


def _attn(B, Q, H, G, D, bs, K, ctx, dtype, qt):
    return {"op": "attn", "B": B, "Q": Q, "H": H, "G": G, "D": D, "bs": bs, "K": K, "ctx": ctx, "dtype": dtype,
            "qt": qt}


def listed():
    return [
        # one sequence decodes one token: launch latency is all there is
        dict(_rope(1, 1, 32, 8, 128, 128, "bf16"), name="rope_decode_1"),
        # a long prompt's prefill: bandwidth
        dict(_rope(1, 8192, 32, 8, 128, 128, "bf16"), name="rope_prefill_8192"),
        # a padded batch of short prompts, part of each head rotated in adjacent pairs
        dict(_rope(5, 333, 24, 4, 64, 32, "fp16", interleaved=True, pad=1), name="rope_padded_5x333"),
        # a decode batch appends one token to each sequence
        dict(_write(64, 1, 8, 128, 64, 4096, "bf16", "e4m3"), name="write_decode_64"),
        # two prompts of up to 4096 tokens, the second one shorter and padded
        dict(_write(2, 4096, 8, 128, 64, 8192, "bf16", "e4m3", pad=1), name="write_prefill_2x4096"),
        # one short context read back for a dense pass
        dict(_read(1, 8, 128, 64, 333, "bf16", "e4m3"), name="read_1x333"),
        # eight long contexts of unlike length read back
        dict(_read(8, 8, 128, 64, 8192, "bf16", "e4m3"), name="read_8x8192"),
        # chunked prefill: 512 new tokens written, then the whole context read back
        dict(_chunk(4, 512, 4, 64, 32, 4000, "fp16", "int8"), name="chunk_4x512_int8"),
        # one sequence decodes: few rows, the selection is split over many blocks of threads
        dict(_attn(1, 1, 8, 4, 128, 64, 32, 8192, "bf16", "e4m3"), name="attn_decode_1"),
        # a decode batch with the widest selection: HBM bandwidth
        dict(_attn(32, 1, 8, 8, 128, 64, 128, 16384, "bf16", "e4m3"), name="attn_decode_32"),
        # four drafted tokens of each sequence verified at once
        dict(_attn(16, 4, 2, 16, 64, 128, 32, 12000, "fp16", "int8"), name="attn_verify_16x4_int8"),
        # the last part of a prompt, 16 query heads to a key head: tensor-core work
        dict(_attn(1, 256, 4, 16, 128, 64, 32, 16384, "bf16", "e4m3"), name="attn_prefill_256"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges; at most the largest listed case's work."""
    op = rng.choice(["rope", "write", "read", "chunk", "attn", "attn"])
    dtype, qt = rng.choice(["bf16", "fp16"]), rng.choice(["e4m3", "int8"])
    D = rng.choice([64, 128, 256])
    H = rng.randint(1, 8)
    B = _log(rng, 1, 64)
    bs = rng.choice([16, 32, 48, 64, 128])
    if op == "rope":
        Q = max(1, min(_log(rng, 1, 8192), 8192 * 128 // (B * D)))
        D = rng.choice([64, 80, 96, 128, 192, 256])
        return _rope(B, Q, H * rng.randint(1, 4), H, D, rng.choice([D, 32]), dtype, rng.random() < 0.4,
                     int(Q > 8 and rng.random() < 0.5))
    if op == "write":
        Q = max(1, min(_log(rng, 1, 4096), 8192 * 128 // (B * D)))
        return _write(B, Q, H, D, bs, Q + _log(rng, 16, 4096), dtype, qt, int(Q > 8 and rng.random() < 0.5))
    if op == "read":
        ctx = max(16, min(_log(rng, 16, 8192), 65536 * 128 // (B * D)))
        return _read(B, H, D, bs, ctx, dtype, qt)
    if op == "chunk":
        ctx = max(33, min(_log(rng, 64, 8192), 32768 * 128 // (B * D)))
        return _chunk(B, rng.randint(1, max(1, ctx // 4)), H, D, bs, ctx, dtype, qt)
    B = _log(rng, 1, 32)
    Q = rng.choice([1, 1, 2, 4, _log(rng, 5, 128)])
    G = rng.choice([1, 2, 4, 5, 8, 16])
    ctx = _log(rng, max(64, Q), 16384)
    K = rng.randint(1, 128)
    # rows x selected tokens x head size within the decode batch's, caches within its size
    K = max(1, min(K, 32 * 8 * 128 * 64 * 128 // (B * Q * H * bs * D)))
    ctx = max(Q, min(ctx, 32 * 8 * 16384 * 128 // (B * H * D)))
    return _attn(B, Q, H, G, D, bs, K, ctx, dtype, qt)


# ------------------------------------------------------- sizes from the case
def _lens(c):
    """Sequence lengths: the first is ctx, the others fall off to half of it (never below the new tokens)."""
    lo = c.get("Q", 1)
    return [max(lo, c["ctx"] - b * c["ctx"] // (2 * c["B"])) for b in range(c["B"])]


def _new(c):
    """New tokens of each sequence: with padding, every second sequence has a fifth less of them."""
    return [c["Q"] - (c["Q"] // 5 if c["pad"] and b % 2 == 1 else 0) for b in range(c["B"])]


def _nb(c):
    return -(-c["ctx"] // c["bs"])


def _valid_blocks(c):
    return [-(-n // c["bs"]) for n in _lens(c)]


def work(case):
    c, e = case, 2
    if c["op"] == "rope":
        t = sum(_new(c))
        head = c["D"] * e
        return {"bytes": 2 * t * (c["Hq"] + c["H"]) * head + t * (4 * c["rot"] + 8) + 2 * c["D"] * e,
                "flops": 8 * t * (c["Hq"] + c["H"]) * c["D"]}
    if c["op"] in ("write", "read", "chunk"):
        w = sum(_new(c)) if c["op"] != "read" else 0
        r = sum(_lens(c)) if c["op"] != "write" else 0
        vec = 2 * c["H"]  # a key and a value for every head
        per = c["D"] * e + c["D"] + 4
        return {"bytes": (w + r) * vec * per + (w + r // c["bs"]) * 8, "flops": (4 * w + r) * vec * c["D"]}
    rows, toks, uniq = c["H"] * c["Q"], 0, 0.0
    for n, nb in zip(_lens(c), _valid_blocks(c)):
        k = min(c["K"], nb)
        toks += rows * min(n, k * c["bs"])
        # expected number of different blocks that the Q rows of a head select
        uniq += c["H"] * min(n, c["bs"] * nb * (1 - (1 - k / nb) ** c["Q"]))
    R = c["B"] * rows
    return {"bytes": 2 * uniq * (c["D"] + 4) + R * (2 * c["G"] * c["D"] * e + 8 * c["K"]),
            "flops": 4 * c["G"] * c["D"] * toks}


# ------------------------------------------------------------------ the state
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _cache(g, c, pages):
    """A cache as its writer leaves it: tokens of unlike size, the largest value of each vector at the end of the range."""
    shape = (pages, c["H"], c["bs"], c["D"])
    size = torch.exp(0.5 * _randn(g, *shape[:3]))
    x = _randn(g, *shape)
    scale = x.abs().amax(-1) / _QMAX[c["qt"]]
    x = x / scale[..., None]
    codes = x.to(torch.float8_e4m3fn) if c["qt"] == "e4m3" else torch.round(x).to(torch.int8)
    return codes, scale * size


def _pages(g, c):
    """(page_table [B, NB], number of pages): pages handed out in no order, a few of them in nobody's hands."""
    n = c["B"] * _nb(c)
    return torch.randperm(n + 3, generator=g, device="cuda")[:n].view(c["B"], _nb(c)).to(torch.int32), n + 3


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    dt = _DT[c["dtype"]]
    B = c["B"]
    if c["op"] == "rope":
        Q, Hq, H, D = c["Q"], c["Hq"], c["H"], c["D"]
        # one fused projection gives queries, keys and values side by side
        qkv = _randn(g, B, Q, (Hq + 2 * H) * D, dtype=dt)
        s["q"] = qkv[..., :Hq * D].view(B, Q, Hq, D)
        s["k"] = qkv[..., Hq * D:(Hq + H) * D].view(B, Q, H, D)
        s["q_gamma"] = (1 + 0.1 * _randn(g, D)).to(dt)
        s["k_gamma"] = (1 + 0.1 * _randn(g, D)).to(dt)
        half = c["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        ang = torch.arange(c["max_pos"], device="cuda", dtype=torch.float64)[:, None] * freq
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], dim=1).float()
        first = torch.randint(0, c["max_pos"] - Q + 1, (B, 1), generator=g, device="cuda")
        i = torch.arange(Q, device="cuda")
        new = torch.tensor(_new(c), device="cuda")[:, None]
        s["positions"] = torch.where(i < new, first + i, -1).to(torch.int32)
        s["q_out"] = torch.zeros(B, Q, Hq, D, dtype=dt, device="cuda")
        s["k_out"] = torch.zeros(B, Q, H, D, dtype=dt, device="cuda")
        return s
    s["page_table"], pages = _pages(g, c)
    s["k_cache"], s["k_scale"] = _cache(g, c, pages)
    s["v_cache"], s["v_scale"] = _cache(g, c, pages)
    lens = torch.tensor(_lens(c), device="cuda")
    s["kv_lens"] = lens.to(torch.int32)
    if c["op"] in ("write", "chunk"):
        kv = _randn(g, B, c["Q"], 2 * c["H"] * c["D"], dtype=dt)
        s["k"] = kv[..., :c["H"] * c["D"]].view(B, c["Q"], c["H"], c["D"])
        s["v"] = kv[..., c["H"] * c["D"]:].view(B, c["Q"], c["H"], c["D"])
        i = torch.arange(c["Q"], device="cuda")
        new = torch.tensor(_new(c), device="cuda")[:, None]
        s["q_pos"] = torch.where(i < new, lens[:, None] - c["Q"] + i, -1).to(torch.int32)
    if c["op"] in ("read", "chunk"):
        s["k_out"] = torch.zeros(B, c["ctx"], c["H"], c["D"], dtype=dt, device="cuda")
        s["v_out"] = torch.zeros(B, c["ctx"], c["H"], c["D"], dtype=dt, device="cuda")
    if c["op"] == "attn":
        Q, H, K = c["Q"], c["H"], c["K"]
        s["q"] = 2 * _randn(g, B, Q, H * c["G"], c["D"], dtype=dt)
        pos = lens[:, None] - Q + torch.arange(Q, device="cuda")
        s["q_pos"] = pos.to(torch.int32)
        # a selection in the order of its scores; the first block and the row's own are always in it
        nb = _nb(c)
        score = torch.rand(B, H, Q, nb, generator=g, device="cuda")
        at = torch.arange(nb, device="cuda")
        last = (pos // c["bs"])[:, None, :, None]
        score = torch.where((at == 0) | (at == last), score + 1, score)
        score = torch.where(at <= last, score, -1.0)
        top, blocks = score.topk(min(K, nb), dim=-1)
        blocks = torch.where(top >= 0, blocks, -1)
        blocks = torch.nn.functional.pad(blocks, (0, K - blocks.shape[-1]), value=-1)
        table = s["page_table"].long()[:, None, None, :].expand(B, H, Q, nb)
        s["pages"] = torch.where(blocks >= 0, table.gather(3, blocks.clamp(min=0)), -1).to(torch.int32)
        s["blocks"] = blocks.to(torch.int32)
        s["out"] = torch.empty(B, Q, H * c["G"], c["D"], dtype=dt, device="cuda")
        s["lse"] = torch.empty(B, Q, H * c["G"], device="cuda")
        s["softmax_scale"] = c["D"] ** -0.5
    return s


# --------------------------------------------------------------------- a pass
_entry = {}


def _pkg():
    if not _entry:
        import flagos_kernelgen_72h_shanghai_2026_b200 as pkg
        _entry["pkg"] = pkg
    return _entry["pkg"]


def _own_run(s):
    c, p = s["case"], _pkg()
    if c["op"] == "rope":
        return p.qk_rmsnorm_rope(s["q"], s["k"], s["q_gamma"], s["k_gamma"], s["cos_sin"], s["positions"], s["q_out"],
                                 s["k_out"], _EPS, interleaved=c["interleaved"])
    cache = (s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"])
    if c["op"] == "attn":
        return p.dsa_paged_attention(s["q"], *cache, s["blocks"], s["pages"], s["q_pos"], s["kv_lens"], s["out"],
                                     s["lse"], s["softmax_scale"])
    if c["op"] in ("write", "chunk"):
        p.paged_kv_quant_write(s["k"], s["v"], *cache, s["page_table"], s["q_pos"])
    if c["op"] == "write":
        return _stored(s)
    return p.paged_kv_dequant_read(*cache, s["page_table"], s["kv_lens"], s["k_out"], s["v_out"])


def _stored(s):
    """The cache after a write. Whole codes stand for code times scale."""
    if s["case"]["qt"] == "e4m3":
        return s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]
    k, v = ((s[n + "_cache"].float() * s[n + "_scale"][..., None]).to(torch.bfloat16) for n in "kv")
    return k, s["k_scale"], v, s["v_scale"]


def run(state):
    if own:
        return _own_run(state)
    op = state["case"]["op"]
    if op == "rope":
        return _plain_rope(state)
    if op == "attn":
        return _plain_attn(state)
    if op in ("write", "chunk"):
        _plain_write(state)
    return _stored(state) if op == "write" else _plain_read(state)


def _plain_rotate(x, gamma, cos, sin, keep, old, interleaved):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * gamma.float()
    rot = 2 * cos.shape[-1]
    r, rest = y[..., :rot], y[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.where(keep, torch.cat([r, rest], dim=-1).to(x.dtype), old)


def _plain_rope(s):
    pos, inter = s["positions"], s["case"]["interleaved"]
    half = s["cos_sin"].shape[1] // 2
    row = s["cos_sin"][pos.clamp(min=0).long()][:, :, None, :]
    cos, sin = row[..., :half], row[..., half:]
    keep = (pos >= 0)[:, :, None, None]
    return (_plain_rotate(s["q"], s["q_gamma"], cos, sin, keep, s["q_out"], inter),
            _plain_rotate(s["k"], s["k_gamma"], cos, sin, keep, s["k_out"], inter))


def _plain_quant(x, qt):
    y = x.float()
    scale = (y.abs().amax(-1) / _QMAX[qt]).clamp(min=_MIN_SCALE)
    y = y * (1.0 / scale)[..., None]
    return (y.to(torch.float8_e4m3fn) if qt == "e4m3" else torch.round(y).to(torch.int8)).view(torch.uint8), scale


def _plain_write(s):
    c = s["case"]
    pos = s["q_pos"].long()
    page = s["page_table"].long().gather(1, pos.clamp(min=0) // c["bs"])
    # a padded token stands in for the first token of the batch, which is never padded
    n = torch.where(pos.flatten() >= 0, torch.arange(pos.numel(), device="cuda"), 0)
    page, off = page.flatten()[n], (pos % c["bs"]).flatten()[n]
    for x, codes, scales in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        q, sc = _plain_quant(x, c["qt"])
        codes.view(torch.uint8)[page, :, off] = q.flatten(0, 1)[n]
        scales[page, :, off] = sc.flatten(0, 1)[n]


def _plain_read(s):
    c = s["case"]
    keep = (torch.arange(c["ctx"], device="cuda") < s["kv_lens"][:, None])[:, :, None, None]
    table = s["page_table"].long()
    got = []
    for codes, scales, out in ((s["k_cache"], s["k_scale"], s["k_out"]), (s["v_cache"], s["v_scale"], s["v_out"])):
        x = codes.view(torch.uint8)[table].view(codes.dtype).float() * scales[table][..., None]  # [B, NB, H, bs, D]
        x = x.permute(0, 1, 3, 2, 4).flatten(1, 2)[:, :c["ctx"]]
        got.append(torch.where(keep, x.to(out.dtype), out))
    return tuple(got)


def _plain_attn(s):
    c = s["case"]
    B, Q, H, G, D, K, bs = (c[n] for n in ("B", "Q", "H", "G", "D", "K", "bs"))
    page = s["pages"].clamp(min=0).long()
    head = torch.arange(H, device="cuda")[:, None, None]
    at = s["blocks"][..., None].long() * bs + torch.arange(bs, device="cuda")
    seen = (s["blocks"][..., None] >= 0) & (at <= s["q_pos"][:, None, :, None, None]) & (
        at < s["kv_lens"][:, None, None, None, None])
    seen = seen.view(B, H, Q, 1, K * bs)

    def tokens(codes, scales):
        x = codes.view(torch.uint8)[page, head].view(codes.dtype).float()
        return (x * scales[page, head][..., None]).view(B, H, Q, K * bs, D)

    q = s["q"].float().view(B, Q, H, G, D).permute(0, 2, 1, 3, 4)
    score = torch.matmul(q, tokens(s["k_cache"], s["k_scale"]).transpose(-1, -2)) * s["softmax_scale"]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, tokens(s["v_cache"], s["v_scale"])) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1)
    return (out.permute(0, 2, 1, 3, 4).reshape(B, Q, H * G, D).to(s["q"].dtype),
            lse.permute(0, 2, 1, 3).reshape(B, Q, H * G))


# ---------------------------------------------------------------- in 64 bits
def _e4m3(v):
    """The e4m3 value nearest to v (ties to the even one), for |v| <= 448."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def _exact_rotate(x, gamma, cs, pos, old, interleaved):
    y = x.double()
    y = gamma.double() * y / torch.sqrt(y.square().sum(-1, keepdim=True) / y.shape[-1] + _EPS)
    half = cs.shape[1] // 2
    z = torch.view_as_complex(cs.double().view(-1, 2, half).transpose(1, 2).contiguous())[pos.clamp(min=0).long()]
    r = y[..., :2 * half].unflatten(-1, (half, 2) if interleaved else (2, half))
    r = (r if interleaved else r.transpose(-1, -2)).contiguous()
    r = torch.view_as_real(torch.view_as_complex(r) * z[:, :, None, :])
    y[..., :2 * half] = (r if interleaved else r.transpose(-1, -2)).flatten(-2)
    pad = pos < 0
    y[pad] = old.double()[pad]
    return y


def _exact_stored(s):
    """Values that the codes of both caches stand for without their scales, and the scales, after the write."""
    c, got = s["case"], []
    for x, codes, scales in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        val, sc = codes.double(), scales.double()
        for b in range(c["B"]):
            n = _new(c)[b]
            pos = s["q_pos"][b, :n].long()
            page, off = s["page_table"][b].long()[pos // c["bs"]], pos % c["bs"]
            y = x[b, :n].double()
            a = (y.abs().amax(-1) / _QMAX[c["qt"]]).clamp(min=_MIN_SCALE)
            y = y / a[..., None]
            val[page, :, off] = _e4m3(y) if c["qt"] == "e4m3" else torch.round(y)
            sc[page, :, off] = a
        got.append((val, sc))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "rope":
        return tuple(_exact_rotate(s[n], s[n + "_gamma"], s["cos_sin"], s["positions"], s[n + "_out"], c["interleaved"])
                     for n in "qk")
    if c["op"] in ("write", "chunk"):
        (kv, ks), (vv, vs) = _exact_stored(s)
    else:
        kv, ks, vv, vs = s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]
    if c["op"] == "write":
        if c["qt"] == "e4m3":
            return kv, ks, vv, vs
        return kv * ks[..., None], ks, vv * vs[..., None], vs
    lens = _lens(c)
    if c["op"] in ("read", "chunk"):
        got = []
        for val, sc, out in ((kv, ks, s["k_out"]), (vv, vs, s["v_out"])):
            full = out.double()
            for b in range(c["B"]):
                t = torch.arange(lens[b], device="cuda")
                page, off = s["page_table"][b].long()[t // c["bs"]], t % c["bs"]
                full[b, :lens[b]] = val[page, :, off].double() * sc[page, :, off].double()[..., None]
            got.append(full)
        return tuple(got)
    B, Q, H, G, D, bs = (c[n] for n in ("B", "Q", "H", "G", "D", "bs"))
    out = torch.zeros(B, Q, H, G, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Q, H, G), -math.inf, dtype=torch.float64, device="cuda")
    nb = _nb(c)
    t = torch.arange(nb * bs, device="cuda")
    for b in range(B):
        table = s["page_table"][b].long()
        for h in range(H):
            # the sequence's tokens in their order, each as often as a row selects its block
            k = (kv[table, h].double() * ks[table, h].double()[..., None]).view(nb * bs, D)
            v = (vv[table, h].double() * vs[table, h].double()[..., None]).view(nb * bs, D)
            sel = s["blocks"][b, h].long()
            times = torch.zeros(Q, nb + 1, dtype=torch.float64, device="cuda")
            times.scatter_add_(1, torch.where(sel >= 0, sel, nb), torch.ones_like(sel, dtype=torch.float64))
            often = times[:, :nb].repeat_interleave(bs, dim=1)
            often = often * ((t <= s["q_pos"][b, :, None]) & (t < s["kv_lens"][b]))
            for i in range(0, Q, 32):
                x = s["q"][b, i:i + 32].double().view(-1, H, G, D)[:, h]
                z = x @ k.t() * s["softmax_scale"] + torch.log(often[i:i + 32])[:, None, :]
                some = (often[i:i + 32].sum(-1) > 0)[:, None].expand(-1, G)
                one = torch.logsumexp(z, dim=-1)
                out[b, i:i + 32, h] = torch.where(some[..., None], torch.exp(z - one[..., None]) @ v, 0.0)
                lse[b, i:i + 32, h] = one
    return out.view(B, Q, H * G, D), lse.view(B, Q, H * G)
