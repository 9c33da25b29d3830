"""The attention side of a decode or speculative step that is timed on an MI355X: what happens between the fused q/k/v
linear and the o linear, the quantized paged cache that it fills and reads, and the verification of drafted tokens.

  norm_rope  norms of every query and key head with the position rotation (`ops.qk_norm_rope`).
  append     new keys and values quantized into the paged cache (`ops.kv_append`), and the pages read back
             (`ops.kv_gather`): only the touched pages, or the whole sequences as a prefill chunk's attention needs them.
  gather     a cached prefix read back as fp16 (`ops.kv_gather`).
  tree       attention of each sequence's drafted tokens, a tree or a chain, over the cache and over each other
             (`ops.kv_tree_attention`).
  verify     drafted tokens against the target's probabilities from given random numbers (`ops.verify_drafts`).

Caches hold 8- or 4-bit codes with one fp16 scale per (page of 16 tokens, kv head); heads are 128 wide.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
D = 128
PAGE = 16
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # one user's decode step: the heads of one token, as the fused q/k/v linear leaves them
        dict(name="norm_rope_t1", kind="norm_rope", tokens=1, q_heads=40, kv_heads=8, rotary=128, interleaved=False,
             dtype="bf16", out="fp16"),
        # the drafted tokens of a few users; rotation of half of each head, in neighbouring pairs
        dict(name="norm_rope_t77_pairs", kind="norm_rope", tokens=77, q_heads=32, kv_heads=2, rotary=64,
             interleaved=True, dtype="fp16", out="fp16"),
        # a prefill chunk
        dict(name="norm_rope_t8192", kind="norm_rope", tokens=8192, q_heads=40, kv_heads=8, rotary=128,
             interleaved=False, dtype="bf16", out="bf16"),
        # a decode batch: one token per sequence, somewhere inside a page that has to be kept in scale
        dict(name="append8_b16_n1", kind="append", batch=16, new=1, longest=4096, kv_heads=8, bits=8, dtype="fp16",
             readback="touched"),
        # prefill chunks of ragged lengths onto cached prefixes, the whole sequences read back for the chunk's attention
        dict(name="append4_b3_n2900", kind="append", batch=3, new=2900, longest=13001, kv_heads=8, bits=4, dtype="bf16",
             readback="all"),
        # one user's short cached prompt
        dict(name="gather8_b1_333", kind="gather", batch=1, longest=333, kv_heads=8, bits=8, dtype="fp16"),
        # long cached prefixes of a few users
        dict(name="gather8_b7_32k", kind="gather", batch=7, longest=32768, kv_heads=8, bits=8, dtype="bf16"),
        # one user, a short chain of drafts on a short context: latency
        dict(name="tree8_b1_n5_700", kind="tree", batch=1, nodes=5, tree=False, longest=700, q_heads=40, kv_heads=8,
             bits=8),
        # a batch of users with small draft trees, ragged lengths up to 4k
        dict(name="tree8_b16_n16_4k", kind="tree", batch=16, nodes=16, tree=True, longest=4096, q_heads=40, kv_heads=8,
             bits=8),
        # full trees over long contexts: the largest
        dict(name="tree4_b8_n64_32k", kind="tree", batch=8, nodes=64, tree=True, longest=32768, q_heads=40, kv_heads=8,
             bits=4),
        # one user's chain of sampled drafts, with the draft model's probabilities
        dict(name="verify_b1_n6_chain", kind="verify", batch=1, nodes=6, vocab=32003, tree=False),
        # a full batch of draft trees over a large vocabulary
        dict(name="verify_b64_n16_tree", kind="verify", batch=64, nodes=16, vocab=131072, tree=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm_rope", "append", "gather", "tree", "tree", "verify"])
    kv_heads = rng.choice([1, 2, 4, 8])
    if kind == "norm_rope":
        while True:
            tokens, q_heads = _log_int(rng, 1, 8192), kv_heads * rng.choice([1, 4, 5, 8, 16])
            if tokens * (q_heads + kv_heads) <= 8192 * 48:
                break
        return dict(kind=kind, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads,
                    rotary=rng.choice([32, 64, 96, 128, 128]), interleaved=rng.random() < 0.4,
                    dtype=rng.choice(["fp16", "bf16"]), out=rng.choice(["fp16", "fp16", "bf16"]))
    if kind == "append":
        while True:
            batch, new, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 4096), _log_int(rng, 1, 16384)
            if batch * (new + longest) * kv_heads <= 3 * 16000 * 8:
                break
        return dict(kind=kind, batch=batch, new=new, longest=longest, kv_heads=kv_heads, bits=rng.choice([4, 8]),
                    dtype=rng.choice(["fp16", "bf16"]), readback=rng.choice(["touched", "all"]))
    if kind == "gather":
        while True:
            batch, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
            if batch * longest * kv_heads <= 7 * 32768 * 8:
                break
        return dict(kind=kind, batch=batch, longest=longest, kv_heads=kv_heads, bits=rng.choice([4, 8]),
                    dtype=rng.choice(["fp16", "bf16"]))
    if kind == "tree":
        while True:
            batch, nodes, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
            q_heads = kv_heads * rng.choice([1, 4, 5, 8, 16])
            if batch * nodes * q_heads * longest <= 8 * 64 * 40 * 32768 and batch * longest * kv_heads <= 8 * 32768 * 8:
                break
        return dict(kind=kind, batch=batch, nodes=nodes, tree=rng.random() < 0.7, longest=longest, q_heads=q_heads,
                    kv_heads=kv_heads, bits=rng.choice([4, 8]))
    while True:
        batch, nodes, vocab = _log_int(rng, 1, 64), _log_int(rng, 1, 32), _log_int(rng, 1000, 200000)
        if batch * nodes * vocab <= 64 * 16 * 131072 and batch * vocab <= 64 * 131072 // 2:
            break
    return dict(kind=kind, batch=batch, nodes=nodes, vocab=vocab, tree=rng.random() < 0.5)


# ---- inputs ----------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ragged(most, count, g):
    """Users at different points: evenly spread lengths up to `most`, in a random order."""
    return [max(1, most * (i + 1) // count) for i in torch.randperm(count, generator=g, device="cuda").tolist()]


def _table(g, tokens, spare):
    """Distinct pages in a random order for sequences of `tokens` tokens, and the number of pages."""
    need = [-(-n // PAGE) for n in tokens]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(tokens), max(need)), dtype=torch.int32, device="cuda")
    for b, part in enumerate(torch.split(perm[:sum(need)], need)):
        table[b, :need[b]] = part
    return table, pages


def _codes(g, pages, kv_heads, bits):
    """Normal keys or values on the code grid (three sigmas to the largest code), and their pages' scales."""
    qmax = 127 if bits == 8 else 7
    c = torch.empty((pages, kv_heads, PAGE, D), dtype=torch.int8, device="cuda")
    for p in range(0, pages, 4096):
        part = torch.randn(c[p:p + 4096].shape, generator=g, device="cuda") * (qmax / 3.0)
        c[p:p + 4096] = part.round_().clamp_(-qmax, qmax).to(torch.int8)
    scale = ((0.5 + torch.rand((pages, kv_heads), generator=g, device="cuda")) * 3.0 / qmax).half()
    return (c if bits == 8 else ((c[..., 0::2] & 15) | (c[..., 1::2] << 4)).view(torch.uint8)), scale


def _tree(nodes, tree, batch, seed):
    """Parents (int32 [batch, nodes], -1 for the root) and ancestor masks (int64, bit j: node j is i or above it)."""
    r = np.random.default_rng(seed)
    parents = np.full((batch, nodes), -1, dtype=np.int32)
    masks = np.zeros((batch, nodes), dtype=np.uint64)
    for b in range(batch):
        for i in range(nodes):
            if i:
                parents[b, i] = r.integers(max(0, i - 8), i) if tree else i - 1
            masks[b, i] = (masks[b, parents[b, i]] if i else np.uint64(0)) | np.uint64(1) << np.uint64(i)
    return torch.from_numpy(parents).cuda(), torch.from_numpy(masks.view(np.int64)).cuda()


def _prepare_norm_rope(case, g, seed):
    T, Hq, Hkv, r = case["tokens"], case["q_heads"], case["kv_heads"], case["rotary"]
    width = (Hq + 2 * Hkv) * D
    qkv = _randn(g, T, width).to(DTYPES[case["dtype"]])
    # the rotation's table for every position of a 40k context, from 64-bit angles
    angle = torch.arange(40960, device="cuda").double()[:, None] \
        * THETA ** (-torch.arange(0, r, 2, device="cuda").double() / r)
    return {"q": qkv[:, :Hq * D].unflatten(1, (Hq, D)), "k": qkv[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D)),
            "q_weight": (1 + 0.2 * _randn(g, D)).to(DTYPES[case["dtype"]]),
            "k_weight": (1 + 0.2 * _randn(g, D)).to(DTYPES[case["dtype"]]),
            "cos_sin": torch.cat([angle.cos(), angle.sin()], dim=1).float(),
            "positions": torch.randint(0, 40960, (T,), generator=g, device="cuda")}


def _prepare_cache(case, g, lens, room):
    table, pages = _table(g, [n + room[b] for b, n in enumerate(lens)], 3)
    k, ks = _codes(g, pages, case["kv_heads"], case["bits"])
    v, vs = _codes(g, pages, case["kv_heads"], case["bits"])
    return {"cache": (k, v, ks, vs), "table": table, "lens": _int(lens)}


def _starts(counts):
    return _int(np.concatenate([[0], np.cumsum(counts)]).tolist())


def _prepare_append(case, g, seed):
    lens, new = _ragged(case["longest"], case["batch"], g), _ragged(case["new"], case["batch"], g)
    s = _prepare_cache(case, g, lens, new)
    first = [n // PAGE * PAGE if case["readback"] == "touched" else 0 for n in lens]
    back = [n + m - f for n, m, f in zip(lens, new, first)]
    rows, Hkv = sum(new), case["kv_heads"]
    kv = _randn(g, rows, 2 * Hkv * D).to(DTYPES[case["dtype"]])  # the k and v columns of the fused linear's output
    return s | {"k": kv[:, :Hkv * D].unflatten(1, (Hkv, D)), "v": kv[:, Hkv * D:].unflatten(1, (Hkv, D)),
                "row_start": _starts(new), "max_new": max(new), "lens_after": _int([n + m for n, m in zip(lens, new)]),
                "first": _int(first), "back_start": _starts(back), "back_rows": sum(back)}


def _prepare_gather(case, g, seed):
    lens = _ragged(case["longest"], case["batch"], g)
    return _prepare_cache(case, g, lens, [0] * len(lens)) | {"row_start": _starts(lens), "rows": sum(lens)}


def _prepare_tree(case, g, seed):
    B, N, Hq, Hkv = case["batch"], case["nodes"], case["q_heads"], case["kv_heads"]
    lens = _ragged(case["longest"], B, g)
    s = _prepare_cache(case, g, lens, [N] * B)
    x = _randn(g, B, N, (Hq + 2 * Hkv) * D).half()
    q, k, v = torch.split(x, [Hq * D, Hkv * D, Hkv * D], dim=2)
    parents, mask = _tree(N, case["tree"], B, seed)
    return s | {"q": q.unflatten(2, (Hq, D)), "k": k.unflatten(2, (Hkv, D)), "v": v.unflatten(2, (Hkv, D)),
                "mask": mask if case["tree"] else None, "longest": max(lens)}


def _prepare_verify(case, g, seed):
    B, N, V = case["batch"], case["nodes"], case["vocab"]
    logits = 3.0 * _randn(g, B, N, V)
    p = torch.softmax(logits, dim=2)
    u = torch.rand((B, N), generator=g, device="cuda")
    parents, mask = _tree(N, case["tree"], B, seed)
    tokens = torch.zeros((B, N), dtype=torch.int64, device="cuda")
    if case["tree"]:  # each node's candidates are the likeliest tokens after it, in order
        top = torch.topk(p, 8, dim=2).indices
        up = parents.long().clamp(min=0)
        rank = ((up[:, :, None] == up[:, None, :]).tril(-1)[:, :, 1:].sum(2)) % 8
        tokens[:] = top.flatten(1).gather(1, up * 8 + rank)
        return {"p": p, "q": None, "u": u, "tokens": tokens.int(), "parents": parents, "mask": mask}
    q = torch.softmax(0.9 * logits + 1.0 * _randn(g, B, N, V), dim=2)  # a draft model that is near the target
    if N > 1:  # token i is drawn from the draft's distribution after token i - 1
        draw = torch.multinomial(q[:, :N - 1].flatten(0, 1), 1, generator=g)
        tokens[:, 1:] = draw.view(B, N - 1)
    return {"p": p, "q": q, "u": u, "tokens": tokens.int(), "parents": None, "mask": None}


_PREPARE = {"norm_rope": _prepare_norm_rope, "append": _prepare_append, "gather": _prepare_gather,
            "tree": _prepare_tree, "verify": _prepare_verify}


def prepare(case, seed):
    return {"case": case} | _PREPARE[case["kind"]](case, _gen(seed), seed)


# ---- one pass --------------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


def _own(s):
    from trellis_serve_amd import ops
    case = s["case"]
    if case["kind"] == "norm_rope":
        return ops.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos_sin"], s["positions"], EPS,
                                interleaved=case["interleaved"], out_dtype=DTYPES[case["out"]])
    if case["kind"] == "append":
        ops.kv_append(s["k"], s["v"], *s["cache"], s["table"], s["lens"], case["bits"], row_start=s["row_start"],
                      max_new=s["max_new"])
        return ops.kv_gather(*s["cache"], s["table"], s["lens_after"], case["bits"], s["back_start"], s["back_rows"],
                             starts=s["first"])
    if case["kind"] == "gather":
        return ops.kv_gather(*s["cache"], s["table"], s["lens"], case["bits"], s["row_start"], s["rows"],
                             dtype=DTYPES[case["dtype"]])
    if case["kind"] == "tree":
        return ops.kv_tree_attention(s["q"], s["k"], s["v"], s["mask"], *s["cache"], s["table"], s["lens"],
                                     case["bits"])
    return ops.verify_drafts(s["p"], s["tokens"], s["u"], parents=s["parents"], draft_probs=s["q"])


def _plain_norm_rope(s):
    case = s["case"]
    r, out = case["rotary"], DTYPES[case["out"]]
    cs = s["cos_sin"][s["positions"]][:, None, :]
    c, sn = cs[..., :r // 2], cs[..., r // 2:]

    def one(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        if case["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            z = torch.stack([a * c - b * sn, b * c + a * sn], dim=-1).flatten(-2)
        else:
            a, b = y[..., :r // 2], y[..., r // 2:r]
            z = torch.cat([a * c - b * sn, b * c + a * sn], dim=-1)
        return torch.cat([z, y[..., r:]], dim=-1).to(out)

    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


def _unpack(codes, bits):
    """The codes as float32, last dimension 128."""
    if bits == 8:
        return codes.float()
    u = codes.int()
    return torch.stack([((u & 15) ^ 8) - 8, (u >> 4 ^ 8) - 8], dim=-1).flatten(-2).float()


def _pack(codes, bits):
    c = codes.to(torch.int8)
    return c if bits == 8 else ((c[..., 0::2] & 15) | (c[..., 1::2] << 4)).view(torch.uint8)


def _rows_of(row_start, rows):
    """The sequence of each row, and the row's place in it."""
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(row_start, row, right=True) - 1
    return b, row - row_start[b]


def _plain_gather(cache, table, bits, row_start, rows, starts, dtype):
    k, v, ks, vs = cache
    b, at = _rows_of(row_start, rows)
    t = at + starts[b]
    page, off = table[b, t // PAGE].long(), (t % PAGE).long()
    return tuple((_unpack(c[page, :, off], bits) * sc[page].float()[..., None]).to(dtype) for c, sc in ((k, ks), (v, vs)))


def _page_scale(most, qmax):
    """The smallest float16 that is not below most / qmax."""
    h = (most / qmax).half()
    short = h.double() * qmax < most.double()
    return (h.view(torch.int16) + short.to(torch.int16)).view(torch.float16).float()


def _plain_append(s):
    bits, (kc, vc, ks, vs) = s["case"]["bits"], s["cache"]
    qmax = 127.0 if bits == 8 else 7.0
    table, lens = s["table"], s["lens"]
    b, at = _rows_of(s["row_start"], s["k"].shape[0])
    t = at + lens[b]
    page, off = table[b, t // PAGE].long(), (t % PAGE).long()
    tail = table.gather(1, (lens // PAGE)[:, None].long())[:, 0].long()  # the page that each sequence's first row enters
    kept = torch.arange(PAGE, device="cuda")[None, :] < (lens % PAGE)[:, None]  # its slots that hold older tokens

    def write(x, codes, scale):
        x = x.float()
        new = _page_scale(torch.zeros(scale.shape, device="cuda").index_reduce(0, page, x.abs().amax(-1), "amax"), qmax)
        old = scale[tail].float() * (lens % PAGE > 0)[:, None]
        new[tail] = torch.maximum(new[tail], old)
        moved = torch.round(_unpack(codes[tail], bits) * old[..., None, None] / new[tail][..., None, None])
        codes[tail] = torch.where(kept[:, None, :, None], _pack(moved, bits), codes[tail])
        code = torch.round(x / new[page][..., None]).clamp(-qmax, qmax)
        codes[page, :, off] = _pack(code, bits)
        scale[page] = new[page].half()

    write(s["k"], kc, ks)
    write(s["v"], vc, vs)
    return _plain_gather(s["cache"], table, bits, s["back_start"], s["back_rows"], s["first"], torch.float16)


def _plain_tree(s):
    case, (kc, vc, ks, vs) = s["case"], s["cache"]
    q, table, lens, longest = s["q"].float(), s["table"], s["lens"], s["longest"]
    B, N, Hq, _ = q.shape
    Hkv = kc.shape[1]
    pages = table[:, :-(-longest // PAGE)].long()

    def cached(codes, scale):  # [B, Hkv, tokens, D]
        x = _unpack(codes[pages], case["bits"]) * scale[pages].float()[..., None, None]
        return x.transpose(1, 2).flatten(2, 3)

    k = torch.cat([cached(kc, ks), s["k"].float().transpose(1, 2)], dim=2)
    v = torch.cat([cached(vc, vs), s["v"].float().transpose(1, 2)], dim=2)
    tokens = k.shape[2] - N
    if s["mask"] is None:
        seen = torch.ones((N, N), device="cuda").tril().bool().expand(B, N, N)
    else:
        seen = (s["mask"][:, :, None] >> torch.arange(N, device="cuda") & 1).bool()
    live = (torch.arange(tokens, device="cuda") < lens[:, None])[:, None, :].expand(B, N, tokens)
    seen = torch.cat([live, seen], dim=2)[:, None, :, None, :]  # [B, 1, N, 1, keys]
    rows = q.view(B, N, Hkv, Hq // Hkv, D).transpose(1, 2).flatten(2, 3)
    logits = torch.matmul(rows, k.transpose(2, 3).contiguous()).unflatten(2, (N, Hq // Hkv)) * D ** -0.5
    logits = logits.masked_fill_(~seen, -math.inf)
    p = torch.exp(logits.sub_(logits.amax(-1, keepdim=True)))
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (N, Hq // Hkv)) / p.sum(-1, keepdim=True)
    return o.transpose(1, 2).flatten(2, 3).half()


def _next_token(w, fallback, u):
    """The first index whose running sum passes u of the total, in 64 bits."""
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, fallback)
    run = torch.cumsum(w, dim=-1)
    return (run <= u[:, None] * run[:, -1:]).sum(-1)


def _plain_verify(s):
    p, q, u, tok = s["p"], s["q"], s["u"].double(), s["tokens"].long()
    B, N, V = p.shape
    node, seq = torch.arange(N, device="cuda"), torch.arange(B, device="cuda")
    if q is not None:  # a chain: node i was drawn from q after node i - 1
        pt = p[:, :N - 1].gather(2, tok[:, 1:, None])[..., 0].double()
        qt = q[:, :N - 1].gather(2, tok[:, 1:, None])[..., 0].double()
        taken = ((pt > 0) & (u[:, 1:] * qt < pt)).long().cumprod(1).sum(1)
        on_path = node <= taken[:, None]
        last = p[seq, taken].double()
        rest = (last - q[seq, taken].double()).clamp(min=0)
        w = torch.where((taken < N - 1)[:, None], rest, last)
    else:  # a tree of candidates: brothers in order, each refused token is struck from the target's row
        up = s["parents"].long().clamp(min=0)
        pt = p.flatten(1).gather(1, up * V + tok).double()
        brothers = (up[:, :, None] == up[:, None, :]).tril(-1) & (node > 0)  # [B, i, j]: j comes before i
        brothers[:, 0] = False
        pt = torch.where((brothers & (tok[:, :, None] == tok[:, None, :])).any(2), 0.0, pt)
        left = 1 - (brothers * pt[:, None, :]).sum(2)
        fits = (pt > 0) & (u * left < pt)
        chosen = fits & ~(brothers & fits[:, None, :]).any(2)
        chosen[:, 0] = True
        above = (s["mask"][:, :, None] >> node & 1).bool()
        on_path = (~above | chosen[:, None, :]).all(2)
        at = (on_path * node).amax(1)
        last = p[seq, at].double()
        struck = torch.where((up == at[:, None]) & (node > 0), tok, V)
        w = torch.cat([last, last[:, :1]], dim=1).scatter(1, struck, 0.0)[:, :V]
    nxt = _next_token(w, last, u[:, 0])
    count = on_path.sum(1)
    nodes = torch.where(on_path, node, N).sort(1).values
    nodes = torch.where(nodes < N, nodes, -1)
    out = torch.where(node < count[:, None] - 1, tok.gather(1, nodes.roll(-1, 1).clamp(min=0)), -1)
    out = torch.where(node == count[:, None] - 1, nxt[:, None], out)
    return nodes.int(), count.int(), out.int()


_PLAIN = {"norm_rope": _plain_norm_rope, "append": _plain_append, "tree": _plain_tree, "verify": _plain_verify,
          "gather": lambda s: _plain_gather(s["cache"], s["table"], s["case"]["bits"], s["row_start"], s["rows"],
                                            torch.zeros_like(s["lens"]), DTYPES[s["case"]["dtype"]])}


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    kind, B = case["kind"], case.get("batch", 1)
    spread = lambda most: sum(max(1, most * (i + 1) // B) for i in range(B))  # noqa: E731
    if kind == "norm_rope":
        values = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * D
        return {"bytes": 4 * values + case["tokens"] * (4 * case["rotary"] + 8) + 4 * D, "flops": 8 * values}
    if kind == "verify":
        rows = B * (1 if case["tree"] else 2)
        return {"bytes": 4 * rows * case["vocab"] + 32 * B * case["nodes"], "flops": 2 * rows * case["vocab"]}
    per_token = 2 * case["kv_heads"] * (D * case["bits"] // 8)  # codes of one token, keys and values
    tokens = spread(case["longest"])
    if kind == "gather":
        return {"bytes": tokens * (per_token + 4 * case["kv_heads"] * D), "flops": 2 * tokens * case["kv_heads"] * D}
    if kind == "append":
        new = spread(case["new"])
        back = new + (B * PAGE // 2 if case["readback"] == "touched" else tokens)
        wide = 4 * case["kv_heads"] * D
        return {"bytes": new * (wide + per_token) + back * (per_token + wide),
                "flops": 4 * (new + back) * case["kv_heads"] * D}
    N, Hq = case["nodes"], case["q_heads"]
    seen = (N + 1) / 2 if not case["tree"] else math.log2(N + 1)
    return {"bytes": tokens * per_token + B * N * (4 * Hq + 4 * case["kv_heads"]) * D,
            "flops": 4 * N * Hq * D * (tokens + B * seen)}


# ---- the same outputs in 64 bits -------------------------------------------------------------------------------

def _exact_values(codes, scale, pages, bits):
    """float64 [tokens, Hkv, D] of the pages in `pages`."""
    c = codes[pages.long()].cpu().numpy()
    if bits == 4:
        low, high = (c & 15).astype(np.int16), (c >> 4).astype(np.int16)
        c = np.empty(c.shape[:-1] + (D,), dtype=np.int16)
        c[..., 0::2], c[..., 1::2] = low - 16 * (low > 7), high - 16 * (high > 7)
    c = c.astype(np.float64) * scale[pages.long()].cpu().numpy().astype(np.float64)[..., None, None]
    return c.transpose(0, 2, 1, 3).reshape(-1, c.shape[1], D)


def _exact_norm_rope(case, s):
    r = case["rotary"]
    turn = torch.zeros((case["tokens"], D // 2), dtype=torch.complex128, device="cuda") + 1  # one factor a pair
    cs = s["cos_sin"].double()[s["positions"]]
    turn[:, :r // 2] = torch.complex(cs[:, :r // 2], cs[:, r // 2:])
    i = torch.arange(D // 2, device="cuda")
    if case["interleaved"]:
        first, second = 2 * i, 2 * i + 1
    else:  # the pairs of the rotated part, then the rest two by two
        first = torch.where(i < r // 2, i, 2 * i)
        second = torch.where(i < r // 2, i + r // 2, 2 * i + 1)

    def one(x, w):
        x = x.double()
        y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
        out = torch.empty_like(y)
        out[..., first], out[..., second] = z.real, z.imag
        return out

    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


def _exact_append(case, s):
    bits, (kc, vc, ks, vs) = case["bits"], s["cache"]
    qmax = 127 if bits == 8 else 7
    outs = []
    for x, codes, scale in ((s["k"], kc, ks), (s["v"], vc, vs)):
        rows = []
        x = x.double().cpu().numpy()
        for b, (n, after) in enumerate(zip(s["lens"].tolist(), s["lens_after"].tolist())):
            first, r0 = n // PAGE * PAGE, int(s["row_start"][b])
            npages = -(-after // PAGE)
            pages = s["table"][b, :npages]
            old = _exact_values(codes, scale, pages[:-(-n // PAGE)], bits)[:n]
            work = np.zeros((npages * PAGE - first,) + x.shape[1:])
            work[n - first:after - first] = x[r0:r0 + after - n]
            by_page = work.reshape(-1, PAGE, *x.shape[1:])
            need = np.abs(by_page).max(axis=(1, 3)) / qmax
            sc = need.astype(np.float16)
            sc = np.where(sc.astype(np.float64) < need, np.nextafter(sc, np.float16(np.inf)), sc).astype(np.float64)
            if n > first:
                sc[0] = np.maximum(sc[0], scale[int(pages[n // PAGE])].double().cpu().numpy())
                by_page[0, :n - first] = old[first:]
            value = np.clip(np.rint(by_page / sc[:, None, :, None]), -qmax, qmax) * sc[:, None, :, None]
            value = np.concatenate([old[:first], value.reshape(-1, *x.shape[1:])])[:after]
            rows.append(value[int(s["first"][b]):])
        outs.append(torch.from_numpy(np.concatenate(rows)))
    return tuple(outs)


def _exact_gather(case, s):
    return tuple(torch.from_numpy(np.concatenate([
        _exact_values(codes, scale, s["table"][b, :-(-n // PAGE)], case["bits"])[:n]
        for b, n in enumerate(s["lens"].tolist())])) for codes, scale in ((s["cache"][0], s["cache"][2]),
                                                                          (s["cache"][1], s["cache"][3])))


def _exact_tree(case, s):
    B, N, Hq, _ = s["q"].shape
    G = Hq // case["kv_heads"]
    k, v, ks, vs = s["cache"]
    out = torch.empty((B, N, Hq, D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // PAGE)].long()

        def values(codes, scale, fresh, h):
            c = codes[pages, h]
            if case["bits"] == 4:
                wide = torch.empty(c.shape[:-1] + (D,), dtype=torch.float64, device="cuda")
                wide[..., 0::2], wide[..., 1::2] = (c % 16).double(), (c // 16).double()
                c = wide - 16 * (wide >= 8)
            c = c.double() * scale[pages, h].double()[:, None, None]
            return torch.cat([c.reshape(-1, D)[:n], fresh[b, :, h].double()])

        seen = np.ones((N, n + N), dtype=bool)
        seen[:, n:] = [[j <= i if s["mask"] is None else s["mask_rows"][b][i] >> j & 1 for j in range(N)]
                       for i in range(N)]
        seen = torch.from_numpy(seen).cuda()
        for h in range(case["kv_heads"]):
            kk, vv = values(k, ks, s["k"], h), values(v, vs, s["v"], h)
            rows = s["q"][b, :, h * G:(h + 1) * G].double().reshape(N * G, D)
            a = (rows @ kk.T / math.sqrt(D)).reshape(N, G, -1)
            a = torch.softmax(a.masked_fill(~seen[:, None], -math.inf), dim=-1)
            out[b, :, h * G:(h + 1) * G] = (a.reshape(N * G, -1) @ vv).reshape(N, G, D)
    return out


def _exact_verify(case, s):
    B, N, V = s["p"].shape
    nodes, out = np.full((B, N), -1, dtype=np.int32), np.full((B, N), -1, dtype=np.int32)
    counts = np.zeros(B, dtype=np.int32)
    tok, u = s["tokens"].tolist(), s["u"].double().tolist()
    for b in range(B):
        parents = list(range(-1, N - 1)) if s["parents"] is None else s["parents"][b].tolist()
        path, left, refused = [0], 1.0, []
        for i in range(1, N):
            if parents[i] != path[-1]:
                continue
            pt = 0.0 if tok[b][i] in refused else float(s["p"][b, path[-1], tok[b][i]])
            bar = u[b][i] * (left if s["q"] is None else float(s["q"][b, path[-1], tok[b][i]]))
            if pt > 0 and bar < pt:
                path, left, refused = path + [i], 1.0, []
            else:
                left, refused = left - pt, refused + [tok[b][i]]
        p = s["p"][b, path[-1]].double().cpu().numpy()
        w = p.copy()
        if refused and s["q"] is None:
            w[refused] = 0.0
        elif refused:
            w = np.maximum(p - s["q"][b, path[-1]].double().cpu().numpy(), 0.0)
        w = w if w.sum() > 0 else p
        total = np.cumsum(w)
        counts[b], nodes[b, :len(path)] = len(path), path
        out[b, :len(path)] = [tok[b][i] for i in path[1:]] + [int(np.searchsorted(total, u[b][0] * total[-1], "right"))]
    return torch.from_numpy(nodes), torch.from_numpy(counts), torch.from_numpy(out)


_EXACT = {"norm_rope": _exact_norm_rope, "append": _exact_append, "gather": _exact_gather, "tree": _exact_tree,
          "verify": _exact_verify}


def exact(case, seed):
    s = prepare(case, seed)
    if s.get("mask") is not None:
        s["mask_rows"] = (s["mask"].cpu().numpy().view(np.uint64)).tolist()
    return _EXACT[case["kind"]](case, s)
