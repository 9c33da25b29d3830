"""The operators around the attention and at the ends of a serving step that are timed on an MI355X.

  plan     a step's pages, rows, positions and slots from the requests' lengths (`ops.kv_step_plan`).
  norm     the norm after a block, its gate and scale, the residual, and the norm before the next block (`ops.add_norm`).
  bounds   the largest and smallest key codes of a page's tokens (`ops.kv_page_bounds`).
  sparse   the pages that each query's bounds make worth reading, and attention over them (`ops.kv_select_pages`,
           `ops.kv_sparse_attention`).
  sample   tokens from logits by temperature, top-k, top-p and min-p from given random numbers (`ops.sample_tokens`), and the
           distribution that they are drawn from.

Caches hold 8- or 4-bit codes with one fp16 scale per (page of 16 tokens, kv head); heads are 128 wide.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
D = 128
PAGE = 16
EPS = 1e-6


def listed():
    return [
        # a few users' decode step: one token each, a page now and then
        dict(name="plan_b8_n1", kind="plan", batch=8, new=1, longest=4096, finished=False),
        # a busy server's step: prompt chunks, decode tokens, sequences that ended
        dict(name="plan_b1024_n127", kind="plan", batch=1024, new=127, longest=8192, finished=True),
        # one user's decode step between two blocks
        dict(name="norm_t1_5120", kind="norm", tokens=1, dim=5120, dtype="bf16", residual="bf16", post=False, gate="none",
             sigmoid=False, scale=1.0, unit_offset=False),
        # a prefill chunk with norms on both sides of the block and a gate for each channel
        dict(name="norm_t8192_5120", kind="norm", tokens=8192, dim=5120, dtype="bf16", residual="bf16", post=True,
             gate="channel", sigmoid=False, scale=0.5, unit_offset=True),
        # a decode batch: the page that each sequence's token went into
        dict(name="bounds8_b16_n1", kind="bounds", batch=16, new=1, longest=4096, kv_heads=8, bits=8),
        # the whole prompts of a few users
        dict(name="bounds4_b7_32k", kind="bounds", batch=7, new=32768, longest=32768, kv_heads=8, bits=4),
        # one user's decode step on a long context
        dict(name="sparse8_b1_32k", kind="sparse", batch=1, rows=1, longest=32768, q_heads=40, kv_heads=8, bits=8,
             top=64),
        # a batch of users at different lengths
        dict(name="sparse8_b16_24k", kind="sparse", batch=16, rows=1, longest=24001, q_heads=32, kv_heads=8, bits=8,
             top=128),
        # a few rows for each of some users on the longest contexts
        dict(name="sparse4_b8_n4_128k", kind="sparse", batch=8, rows=4, longest=131072, q_heads=40, kv_heads=8, bits=4,
             top=256),
        # one user's next token
        dict(name="sample_b1_32003", kind="sample", batch=1, vocab=32003, dtype="fp32", top_k=0, top_p=0.9, min_p=0.0,
             mixed=False, probs=False),
        # drafted tokens with the distribution that their verification needs
        dict(name="sample_b48_100352_probs", kind="sample", batch=48, vocab=100352, dtype="fp16", top_k=0, top_p=0.95,
             min_p=0.0, mixed=False, probs=True),
        # a full batch of users with settings of their own over a large vocabulary
        dict(name="sample_b64_131072_mixed", kind="sample", batch=64, vocab=131072, dtype="bf16", top_k=40, top_p=0.9,
             min_p=0.05, mixed=True, probs=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "norm", "bounds", "sparse", "sparse", "sample", "sample"])
    if kind == "plan":
        while True:
            batch, new = _log_int(rng, 1, 1024), _log_int(rng, 1, 4096)
            if batch * new <= 1024 * 127:
                break
        return dict(kind=kind, batch=batch, new=new, longest=_log_int(rng, 1, 8192), finished=rng.random() < 0.5)
    if kind == "norm":
        while True:
            tokens = _log_int(rng, 1, 8192)
            dim = _log_int(rng, 64, 16384)
            if rng.random() < 0.8:
                dim = dim // 8 * 8
            if tokens * dim <= 8192 * 5120 // 2:
                break
        dtype = rng.choice(["fp16", "bf16"])
        return dict(kind=kind, tokens=tokens, dim=dim, dtype=dtype, residual=rng.choice([dtype, dtype, "fp32"]),
                    post=rng.random() < 0.5, gate=rng.choice(["none", "channel", "token", "full"]),
                    sigmoid=rng.random() < 0.5, scale=rng.choice([1.0, 0.5, 0.22]), unit_offset=rng.random() < 0.4)
    kv_heads, bits = rng.choice([1, 2, 4, 8]), rng.choice([4, 8])
    if kind == "bounds":
        while True:
            batch, new, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 32768), _log_int(rng, 1, 32768)
            if batch * longest * kv_heads * bits <= 7 * 32768 * 8 * 4:
                break
        return dict(kind=kind, batch=batch, new=min(new, longest), longest=longest, kv_heads=kv_heads, bits=bits)
    if kind == "sparse":
        while True:
            batch, rows, longest = _log_int(rng, 1, 64), _log_int(rng, 1, 8), _log_int(rng, 1, 131072)
            top = _log_int(rng, 4, 512)
            if batch * longest * kv_heads * bits <= 8 * 131072 * 8 * 4 and batch * rows <= 32 \
                    and batch * rows * top * kv_heads <= 32 * 256 * 8 and rows * batch * longest <= 4 * 8 * 131072 // 2:
                break
        return dict(kind=kind, batch=batch, rows=min(rows, longest), longest=longest,
                    q_heads=kv_heads * rng.choice([1, 4, 5, 8, 16]), kv_heads=kv_heads, bits=bits, top=top)
    while True:
        batch, vocab = _log_int(rng, 1, 256), _log_int(rng, 1000, 262144)
        if batch * vocab <= 48 * 100352 // 2:
            break
    return dict(kind=kind, batch=batch, vocab=vocab, dtype=rng.choice(["fp16", "bf16", "fp32"]),
                top_k=rng.choice([0, 0, 1, _log_int(rng, 2, 2000)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), mixed=rng.random() < 0.4, probs=rng.random() < 0.4)


# ---- inputs ----------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ragged(most, count, g):
    """Users at different points: evenly spread lengths up to `most`, in a random order."""
    return [max(1, most * (i + 1) // count) for i in torch.randperm(count, generator=g, device="cuda").tolist()]


def _table(g, tokens, spare, width=0):
    """Distinct pages in a random order for sequences of `tokens` tokens, the number of pages, and the unused ones."""
    need = [-(-n // PAGE) for n in tokens]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(tokens), max(width, *need)), dtype=torch.int32, device="cuda")
    for b, part in enumerate(torch.split(perm[:sum(need)], need)):
        table[b, :need[b]] = part
    return table, pages, perm[sum(need):]


def _grown(case):
    """The tokens that a step's sequences get, in order of their size; half of them none where some have ended."""
    sizes = [max(1, case["new"] * (i + 1) // case["batch"]) for i in range(case["batch"])]
    return [0 if case["finished"] and i % 8 < 4 else n for i, n in enumerate(sizes)]


def _prepare_plan(case, g, seed):
    B = case["batch"]
    lens = _ragged(case["longest"], B, g)
    order = torch.randperm(B, generator=g, device="cuda").tolist()
    new = _grown(case)
    new = [new[i] for i in order]
    if case["finished"]:  # one in eight ends, one in eight takes its last tokens back, a quarter waits
        new = [{0: -lens[b], 1: -min(lens[b], 3)}.get(order[b] % 8, new[b]) for b in range(B)]
    rows = sum(max(n, 0) for n in new)
    width = -(-(case["longest"] + case["new"]) // PAGE) + 4
    table, pages, unused = _table(g, lens, sum(-(-max(n, 0) // PAGE) for n in new) + B, width)
    ring = torch.zeros(pages, dtype=torch.int32, device="cuda")
    head = pages - len(unused) // 2  # the ring's live part passes its end
    at = (head + torch.arange(len(unused), device="cuda")) % pages
    ring[at] = unused
    return {"table": table, "lens": _int(lens), "new": _int(new), "ring": ring, "rows": rows,
            "ring_state": _int([head % pages, len(unused)]), "ring_after": _int([0, 0])}


def _prepare_norm(case, g, seed):
    T, n, dtype = case["tokens"], case["dim"], DTYPES[case["dtype"]]
    shift = 0.0 if case["unit_offset"] else 1.0
    shape = {"none": None, "channel": (n,), "token": (T, 1), "full": (T, n)}[case["gate"]]
    return {"x": _randn(g, T, n).to(dtype), "residual": (3 * _randn(g, T, n)).to(DTYPES[case["residual"]]),
            "weight": (shift + 0.2 * _randn(g, n)).to(dtype),
            "post": (shift + 0.2 * _randn(g, n)).to(dtype) if case["post"] else None,
            "gate": None if shape is None else _randn(g, *shape).to(dtype)}


def _key_codes(g, pages, kv_heads, bits):
    """Keys on the code grid that differ from page to page (three sigmas to the largest code), and their scales."""
    qmax = 127 if bits == 8 else 7
    c = torch.empty((pages, kv_heads, PAGE, D), dtype=torch.int8, device="cuda")
    for p in range(0, pages, 4096):
        n = min(4096, pages - p)
        part = 0.8 * _randn(g, n, kv_heads, PAGE, D) + 0.6 * _randn(g, n, kv_heads, 1, D)
        c[p:p + n] = part.mul_(qmax / 3.0).round_().clamp_(-qmax, qmax).to(torch.int8)
    scale = ((0.5 + _rand(g, pages, kv_heads)) * 3.0 / qmax).half()
    return c, scale


def _packed(c, bits):
    return c if bits == 8 else ((c[..., 0::2] & 15) | (c[..., 1::2] << 4)).view(torch.uint8)


def _code_bounds(codes, table, lens):
    """int8 [pages, kv heads, 2, 128]: each page's largest and smallest code of every channel, over the tokens below the
    sequence's length."""
    out = torch.empty((codes.shape[0], codes.shape[1], 2, D), dtype=torch.int8, device="cuda")
    for p in range(0, codes.shape[0], 4096):
        out[p:p + 4096, :, 0], out[p:p + 4096, :, 1] = codes[p:p + 4096].amax(2), codes[p:p + 4096].amin(2)
    for b, n in enumerate(lens):
        if n % PAGE:
            page = int(table[b, n // PAGE])
            live = codes[page, :, :n % PAGE]
            out[page, :, 0], out[page, :, 1] = live.amax(1), live.amin(1)
    return out


def _prepare_bounds(case, g, seed):
    B = case["batch"]
    lens = _ragged(case["longest"], B, g)
    table, pages, _ = _table(g, lens, 3)
    codes, _ = _key_codes(g, pages, case["kv_heads"], case["bits"])
    k = _packed(codes, case["bits"])
    return {"k": k, "table": table, "lens": _int(lens), "first": _int([max(0, n - case["new"]) for n in lens]),
            "bounds": torch.zeros((pages, case["kv_heads"], 2, k.shape[-1]), dtype=k.dtype, device="cuda"),
            "max_new": case["new"]}


def _prepare_sparse(case, g, seed):
    B, n, Hq, Hkv, bits = case["batch"], case["rows"], case["q_heads"], case["kv_heads"], case["bits"]
    lens = [max(n, m) for m in _ragged(case["longest"], B, g)]
    table, pages, _ = _table(g, lens, 3)
    codes, ks = _key_codes(g, pages, Hkv, bits)
    bounds = _packed(_code_bounds(codes, table, lens), bits)
    k = _packed(codes, bits)
    codes, vs = _key_codes(g, pages, Hkv, bits)
    seen = [m - n + 1 + i for m in lens for i in range(n)]
    return {"q": _randn(g, B * n, Hq, D).half(), "cache": (k, _packed(codes, bits), ks, vs), "bounds": bounds,
            "table": table, "seen": _int(seen), "longest": max(lens),
            "row_seq": None if n == 1 else _int([b for b in range(B) for _ in range(n)])}


def _prepare_sample(case, g, seed):
    B, V = case["batch"], case["vocab"]
    logits = 2.5 * _randn(g, B, V)
    for b in range(B):  # a few likely tokens
        at = torch.randint(0, V, (8,), generator=g, device="cuda")
        logits[b, at] += 4 + 6 * _rand(g, 8)
    s = {"logits": logits.to(DTYPES[case["dtype"]]), "u": _rand(g, B)}
    if not case["mixed"]:
        return s | {"temperature": 0.8, "top_k": case["top_k"], "top_p": case["top_p"], "min_p": case["min_p"]}
    on = _rand(g, 4, B)
    t = 0.3 + 1.2 * _rand(g, B)
    t[on[0] < 0.1] = 0.0  # greedy
    k = (case["top_k"] * (0.5 + _rand(g, B))).ceil().int()
    k[on[1] < 0.4] = 0
    p = 1 - (1 - case["top_p"]) * (0.5 + _rand(g, B))
    p[on[2] < 0.3] = 1.0
    m = case["min_p"] * (0.5 + _rand(g, B))
    m[on[3] < 0.5] = 0.0
    return s | {"temperature": t, "top_k": k, "top_p": p, "min_p": m}


_PREPARE = {"plan": _prepare_plan, "norm": _prepare_norm, "bounds": _prepare_bounds, "sparse": _prepare_sparse,
            "sample": _prepare_sample}


def prepare(case, seed):
    return {"case": case} | _PREPARE[case["kind"]](case, _gen(seed), seed)


# ---- one pass --------------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


def _own(s):
    from trellis_serve_amd import ops
    case = s["case"]
    if case["kind"] == "plan":
        plan = ops.kv_step_plan(s["table"], s["lens"], s["new"], s["ring"], s["ring_state"], s["rows"],
                                state_out=s["ring_after"])
        return (*plan, s["table"], s["ring"], s["ring_after"])
    if case["kind"] == "norm":
        return ops.add_norm(s["x"], s["residual"], s["weight"], EPS, post_weight=s["post"], gate=s["gate"],
                            gate_sigmoid=case["sigmoid"], scale=case["scale"], unit_offset=case["unit_offset"])
    if case["kind"] == "bounds":
        ops.kv_page_bounds(s["k"], s["table"], s["lens"], case["bits"], s["bounds"], first=s["first"],
                           max_new=s["max_new"])
        return s["bounds"]
    if case["kind"] == "sparse":
        pages = ops.kv_select_pages(s["q"], s["bounds"], s["cache"][2], s["table"], s["seen"], case["bits"], case["top"],
                                    row_seq=s["row_seq"])
        out = ops.kv_sparse_attention(s["q"], *s["cache"], s["table"], s["seen"], case["bits"], pages,
                                      row_seq=s["row_seq"])
        return pages, out
    return ops.sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                             return_probs=case["probs"])


def _plain_plan(s):
    table, ring, rows = s["table"], s["ring"], s["rows"]
    B, W = table.shape
    P = ring.numel()
    head, count = s["ring_state"][0].long(), s["ring_state"][1].long()
    length, new = s["lens"].long().clamp(0, W * PAGE), s["new"].long()
    grow, drop = new.clamp(min=0), torch.minimum((-new).clamp(min=0), length)
    end = grow.cumsum(0)
    start = end - grow
    have = (length + PAGE - 1) // PAGE
    fits = (length + grow <= W * PAGE) & (end <= rows)
    need = torch.where(fits, (length + grow + PAGE - 1) // PAGE - have, 0)
    sums = need.cumsum(0)
    ok = fits & ((need == 0) | (sums <= count))
    counts = torch.where(ok, grow, 0)
    after = length + counts - drop
    # pages taken: entry have + j of a sequence's table is the ring's next
    col = torch.arange(W, device="cuda")
    turn = (sums - need)[:, None] + col - have[:, None]
    taken = ok[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    table.copy_(torch.where(taken, ring[(head + turn) % P], table))
    popped = torch.where(ok, need, 0).sum()
    # pages given back, at the ring's end
    keep = (after + PAGE - 1) // PAGE
    give = torch.where(drop > 0, have - keep, 0)
    sums = give.cumsum(0)
    back = (drop > 0)[:, None] & (col >= keep[:, None]) & (col < have[:, None])
    to = (head + count + (sums - give)[:, None] + col - keep[:, None]) % P
    spill = torch.cat([ring, ring[:1]])
    spill[torch.where(back, to, P)] = table
    ring.copy_(torch.where(torch.zeros(P + 1, device="cuda").index_fill_(0, torch.where(back, to, P).flatten(), 1.0)[:P] > 0,
                           spill[:P], ring))
    s["ring_after"].copy_(torch.stack([(head + popped) % P, count - popped + give.sum()]))
    # the rows
    row = torch.arange(rows, device="cuda")
    b = torch.searchsorted(end, row, right=True).clamp(max=B - 1)
    live = ok[b] & (row < end[b]) & (row >= start[b])
    pos = torch.where(live, length[b] + row - start[b], -1)
    page = table[b, pos.clamp(min=0) // PAGE].long()
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), end]).clamp(max=rows)
    return (starts.int(), counts.int(), after.int(), pos.int(), (pos + 1).int(), torch.where(live, b, -1).int(),
            torch.where(live, page * PAGE + pos % PAGE, -1), table, ring, s["ring_after"])


def _plain_norm(s):
    case = s["case"]
    shift = 1.0 if case["unit_offset"] else 0.0

    def norm(x, w):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (w.float() + shift)

    u = s["x"].float()
    if s["post"] is not None:
        u = norm(u, s["post"])
    if s["gate"] is not None:
        gate = s["gate"].float()
        u = u * (1 / (1 + torch.exp(-gate)) if case["sigmoid"] else gate)
    h = s["residual"].float() + case["scale"] * u
    return norm(h, s["weight"]).to(s["x"].dtype), h.to(s["residual"].dtype)


def _unpack(codes, bits):
    """The codes as float32, last dimension 128."""
    if bits == 8:
        return codes.float()
    u = codes.int()
    return torch.stack([((u & 15) ^ 8) - 8, (u >> 4 ^ 8) - 8], dim=-1).flatten(-2).float()


def _plain_bounds(s):
    bits, table, lens, first = s["case"]["bits"], s["table"], s["lens"], s["first"]
    W = table.shape[1]
    col = torch.arange(W, device="cuda")
    touched = (col >= (first // PAGE)[:, None]) & (col < ((lens + PAGE - 1) // PAGE)[:, None])
    b, lp = torch.nonzero(touched, as_tuple=True)
    for i in range(0, b.numel(), 4096):
        bi, li = b[i:i + 4096], lp[i:i + 4096]
        page = table[bi, li].long()
        c = _unpack(s["k"][page], bits)
        live = ((li * PAGE)[:, None] + torch.arange(PAGE, device="cuda") < lens[bi][:, None])[:, None, :, None]
        both = torch.stack([c.masked_fill(~live, -math.inf).amax(2), c.masked_fill(~live, math.inf).amin(2)], dim=2)
        s["bounds"][page] = _packed(both.to(torch.int8), bits)
    return s["bounds"]


FIRST, LAST = 1, 2  # pages of a sequence's beginning and end that every query reads


def _plain_sparse(s):
    case, (kc, vc, ks, vs) = s["case"], s["cache"]
    bits, top, table, seen = case["bits"], case["top"], s["table"], s["seen"].long()
    q = s["q"].float()
    R, Hq, _ = q.shape
    Hkv, W = kc.shape[1], -(-s["longest"] // PAGE)
    G = Hq // Hkv
    seq = torch.arange(R, device="cuda") if s["row_seq"] is None else s["row_seq"].long()
    a = q.abs().amax(-1, keepdim=True)
    q8 = torch.where(a > 0, torch.round(q * 127 / a), 0.0).view(R, Hkv, G, D)
    both = torch.cat([q8.clamp(min=0), q8.clamp(max=0)], dim=-1)  # against the largest codes, and the smallest
    a = a.view(R, Hkv, G)
    score = torch.empty((R, Hkv, W), device="cuda")
    for r in range(R):
        pages = table[seq[r], :W].long()
        edge = _unpack(s["bounds"][pages], bits).flatten(2).permute(1, 2, 0).contiguous()  # [Hkv, 2 D, W]
        total = torch.matmul(both[r], edge)  # whole numbers below 2^24
        score[r] = (total * (a[r][:, :, None] * ks[pages].float().t()[:, None, :])).amax(1)
    pages_of = (seen + PAGE - 1) // PAGE
    col = torch.arange(W, device="cuda")
    forced = (col < FIRST) | (col >= (pages_of - LAST)[:, None])
    score = torch.where(forced[:, None], math.inf, score)
    score = torch.where((col < pages_of[:, None])[:, None], score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    order = torch.where(order < pages_of[:, None, None], order, 1 << 30).sort(-1).values
    chosen = torch.full((R, Hkv, top), -1, dtype=torch.int32, device="cuda")
    chosen[..., :order.shape[-1]] = torch.where(order < 1 << 30, order, -1)

    out = torch.empty((R, Hq, D), device="cuda")
    for r in range(R):
        lp = chosen[r].long()
        page, h = table[seq[r]][lp.clamp(min=0)].long(), torch.arange(Hkv, device="cuda")[:, None]
        k = (_unpack(kc[page, h], bits) * ks[page, h].float()[..., None, None]).flatten(1, 2)
        v = (_unpack(vc[page, h], bits) * vs[page, h].float()[..., None, None]).flatten(1, 2)
        token = (lp[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(1)
        live = (token >= 0) & (token < seen[r])
        logits = torch.matmul(q[r].view(Hkv, G, D), k.transpose(1, 2).contiguous()) * D ** -0.5
        logits = logits.masked_fill(~live[:, None], -math.inf)
        p = torch.exp(logits - logits.amax(-1, keepdim=True))
        out[r] = (torch.matmul(p, v) / p.sum(-1, keepdim=True)).flatten(0, 1)
    return chosen, out.half()


def _plain_sample(s):
    logits = s["logits"].double()
    B, V = logits.shape
    as_row = lambda x: (x.double() if torch.is_tensor(x) else torch.full((B,), float(x), dtype=torch.float64,  # noqa: E731
                                                                       device="cuda"))[:, None]
    t, k, p, m = (as_row(s[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    greedy = t <= 0
    t, k = torch.where(greedy, 1.0, t), torch.where(greedy, 1.0, torch.where(k <= 0, float(V), k))
    z, order = logits.sort(dim=-1, descending=True, stable=True)
    w = torch.exp((z - z[:, :1]) / t)
    rank = torch.arange(V, device="cuda")
    keep = rank < k
    among = torch.where(keep, w, 0.0)
    run = among.cumsum(-1)
    keep &= (p >= 1) | (run - among < p * run[:, -1:])
    keep &= w >= m
    keep |= rank == 0
    weight = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    run = weight.cumsum(-1)
    token = (run <= s["u"].double()[:, None] * run[:, -1:]).sum(-1).int()
    return (token, (weight / run[:, -1:]).float()) if s["case"]["probs"] else token


_PLAIN = {"plan": _plain_plan, "norm": _plain_norm, "bounds": _plain_bounds, "sparse": _plain_sparse,
          "sample": _plain_sample}


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    kind, B = case["kind"], case.get("batch", 1)
    spread = lambda most: [max(1, most * (i + 1) // B) for i in range(B)]  # noqa: E731
    if kind == "plan":
        rows = sum(_grown(case))
        return {"bytes": 24 * B + 20 * rows + 8 * rows / PAGE, "flops": 8 * B + 6 * rows}
    if kind == "norm":
        values = case["tokens"] * case["dim"]
        wide = 4 if case["residual"] == "fp32" else 2
        gate = {"none": 0, "channel": 2 * case["dim"], "token": 2 * case["tokens"], "full": 2 * values}[case["gate"]]
        return {"bytes": values * (4 + 2 * wide) + gate + 2 * case["dim"] * (1 + case["post"]),
                "flops": values * (6 + 4 * case["post"] + 2 * (case["gate"] != "none"))}
    if kind == "sample":
        values = B * case["vocab"]
        size = (4 if case["dtype"] == "fp32" else 2) + 4 * case["probs"]
        return {"bytes": values * size + 24 * B, "flops": 4 * values}
    Hkv, row = case["kv_heads"], D * case["bits"] // 8
    lens = spread(case["longest"])
    if kind == "bounds":
        pages = sum(-(-n // PAGE) - max(0, n - case["new"]) // PAGE for n in lens)
        return {"bytes": pages * Hkv * (PAGE + 2) * row, "flops": pages * Hkv * 2 * PAGE * D}
    n, top = case["rows"], case["top"]
    pages = [-(-max(m, n) // PAGE) for m in lens]
    read = sum(min(m, n * top) for m in pages)
    scored = sum(m for m in pages if m > top)
    used = sum(n * min(m, top) for m in pages)
    return {"bytes": Hkv * (scored * (2 * row + 2) + read * (2 * PAGE * row + 4)) + 4 * B * n * (case["q_heads"] * D
                                                                                            + Hkv * top),
            "flops": 4 * n * scored * case["q_heads"] * D + 4 * used * PAGE * case["q_heads"] * D}


# ---- the same outputs in 64 bits -------------------------------------------------------------------------------

def _exact_plan(case, s):
    table, ring = s["table"].cpu().numpy().copy(), s["ring"].cpu().numpy().copy()
    lens, new, rows = s["lens"].tolist(), s["new"].tolist(), s["rows"]
    head, count = s["ring_state"].tolist()
    (B, W), P = table.shape, len(ring)
    pos, seq, slots = np.full(rows, -1, np.int32), np.full(rows, -1, np.int32), np.full(rows, -1, np.int64)
    starts, counts, after = np.zeros(B + 1, np.int32), np.zeros(B, np.int32), np.zeros(B, np.int32)
    row = asked = taken = 0
    returned = []
    for b in range(B):
        grow, have = max(new[b], 0), -(-lens[b] // PAGE)
        after[b] = lens[b]
        if new[b] < 0:
            after[b] = max(0, lens[b] + new[b])
            returned += table[b, -(-int(after[b]) // PAGE):have].tolist()
        elif lens[b] + grow <= W * PAGE and row + grow <= rows:
            need = -(-(lens[b] + grow) // PAGE) - have
            asked += need
            if need == 0 or asked <= count:
                for j in range(need):
                    table[b, have + j] = ring[(head + taken + j) % P]
                taken += need
                counts[b], after[b] = grow, lens[b] + grow
                t = np.arange(lens[b], lens[b] + grow)
                pos[row:row + grow], seq[row:row + grow] = t, b
                slots[row:row + grow] = table[b, t // PAGE].astype(np.int64) * PAGE + t % PAGE
        row += grow
        starts[b + 1] = min(row, rows)
    for j, page in enumerate(returned):
        ring[(head + count + j) % P] = page
    state = np.array([(head + taken) % P, count - taken + len(returned)], np.int32)
    return tuple(torch.from_numpy(x) for x in (starts, counts, after, pos, pos + 1, seq, slots, table, ring, state))


def _exact_norm(case, s):
    u = s["x"].double()
    one = 1 if case["unit_offset"] else 0
    if s["post"] is not None:
        u = u / (u.square().sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * (s["post"].double() + one)
    if s["gate"] is not None:
        g = s["gate"].double()
        u = u * (torch.sigmoid(g) if case["sigmoid"] else g)
    h = s["residual"].double() + case["scale"] * u
    y = h / (h.square().sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * (s["weight"].double() + one)
    return y, h


def _numpy_codes(t, bits):
    c = t.cpu().numpy()
    if bits == 8:
        return c.astype(np.int16)
    low, high = (c & 15).astype(np.int16), (c >> 4).astype(np.int16)
    out = np.empty(c.shape[:-1] + (D,), np.int16)
    out[..., 0::2], out[..., 1::2] = low - 16 * (low > 7), high - 16 * (high > 7)
    return out


def _exact_bounds(case, s):
    out = s["bounds"].cpu().numpy().copy()
    for b, (n, first) in enumerate(zip(s["lens"].tolist(), s["first"].tolist())):
        ids = s["table"][b, first // PAGE:-(-n // PAGE)].long()
        codes = _numpy_codes(s["k"][ids], case["bits"])  # [pages, Hkv, 16, 128]
        high, low = codes.max(2), codes.min(2)
        if n % PAGE:
            high[-1], low[-1] = codes[-1, :, :n % PAGE].max(1), codes[-1, :, :n % PAGE].min(1)
        both = np.stack([high, low], axis=2)
        if case["bits"] == 4:
            both = ((both[..., 0::2] & 15) | (both[..., 1::2] & 15) << 4)
        out[ids.cpu().numpy()] = both.astype(out.dtype)
    return torch.from_numpy(out)


def _exact_sparse(case, s):
    (k, v, ks, vs), bits, top = s["cache"], case["bits"], case["top"]
    R, Hq, _ = s["q"].shape
    Hkv = case["kv_heads"]
    G = Hq // Hkv
    chosen = np.full((R, Hkv, top), -1, np.int32)
    out = torch.empty((R, Hq, D), dtype=torch.float64)
    codes = lambda t: torch.from_numpy(_numpy_codes(t, bits)).double()  # noqa: E731
    edges = {}
    for r in range(R):
        b = r if s["row_seq"] is None else int(s["row_seq"][r])
        n = int(s["seen"][r])
        last = -(-n // PAGE)
        ids = s["table"][b, :last].long()
        if b not in edges:
            edges = {b: torch.from_numpy(_numpy_codes(s["bounds"][s["table"][b].long()], bits)).cuda().double()}
        for h in range(Hkv):
            q = s["q"][r, h * G:(h + 1) * G].double()
            most = q.abs().amax(1, keepdim=True)
            whole = torch.where(most > 0, torch.round(q * 127 / most), 0.0)  # [G, D]
            edge = edges[b][:last, h]
            top_of = torch.zeros((last, G), dtype=torch.float64, device="cuda")
            for g in range(G):
                top_of[:, g] = torch.maximum(whole[g] * edge[:, 0], whole[g] * edge[:, 1]).sum(1)
            worth = top_of * (most[:, 0] * ks[ids, h].double()[:, None])
            worth = worth.float().amax(1).cpu().numpy()  # rounded once
            fixed = [p for p in range(last) if p < FIRST or p >= last - LAST]
            rest = [p for p in np.argsort(-worth, kind="stable").tolist() if p not in fixed]
            take = sorted((fixed + rest)[:top])
            chosen[r, h, :len(take)] = take
            page = ids[torch.tensor(take, device="cuda")]
            live = (np.array(take)[:, None] * PAGE + np.arange(PAGE)).reshape(-1) < n
            kk = (codes(k[page, h]) * ks[page, h].double().cpu()[:, None, None]).reshape(-1, D)[live]
            vv = (codes(v[page, h]) * vs[page, h].double().cpu()[:, None, None]).reshape(-1, D)[live]
            a = torch.softmax(q.cpu() @ kk.T / math.sqrt(D), dim=-1)
            out[r, h * G:(h + 1) * G] = a @ vv
    return torch.from_numpy(chosen), out


def _exact_sample(case, s):
    B, V = s["logits"].shape
    setting = {name: s[name].double().tolist() if torch.is_tensor(s[name]) else [float(s[name])] * B
               for name in ("temperature", "top_k", "top_p", "min_p")}
    u = s["u"].double().tolist()
    tokens, probs = np.empty(B, np.int32), np.zeros((B, V))
    for b in range(B):
        x = s["logits"][b].double().cpu().numpy()
        t, k, p, m = (setting[name][b] for name in ("temperature", "top_k", "top_p", "min_p"))
        order = np.lexsort((np.arange(V), -x))
        if t <= 0:
            t, k = 1.0, 1
        order = order[:int(k)] if k > 0 else order
        w = np.exp((x[order] - x[order[0]]) / t)
        count = len(order)
        if p < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            count = max(1, int((before < p * w.sum()).sum()))
        count = max(1, min(count, int((w >= m).sum())))
        probs[b, order[:count]] = w[:count] / w[:count].sum()
        run = np.cumsum(probs[b])
        tokens[b] = np.searchsorted(run, u[b] * run[-1], "right")
    return (torch.from_numpy(tokens), torch.from_numpy(probs)) if case["probs"] else torch.from_numpy(tokens)


_EXACT = {"plan": _exact_plan, "norm": _exact_norm, "bounds": _exact_bounds, "sparse": _exact_sparse,
          "sample": _exact_sample}


def exact(case, seed):
    return _EXACT[case["kind"]](case, prepare(case, seed))
