"""Performance cases of the serving and rotation operators: what a program around the attention of
this framework has them do.

Four kinds of work:

  rotary   queries and keys of an attention layer are normed per head (optional) and rotated by their
           positions, in one pass; with "train" the gradients of a training step too
  append   the new tokens of a batch of sequences go into a paged cache: keys normed and rotated on the
           way, values as they are, and the tokens' queries normed and rotated beside them
  packed   causal attention over whole prompts of different lengths that lie packed behind each other,
           query heads in groups that share a key head
  paged    attention of new tokens (one per sequence, or a chunk of a prompt) over a paged cache

A case is a dict of plain values:
  op           which of the four
  lens         tokens of each sequence of the batch ("append": new tokens; "paged": new tokens)
  cached       ("append", "paged") keys of each sequence that the cache holds before them
  Hq, Hk, D    query heads, key heads, head dimension
  dtype        "float16" or "bfloat16"
  rot          rotated dimensions of a head
  interleaved  pairs (2i, 2i + 1) rotate together; else (i, i + rot / 2)
  norm         queries and keys are normed by their root mean square and a weight per dimension
  train        ("rotary") gradients as well
  page         ("append", "paged") tokens per page
  softcap      cap of the scores, 0 = none
  causal       ("packed", "paged") a token attends its own position and those before; else the whole sequence

"exact" works in 64 bits from the definitions, one sequence and head group at a time.
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"float16": torch.float16, "bfloat16": torch.bfloat16}
_EPS = 1e-6


def _ops():
    package = os.path.join(os.getcwd(), "omni-attention_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import omni_attn_torch
    return omni_attn_torch


def _case(op, lens, Hq, Hk, D, dtype, cached=(), rot=0, interleaved=False, norm=False, train=False, page=0,
          softcap=0.0, causal=True):
    return {"op": op, "lens": [int(n) for n in lens], "cached": [int(n) for n in cached], "Hq": Hq, "Hk": Hk, "D": D,
            "dtype": dtype, "rot": rot, "interleaved": interleaved, "norm": norm, "train": train, "page": page,
            "softcap": softcap, "causal": causal}


def _spread(n, low, high, seed):
    """n lengths spread over low .. high by their logarithm."""
    rng = random.Random(seed)
    return [int(round(math.exp(rng.uniform(math.log(low), math.log(high))))) for _ in range(n)]


def listed():
    named = [
        # a short prompt of a small model: launch latency and the host path
        ("rotary_512", _case("rotary", [512], 8, 8, 64, "float16", rot=64)),
        # half of the head rotates, pairs interleaved, an odd length, in training
        ("rotary_train_partial_1157", _case("rotary", [1157] * 4, 16, 16, 64, "float16", rot=32, interleaved=True,
                                            train=True)),
        # a training step's layer with normed heads and shared key heads
        ("rotary_train_norm_4096", _case("rotary", [4096] * 2, 32, 8, 128, "bfloat16", rot=128, norm=True, train=True)),
        # one token of every sequence of a serving batch
        ("append_single_64", _case("append", [1] * 64, 32, 8, 128, "bfloat16", _spread(64, 1, 500, 1), rot=128, norm=True,
                                   page=64)),
        # whole prompts of different lengths enter the cache
        ("append_prompts", _case("append", _spread(12, 100, 2048, 2), 32, 8, 128, "bfloat16", [0] * 12, rot=64, page=64)),
        # a short prompt of a small model
        ("packed_512", _case("packed", [512], 8, 8, 64, "float16")),
        # prompts of different lengths, some a few tokens long, at half the head dimension with capped scores
        ("packed_ragged_softcap", _case("packed", _spread(9, 33, 2048, 3), 16, 16, 64, "float16", softcap=50.0)),
        # a serving batch of prompts of different lengths
        ("packed_ragged", _case("packed", _spread(12, 100, 4096, 4), 32, 8, 128, "bfloat16")),
        # a long document
        ("packed_16384", _case("packed", [16384], 32, 8, 128, "bfloat16")),
        # the next token of one short conversation: latency
        ("paged_single_1", _case("paged", [1], 32, 8, 128, "bfloat16", [700], page=64)),
        # the next tokens of a serving batch of conversations of different lengths
        ("paged_single_64", _case("paged", [1] * 64, 32, 8, 128, "bfloat16", _spread(64, 300, 16000, 5), page=64)),
        # a chunk of a long prompt, the part before it in the cache
        ("paged_chunk_512", _case("paged", [512, 300], 32, 8, 128, "bfloat16", [15000, 7001], page=64)),
    ]
    return [dict(case, name=name) for name, case in named]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Costs no more than the largest listed cases of the same kind."""
    op = rng.choice(["rotary", "append", "packed", "paged"])
    dtype = rng.choice(["float16", "bfloat16"])
    D = rng.choice([32, 64, 128])
    Hk = rng.choice([1, 2, 4, 8])
    Hq = Hk * rng.choice([1, 2, 3, 4, 8] if Hk < 8 else [1, 2, 4])
    softcap = rng.choice([0.0, 0.0, 30.0])
    page = rng.choice([16, 32, 64, 128])
    if op == "rotary":
        B, D = rng.choice([1, 2, 3, 4]), rng.choice([D, 96])
        return _case(op, [_log_uniform(rng, 100, 8000 // B)] * B, Hq, Hk, D, dtype, rot=rng.choice([D, D // 2, D // 4]),
                     interleaved=rng.random() < 0.5, norm=rng.random() < 0.5, train=rng.random() < 0.7)
    if op == "append":
        n = _log_uniform(rng, 1, 64)
        single = rng.random() < 0.5
        lens = [1] * n if single else [_log_uniform(rng, 1, max(2, 8000 // n)) for _ in range(n)]
        cached = [_log_uniform(rng, 1, 500) - 1 for _ in range(n)]
        return _case(op, lens, Hq, Hk, D, dtype, cached, rot=rng.choice([D, D // 2]), interleaved=rng.random() < 0.5,
                     norm=rng.random() < 0.5, page=page)
    if op == "packed":
        n = _log_uniform(rng, 1, 12)
        return _case(op, [_log_uniform(rng, 20, 8000 // n) for _ in range(n)], Hq, Hk, D, dtype, softcap=softcap,
                     causal=rng.random() < 0.8)
    n = _log_uniform(rng, 1, 64)
    if rng.random() < 0.7:
        return _case(op, [1] * n, Hq, Hk, D, dtype, [_log_uniform(rng, 200, 16000) for _ in range(n)], page=page,
                     softcap=softcap)
    n = min(n, 8)
    return _case(op, [_log_uniform(rng, 2, 500) for _ in range(n)], Hq, Hk, D, dtype,
                 [_log_uniform(rng, 200, 8000) for _ in range(n)], page=page, softcap=softcap, causal=rng.random() < 0.8)


# ---- inputs ------------------------------------------------------------------------------------

def _table(rot, rows):
    """[rows, rot] cosines, then sines, of position * 10000^(-2 i / rot): what a model keeps."""
    inverse = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64).unsqueeze(1) * inverse
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, Hq, Hk, D, op = _DT[case["dtype"]], case["Hq"], case["Hk"], case["D"], case["op"]
    lens, cached = case["lens"], case["cached"]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda", dtype=dt)
    s = {"case": case}
    weight = lambda: (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)
    if op == "rotary":
        B, S = len(lens), lens[0]
        # a projection's [B, S, H, D] results, seen as [B, H, S, D]
        s["q"], s["k"] = normal(B, S, Hq, D).transpose(1, 2), normal(B, S, Hk, D).transpose(1, 2)
        s["positions"] = torch.arange(S, device="cuda")
        s["table"] = _table(case["rot"], S)
        s["wq"], s["wk"] = (weight(), weight()) if case["norm"] else (None, None)
        if case["train"]:
            s["dq"], s["dk"] = normal(B, S, Hq, D).transpose(1, 2), normal(B, S, Hk, D).transpose(1, 2)
            for name in ("q", "k", "wq", "wk"):
                if s[name] is not None:
                    s[name] = s[name].requires_grad_()
        return s
    T = sum(lens)
    s["q"] = normal(T, Hq, D)
    s["cu"] = torch.tensor(_offsets(lens), dtype=torch.int32, device="cuda")
    if op == "packed":
        s["k"], s["v"] = normal(T, Hk, D), normal(T, Hk, D)
        return s
    page = case["page"]
    total = [n + c for n, c in zip(lens, cached)]
    pages = [-(-n // page) for n in total]
    order = torch.randperm(sum(pages) + 3, generator=g, device="cuda").to(torch.int32)  # (some pages are nobody's)
    s["page_table"] = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        s["page_table"][b, :n] = order[at:at + n]
        at += n
    s["kv_lens"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    s["k_pages"], s["v_pages"] = normal(order.numel(), Hk, page, D), normal(order.numel(), Hk, page, D)
    if op == "append":
        s["k"], s["v"] = normal(T, Hk, D), normal(T, Hk, D)
        s["table"] = _table(case["rot"], max(total))
        s["wq"], s["wk"] = (weight(), weight()) if case["norm"] else (None, None)
    return s


# ---- plain forms -------------------------------------------------------------------------------

def _halves(x, case):
    """The two members of each rotating pair, and what does not rotate."""
    rot = case["rot"]
    if case["interleaved"]:
        return x[..., 0:rot:2], x[..., 1:rot:2], x[..., rot:]
    return x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]


def _whole(a, b, rest, case):
    if case["interleaved"]:
        return torch.cat([torch.stack([a, b], -1).flatten(-2), rest], -1)
    return torch.cat([a, b, rest], -1)


def _rotate(x, cos, sin, case):
    a, b, rest = _halves(x, case)
    return _whole(a * cos - b * sin, b * cos + a * sin, rest, case)


def _norm(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w


def _norm_rotate_gradients(x, w, dy, cos, sin, case):
    g = _rotate(dy, cos, -sin, case)
    if w is None:
        return g, None
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    n = x * r
    dn = g * w
    return r * (dn - n * (dn * n).mean(-1, keepdim=True)), (g * n).sum(tuple(range(x.dim() - 1)))


def _plain_rotary(s, wide):
    case, rot = s["case"], s["case"]["rot"]
    q, k, dq, dk, wq, wk = (None if s.get(n) is None else s[n].detach().to(wide) for n in ("q", "k", "dq", "dk", "wq", "wk"))
    angles = s["table"].to(wide)[s["positions"]]
    cos, sin = angles[:, :rot // 2], angles[:, rot // 2:]
    out = [_rotate(_norm(x, w), cos, sin, case) for x, w in ((q, wq), (k, wk))]
    if case["train"]:
        grads = [_norm_rotate_gradients(x, w, d, cos, sin, case) for x, w, d in ((q, wq, dq), (k, wk, dk))]
        out += [grads[0][0], grads[1][0]]
        if case["norm"]:
            out += [grads[0][1], grads[1][1]]
    return out


def _append_rows(s, wide):
    """What each token's query, key and value are, and where in the pools the latter two go."""
    case, rot = s["case"], s["case"]["rot"]
    cu, lens = s["cu"].long(), s["kv_lens"].long()
    token = torch.arange(s["k"].shape[0], device=cu.device)
    b = torch.searchsorted(cu[1:], token, right=True)
    at = lens[b] - (cu[b + 1] - token)
    page = s["page_table"].long()[b, at // case["page"]]
    angles = s["table"].to(wide)[at].unsqueeze(1)
    cos, sin = angles[..., :rot // 2], angles[..., rot // 2:]
    wq, wk = (None if s[n] is None else s[n].to(wide) for n in ("wq", "wk"))
    q = _rotate(_norm(s["q"].to(wide), wq), cos, sin, case)
    k = _rotate(_norm(s["k"].to(wide), wk), cos, sin, case)
    return q, k, page, at % case["page"]


def _attend(q, k, v, first, case):
    """q [n, Hq, D] whose first row lies at position `first`, k and v [m, Hk, D], all of one wide type."""
    n, Hq, D = q.shape
    m, Hk = k.shape[0], k.shape[1]
    G = Hq // Hk
    out = torch.empty_like(q)
    rows = max(1, min(n, (1 << 27) // (G * m)))  # (scores of at most 2^27 entries at a time)
    for h in range(Hk):
        kh, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
        for r0 in range(0, n, rows):
            qh = q[r0:r0 + rows, h * G:(h + 1) * G].reshape(-1, D)
            x = (qh @ kh).mul_(1.0 / math.sqrt(D))
            if case["softcap"]:
                x = (x / case["softcap"]).tanh_().mul_(case["softcap"])
            if case["causal"]:
                at = first + r0 + torch.arange(qh.shape[0], device=q.device) // G
                x = x.masked_fill_(torch.arange(m, device=q.device) > at.unsqueeze(1), float("-inf"))
            x = (x - x.amax(1, keepdim=True)).exp_()
            out[r0:r0 + rows, h * G:(h + 1) * G] = ((x @ vh) / x.sum(1, keepdim=True)).view(-1, G, D)
    return out


def _plain_packed(s, wide):
    at = _offsets(s["case"]["lens"])
    q, k, v = (s[n].to(wide) for n in ("q", "k", "v"))
    return torch.cat([_attend(q[a:b], k[a:b], v[a:b], 0, s["case"]) for a, b in zip(at, at[1:])])


def _plain_paged(s, wide):
    case, at = s["case"], _offsets(s["case"]["lens"])
    out = []
    for b, (n, c) in enumerate(zip(case["lens"], case["cached"])):
        pages = s["page_table"][b, :-(-(n + c) // case["page"])].long()
        k, v = (s[p][pages].to(wide).transpose(1, 2).reshape(-1, case["Hk"], case["D"])[:n + c]
                for p in ("k_pages", "v_pages"))
        out.append(_attend(s["q"][at[b]:at[b + 1]].to(wide), k, v, c, case))
    return torch.cat(out)


def run(state):
    s, case = state, state["case"]
    if own:
        return _run_own(s, case)
    dt = _DT[case["dtype"]]
    with torch.no_grad():
        if case["op"] == "rotary":
            return [t.to(dt) for t in _plain_rotary(s, torch.float32)]
        if case["op"] == "append":
            q, k, page, row = _append_rows(s, torch.float32)
            s["k_pages"][page, :, row] = k.to(dt)
            s["v_pages"][page, :, row] = s["v"]
            return [q.to(dt), s["k_pages"], s["v_pages"]]
        return (_plain_packed if case["op"] == "packed" else _plain_paged)(s, torch.float32).to(dt)


def _run_own(s, case):
    ops = _ops()
    if case["op"] == "rotary":
        out = list(ops.omni_qk_rotary(s["q"], s["k"], s["positions"], s["table"], query_norm=s["wq"], key_norm=s["wk"],
                                      eps=_EPS, interleaved=case["interleaved"]))
        if case["train"]:
            leaves = [s[n] for n in ("q", "k", "wq", "wk") if s[n] is not None]
            out += torch.autograd.grad(out, leaves, [s["dq"], s["dk"]])
        return [t.detach() for t in out]
    if case["op"] == "append":
        q = ops.omni_cache_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_lens"], s["cu"],
                                  table=s["table"], query=s["q"], query_norm=s["wq"], key_norm=s["wk"], eps=_EPS,
                                  interleaved=case["interleaved"])
        return [q, s["k_pages"], s["v_pages"]]
    if case["op"] == "packed":
        return ops.omni_attention_packed(s["q"], s["k"], s["v"], s["cu"], causal=case["causal"], softcap=case["softcap"])
    return ops.omni_attention_paged(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_lens"], s["cu"],
                                    causal=case["causal"], softcap=case["softcap"])


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    Hq, Hk, D, rot, lens, cached = (case[n] for n in ("Hq", "Hk", "D", "rot", "lens", "cached"))
    T = sum(lens)
    if case["op"] == "rotary":
        rows, elems = T * (Hq + Hk), T * (Hq + Hk) * D
        table = lens[0] * (rot * 4 + 8)
        norms = 2 * 2 * D * case["norm"]
        flops = 3 * rows * rot + 4 * elems * case["norm"]
        if not case["train"]:
            return {"bytes": 2 * 2 * elems + table + norms, "flops": flops}
        # forward: read, write; gradients: the incoming ones, the inputs where there is a norm, the outgoing ones
        return {"bytes": 2 * elems * (4 + case["norm"]) + 2 * table + 3 * norms,
                "flops": 2 * flops + 6 * elems * case["norm"]}
    if case["op"] == "append":
        elems = T * (Hq + 2 * Hk) * D
        return {"bytes": 2 * 2 * elems + T * rot * 4 + 4 * T + 8 * len(lens) + 4 * D * case["norm"],
                "flops": 3 * T * (Hq + Hk) * rot + 4 * T * (Hq + Hk) * D * case["norm"]}
    pairs, keys = 0, 0
    for i, n in enumerate(lens):
        c = cached[i] if cached else 0
        pairs += n * c + (n * (n + 1) // 2 if case["causal"] else n * n)
        keys += n + c
    return {"bytes": 2 * (2 * T * Hq * D + 2 * keys * Hk * D) + 4 * len(lens)
            + (4 * sum(-(-(n + c) // case["page"]) for n, c in zip(lens, cached)) + 4 * len(lens) if cached else 0),
            "flops": 4 * pairs * Hq * D}


# ---- 64 bits, from the definitions ----------------------------------------------------------------

def _rotation_matrices(table, rot, D, interleaved):
    """[rows, D, D] in 64 bits: y = R x for one position each."""
    P = table.shape[0]
    R = torch.zeros(P, D, D, dtype=torch.float64, device=table.device)
    i = torch.arange(rot // 2, device=table.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    cos, sin = table[:, :rot // 2].double(), table[:, rot // 2:].double()
    R[:, a, a] = cos
    R[:, b, b] = cos
    R[:, a, b] = -sin
    R[:, b, a] = sin
    tail = torch.arange(rot, D, device=table.device)
    R[:, tail, tail] = 1.0
    return R


def _exact_rows(x, w, table, positions, case, dy=None):
    """x [H, n, D] of the rows at `positions`: the results, with dy also dx and the rows' sum of dw."""
    R = _rotation_matrices(table[positions], case["rot"], case["D"], case["interleaved"])  # [n, D, D]
    x = x.double()
    n = x
    if w is not None:
        scale = 1.0 / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["D"] + _EPS)
        n = x * scale
    y = torch.matmul(R, (n if w is None else n * w.double()).permute(1, 2, 0)).permute(2, 0, 1)
    if dy is None:
        return y
    back = torch.matmul(R.transpose(1, 2).contiguous(), dy.double().permute(1, 2, 0).contiguous()).permute(2, 0, 1)
    if w is None:
        return y, back, None
    dn = back * w.double()
    # d/dx of x / sqrt(mean x^2 + eps): (dn - x (x . dn) scale^2 / D) scale
    return y, (dn - x * (x * dn).sum(-1, keepdim=True) * scale.pow(2) / case["D"]) * scale, (back * n).sum((0, 1))


def _exact_rotary(s, case):
    outs, grads, sums = [], [], []
    for name, dname, wname in (("q", "dq", "wq"), ("k", "dk", "wk")):
        x, w = s[name].detach(), None if s[wname] is None else s[wname].detach()
        y = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        dx = torch.empty_like(y)
        dw = torch.zeros(case["D"], dtype=torch.float64, device=x.device)
        for b in range(x.shape[0]):
            for r0 in range(0, x.shape[2], 512):
                rows = slice(r0, min(r0 + 512, x.shape[2]))
                dy = s[dname][b, :, rows] if case["train"] else None
                got = _exact_rows(x[b, :, rows], w, s["table"], s["positions"][rows], case, dy)
                if dy is None:
                    y[b, :, rows] = got
                else:
                    y[b, :, rows], dx[b, :, rows] = got[0], got[1]
                    if w is not None:
                        dw += got[2]
        outs.append(y)
        grads.append(dx)
        sums.append(dw)
    return outs + (grads if case["train"] else []) + (sums if case["train"] and case["norm"] else [])


def _exact_append(s, case):
    q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    at, page = _offsets(case["lens"]), case["page"]
    for b, (n, c) in enumerate(zip(case["lens"], case["cached"])):
        rows = slice(at[b], at[b + 1])
        where = torch.arange(c, c + n, device="cuda")
        in_page, row = s["page_table"][b].long()[torch.div(where, page, rounding_mode="floor")], where.remainder(page)
        k = torch.empty(n, case["Hk"], case["D"], dtype=torch.float64, device="cuda")
        for r0 in range(0, n, 512):
            part = slice(r0, min(r0 + 512, n))
            for x, w, out in ((s["q"][rows][part], s["wq"], q[rows][part]), (s["k"][rows][part], s["wk"], k[part])):
                out.copy_(_exact_rows(x.transpose(0, 1), w, s["table"], where[part], case).transpose(0, 1))
        k_pages[in_page, :, row] = k
        v_pages[in_page, :, row] = s["v"][rows].double()
    return [q, k_pages, v_pages]


def _exact_attention(q, k, v, first, case):
    """Softmax over the allowed keys, in 64 bits; one query head and up to 2048 rows at a time."""
    n, Hq, D = q.shape
    G = Hq // k.shape[1]
    out = torch.empty(n, Hq, D, dtype=torch.float64, device=q.device)
    for h in range(Hq):
        keys, values = k[:, h // G].double(), v[:, h // G].double()
        for r0 in range(0, n, 2048):
            r1 = min(n, r0 + 2048)
            seen = first + r1 if case["causal"] else keys.shape[0]
            scores = torch.mm(q[r0:r1, h].double(), keys[:seen].t()) / math.sqrt(D)
            if case["softcap"]:
                scores = case["softcap"] * torch.tanh(scores / case["softcap"])
            if case["causal"]:
                allowed = torch.ones(r1 - r0, seen, dtype=torch.bool, device=q.device).tril(first + r0)
                scores = torch.where(allowed, scores, -math.inf)
            out[r0:r1, h] = torch.mm(torch.softmax(scores, -1), values[:seen])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rotary":
            return _exact_rotary(s, case)
        if case["op"] == "append":
            return _exact_append(s, case)
        at, page = _offsets(case["lens"]), case["page"]
        out = []
        for b, n in enumerate(case["lens"]):
            q = s["q"][at[b]:at[b + 1]]
            if case["op"] == "packed":
                k, v, c = s["k"][at[b]:at[b + 1]], s["v"][at[b]:at[b + 1]], 0
            else:
                c = case["cached"][b]
                where = torch.arange(n + c, device="cuda")
                in_page = s["page_table"][b].long()[torch.div(where, page, rounding_mode="floor")]
                k, v = s["k_pages"][in_page, :, where.remainder(page)], s["v_pages"][in_page, :, where.remainder(page)]
            out.append(_exact_attention(q, k, v, c, case))
        return torch.cat(out)
