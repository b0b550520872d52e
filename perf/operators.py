"""What is timed for the operators of a paged key / value cache: the work of one call of each, through the public entry points.

A serving program keeps the keys and values of its sequences in pages of a fixed number of positions.  A step brings `n_new` tokens of
every sequence (one while it answers, a chunk of its prompt before that); their q, k and v come side by side out of one product.  Kinds:
  norm    RmsNorm of every head of q and k and the rotation by position, no cache             (LlmContext.qk_norm_rope)
  append  the same, keys and values going into the pages of their sequences, in one pass      (LlmContext.paged_append)
  attend  causal attention of the step's tokens to everything their sequences hold by then    (LlmContext.paged_attention)
`own` says which form `run` takes: plain torch operations, or the library's calls.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

BASE, EPS = 10000.0, 1e-5
MOST_BYTES, MOST_FLOPS, MOST_SCORES = 5.0e8, 2.5e11, 5.3e8  # of a drawn case: what the largest listed ones have


# ---- the cases ---------------------------------------------------------------------------------------------------------
def _case(kind: str, heads: int, kv_heads: int, size: int, *, name: str = "", kv: str = "f16", page: int = 16, order: str = "head", seqs: int = 1,
          ctx: tuple[int, int] = (0, 0), new: int = 1, mix: str = "even", variant: int = 0, norms: bool = True) -> dict:
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, size=size, kv=kv, page=page, order=order, seqs=seqs, ctx_lo=ctx[0], ctx_hi=ctx[1], new=new,
             mix=mix, variant=variant, norms=norms)
    return dict(c, name=name) if name else c


def listed() -> list[dict]:
    return [
        # one token of one conversation, grouped-query heads: nothing but latency
        _case("norm", 64, 8, 128, name="norm_token", ctx=(515, 515), variant=1),
        # a chunk of a long document far into its context, where an angle in 32 bits has lost its digits
        _case("norm", 64, 8, 128, name="norm_chunk_4095", ctx=(120000, 120000), new=4095, variant=1),
        # the tiny story model (odd widths, f32 cache): one token
        _case("append", 6, 6, 48, name="append_tiny_token", kv="f32", ctx=(100, 100), order="pos", norms=False),
        # serving: a token of each of eight conversations, adjacent pairs rotated, no norms
        _case("append", 32, 32, 128, name="append_batch_8", seqs=8, ctx=(515, 546), norms=False),
        # serving: prompt chunks of several new conversations in one step
        _case("append", 64, 8, 128, name="append_chunks_1919", seqs=5, ctx=(0, 1021), new=511, mix="ragged", page=64, variant=1),
        # chat, a token of one conversation
        _case("attend", 32, 32, 128, name="attend_token", ctx=(515, 515)),
        # an answer late in a long conversation
        _case("attend", 64, 8, 128, name="attend_long_token", ctx=(32750, 32750), page=64),
        # serving: a token of each of 64 conversations of all lengths
        _case("attend", 64, 8, 128, name="attend_batch_64", seqs=64, ctx=(100, 3900)),
        # serving with the reference's own f32 cache, position-major pages of an odd size
        _case("attend", 32, 32, 128, name="attend_batch_8_f32", kv="f32", seqs=8, ctx=(515, 1546), page=20, order="pos"),
        # the prompt of the headline workload
        _case("attend", 32, 32, 128, name="attend_prompt_511", new=511),
        # a chunk of a long prompt behind what is cached of it
        _case("attend", 64, 8, 128, name="attend_chunk_1023", ctx=(7001, 7001), new=1023, page=64),
        # a short turn that follows a conversation, f32 cache
        _case("attend", 32, 32, 128, name="attend_turn_37_f32", kv="f32", ctx=(300, 300), new=37),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng) -> dict:
    while True:
        size = rng.choice([128, 128, 128, 64, 64, 48, 80, 96])
        group = rng.choice([1, 1, 2, 4, 4, 8, 3, 5])
        kv_heads = _log_int(rng, 1, 32)
        kind = rng.choice(["norm", "append", "append", "attend", "attend", "attend", "attend"])
        new = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 64, 4095)])
        seqs = 1 if rng.random() < 0.3 else _log_int(rng, 2, 64)
        lo = rng.choice([0, _log_int(rng, 1, 30000)])
        hi = lo + (_log_int(rng, 1, 8000) if seqs > 1 else 0)
        if kind == "norm" and rng.random() < 0.5:
            lo, hi = lo + 100000, hi + 100000
        c = _case(kind, kv_heads * group, kv_heads, size, kv=rng.choice(["f16", "f16", "f16", "f32"]), page=rng.choice([16, 16, 32, 64, 128, 20]),
                  order=rng.choice(["head", "pos"]), seqs=seqs, ctx=(lo, hi), new=new, mix=rng.choice(["even", "ragged", "one"]) if new > 1 else "even",
                  variant=rng.choice([0, 1]), norms=rng.random() < 0.6)
        pos0, n_new = _lengths(c)
        if sum(n_new) > 40000:
            continue
        w = work(c)
        held = sum(-(-(p + n) // c["page"]) for p, n in zip(pos0, n_new)) * c["page"] * kv_heads * size * 2 * (2 if c["kv"] == "f16" else 4)
        # f32 caches are worked on without the help of the matrix units: an eighth of the operations
        if w["bytes"] > MOST_BYTES or w["flops"] > MOST_FLOPS / (8 if c["kv"] == "f32" else 1) or (kind != "norm" and held > 8 * MOST_BYTES / 4):
            continue
        if kind == "attend" and seqs * max(n_new) * max(p + n for p, n in zip(pos0, n_new)) * c["heads"] > MOST_SCORES:
            continue
        return c


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Cached positions and new tokens of each sequence."""
    n, lo, hi, new = case["seqs"], case["ctx_lo"], case["ctx_hi"], case["new"]
    last = max(1, n - 1)
    pos0 = [hi - (hi - lo) * b // last for b in range(n)]
    if case["mix"] == "ragged":
        return pos0, [max(1, new - new * b // (2 * last)) for b in range(n)]
    if case["mix"] == "one":
        return pos0, [new if b == 0 else 1 for b in range(n)]
    return pos0, [new] * n


# ---- state -------------------------------------------------------------------------------------------------------------
class _Operand:
    """A torch tensor handed to the operators: they take anything with a device pointer and a length."""

    def __init__(self, t: torch.Tensor):
        self.t, self.ptr = t, t.data_ptr()
        self.n = 1 + sum((size - 1) * step for size, step in zip(t.shape, t.stride()))  # from its first element to its last

    def __len__(self):
        return self.n


_backend: list = []


def _the_backend():
    """A program has one backend (device context and stream)."""
    from slai_b200.ops import Backend
    if not _backend:
        _backend.append(Backend(0))
    return _backend[0]


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng([seed, 31])
    hq, hk, hs, page = case["heads"], case["kv_heads"], case["size"], case["page"]
    pos0, n_new = _lengths(case)
    rows = sum(n_new)
    dev = lambda a: torch.as_tensor(a, device="cuda")  # noqa: E731
    first = np.concatenate([[0], np.cumsum(n_new)[:-1]])
    seq = np.repeat(np.arange(len(n_new)), n_new)
    inner = np.arange(rows) - first[seq]
    pos = np.asarray(pos0)[seq] + inner
    s = dict(case=case, rows=rows, pos=dev(pos.astype(np.int32)), seq=dev(seq), inner=dev(inner), most_new=max(n_new))
    if case["norms"]:
        s["q_norm"] = 1 + 0.2 * torch.randn(hs, generator=gen, device="cuda")
        s["k_norm"] = 1 + 0.2 * torch.randn(hs, generator=gen, device="cuda")
    if case["kind"] == "attend":
        # queries as long as normalised ones are: some heads attend to a few positions, others to many
        s["q"] = torch.randn(rows, hq, hs, generator=gen, device="cuda") * (0.5 + 2 * torch.rand(1, hq, 1, generator=gen, device="cuda"))
        s["out"] = torch.empty(rows, hq, hs, device="cuda")
    else:
        # one product's rows: q, k, v side by side
        s["qkv"] = torch.randn(rows, (hq + 2 * hk) * hs, generator=gen, device="cuda") * 1.5
        s["q_out"] = torch.empty(rows, hq, hs, device="cuda")
        s["k_out"] = torch.empty(rows, hk, hs, device="cuda")
    if case["kind"] != "norm":
        used = [-(-(p + n) // page) for p, n in zip(pos0, n_new)]
        pages = sum(used) + 3
        order = rng.permutation(pages)[: sum(used)].astype(np.int32)  # pages lie where earlier conversations left room
        table = np.zeros((len(used), max(used)), np.int32)
        at = 0
        for b, u in enumerate(used):
            table[b, :u] = order[at : at + u]
            at += u
        shape = (pages, hk, page, hs) if case["order"] == "head" else (pages, page, hk, hs)
        s["table"] = dev(table.astype(np.int64))
        for name in ("keys", "values"):
            s[name] = torch.randn(shape, generator=gen, device="cuda").to(torch.float16 if case["kv"] == "f16" else torch.float32)
        s["most_pos"] = max(p + n for p, n in zip(pos0, n_new))
    if own:
        _prepare_own(s, pos0, n_new, table if case["kind"] != "norm" else None)
    torch.cuda.synchronize()
    return s


def _prepare_own(s: dict, pos0: list, n_new: list, table) -> None:
    from slai_b200 import _lib, ops
    case = s["case"]
    be = _the_backend()
    hq, hk, hs = case["heads"], case["kv_heads"], case["size"]
    s["ctx"] = ops.LlmContext(be)
    if case["kind"] != "norm":
        page = case["page"]
        s["paged"] = ops.PagedKv(be, n_q_heads=hq, n_kv_heads=hk, head_size=hs, page_size=page, n_pages=s["keys"].shape[0],
                                 kv_dtype=_lib.KV_F16 if case["kv"] == "f16" else _lib.KV_F32, max_seqs=len(n_new), max_tokens=s["rows"],
                                 max_table=table.size)
        s["paged"].step(pos0, n_new, table)
        head_stride, pos_stride = (page * hs, hs) if case["order"] == "head" else (hs, hk * hs)
        s["layer"] = ops.PagedLayer(_Operand(s["keys"]), _Operand(s["values"]), hk * page * hs, head_stride, pos_stride)
    if case["kind"] == "attend":
        s["args"] = (_Operand(s["q"]), _Operand(s["out"]))
        return
    norm = lambda n: _Operand(s[n]) if n in s else None  # noqa: E731
    ld = (hq + 2 * hk) * hs
    s["how"] = ops.QkNormRope(head_size=hs, n_q_heads=hq, n_kv_heads=hk, variant=case["variant"], base_freq=BASE, eps=EPS, q_norm=norm("q_norm"),
                              k_norm=norm("k_norm"), q_ld=ld, k_ld=ld, v_ld=ld)
    q, k, v = _split(s)
    s["args"] = tuple(_Operand(t) for t in (q, k, v, s["q_out"], s["k_out"], s["pos"]))


def _split(s: dict):
    hq, hk, hs = s["case"]["heads"], s["case"]["kv_heads"], s["case"]["size"]
    q, k, v = s["qkv"].split([hq * hs, hk * hs, hk * hs], dim=1)
    return q, k, v


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s: dict):
    kind = s["case"]["kind"]
    if own:
        if kind == "norm":
            q, k, _, q_out, k_out, pos = s["args"]
            s["ctx"].qk_norm_rope(s["how"], pos, q, k, q_out, k_out)
            return s["q_out"], s["k_out"]
        if kind == "append":
            q, k, v, q_out, _, _ = s["args"]
            s["ctx"].paged_append(s["paged"], s["layer"], s["how"], q, k, v, q_out)
            return s["q_out"], s["keys"], s["values"]
        q, out = s["args"]
        s["ctx"].paged_attention(s["paged"], s["layer"], q, out)
        return s["out"]
    if kind == "attend":
        return _attend(s)
    q, k, v = _split(s)
    hs, cs = s["case"]["size"], _angles(s)
    q = _norm_rope(s, q.unflatten(1, (-1, hs)), s.get("q_norm"), cs)
    k = _norm_rope(s, k.unflatten(1, (-1, hs)), s.get("k_norm"), cs)
    if kind == "norm":
        return q, k
    page = s["case"]["page"]
    at, slot = s["table"][s["seq"], s["pos"] // page], s["pos"] % page
    _by_position(s, "keys")[at, slot] = k.to(s["keys"].dtype)
    _by_position(s, "values")[at, slot] = v.unflatten(1, (-1, hs)).to(s["values"].dtype)
    return q, s["keys"], s["values"]


def _by_position(s: dict, name: str) -> torch.Tensor:
    """The pages as [page][position][head][size], whatever their order in memory."""
    return s[name].transpose(1, 2) if s["case"]["order"] == "head" else s[name]


def _angles(s: dict):
    hs = s["case"]["size"]
    freq = BASE ** (-torch.arange(0, hs, 2, device="cuda", dtype=torch.float64) / hs)
    a = s["pos"].double()[:, None, None] * freq
    return torch.cos(a).float(), torch.sin(a).float()


def _norm_rope(s: dict, x: torch.Tensor, w, cs) -> torch.Tensor:
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    c, sn = cs
    if s["case"]["variant"] == 0:  # adjacent pairs
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * sn, a * sn + b * c), -1).flatten(-2)
    a, b = x.chunk(2, -1)          # element i with element i + size / 2
    return torch.cat((a * c - b * sn, a * sn + b * c), -1)


def _attend(s: dict) -> torch.Tensor:
    case, seq, inner = s["case"], s["seq"], s["inner"]
    hq, hk, hs, n = case["heads"], case["kv_heads"], case["size"], case["seqs"]
    group, most = hq // hk, s["most_pos"]
    gather = lambda name: _by_position(s, name)[s["table"]].flatten(1, 2)[:, :most].float().transpose(1, 2)  # noqa: E731  [seq][head][position][size]
    q = s["q"].new_zeros(n, s["most_new"], hk, group, hs)
    q[seq, inner] = s["q"].view(-1, hk, group, hs)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, hk, -1, hs)  # rows: (token, query head of the group)
    last = s["pos"].new_zeros(n, s["most_new"])
    last[seq, inner] = s["pos"]
    seen = torch.arange(most, device="cuda") <= last[..., None]  # [seq][token][position]
    scores = q @ gather("keys").transpose(2, 3) / hs**0.5
    scores = scores.view(n, hk, -1, group, most).masked_fill_(~seen[:, None, :, None], -torch.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    out = scores.view(n, hk, -1, most) @ gather("values") / scores.view(n, hk, -1, most).sum(-1, keepdim=True)
    return out.view(n, hk, -1, group, hs).permute(0, 2, 1, 3, 4)[seq, inner].reshape(-1, hq, hs)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case: dict) -> dict:
    hq, hk, hs, esz = case["heads"], case["kv_heads"], case["size"], 2 if case["kv"] == "f16" else 4
    pos0, n_new = _lengths(case)
    rows = sum(n_new)
    weights = 8.0 * hs if case["norms"] else 0.0
    each = 6.0 + (4.0 if case["norms"] else 0.0)  # operations an element: two products and a sum of a rotation's, an angle's share; the norm
    if case["kind"] == "norm":
        return {"bytes": 8.0 * rows * (hq + hk) * hs + 4.0 * rows + weights, "flops": each * rows * (hq + hk) * hs}
    if case["kind"] == "append":
        return {"bytes": rows * hs * (8.0 * hq + 2.0 * hk * (4 + esz)) + 4.0 * rows + weights, "flops": each * rows * (hq + hk) * hs}
    held = sum(p + n for p, n in zip(pos0, n_new))
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(pos0, n_new))  # (token, position it sees)
    return {"bytes": 8.0 * rows * hq * hs + 2.0 * held * hk * hs * esz + 4.0 * held / case["page"], "flops": 4.0 * pairs * hq * hs}


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------------
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    hq, hk, hs, page = case["heads"], case["kv_heads"], case["size"], case["page"]
    pos0, n_new = _lengths(case)
    head_first = case["order"] == "head"

    def held(name: str, b: int, upto: int) -> torch.Tensor:
        """Positions 0 .. upto of sequence b: [head][position][size]."""
        pages = [s[name][int(i)].double() for i in s["table"][b, : -(-upto // page)].tolist()]
        return torch.cat([p if head_first else p.permute(1, 0, 2) for p in pages], 1)[:, :upto]

    if case["kind"] == "attend":
        done, at = [], 0
        for b, (p, n) in enumerate(zip(pos0, n_new)):
            k, v = held("keys", b, p + n), held("values", b, p + n)
            q = s["q"][at : at + n].double()
            at += n
            out = torch.empty(n, hq, hs, dtype=torch.float64, device="cuda")
            where = torch.arange(p + n, device="cuda")[None, :] > p + torch.arange(n, device="cuda")[:, None]
            for h in range(hq):
                w = torch.softmax((q[:, h] @ k[h // (hq // hk)].T / np.sqrt(hs)).masked_fill(where, -torch.inf), 1)
                out[:, h] = w @ v[h // (hq // hk)]
            done.append(out)
        return torch.cat(done)
    j = torch.arange(hs // 2, dtype=torch.float64, device="cuda")
    turn = torch.exp(1j * s["pos"].double()[:, None] * torch.exp(j * (-2.0 / hs * np.log(BASE))))

    def rotated(x: torch.Tensor, w) -> torch.Tensor:
        x = x.double()
        if w is not None:
            x = w.double() * x / torch.sqrt(x.square().sum(2, keepdim=True) / hs + EPS)
        lo, hi = (slice(0, None, 2), slice(1, None, 2)) if case["variant"] == 0 else (slice(0, hs // 2), slice(hs // 2, None))
        z = torch.complex(x[..., lo], x[..., hi]) * turn[:, None]
        y = torch.empty_like(x)
        y[..., lo], y[..., hi] = z.real, z.imag
        return y

    qkv = s["qkv"].view(s["rows"], hq + 2 * hk, hs)
    q, k, v = rotated(qkv[:, :hq], s.get("q_norm")), rotated(qkv[:, hq : hq + hk], s.get("k_norm")), qkv[:, hq + hk :].double()
    if case["kind"] == "norm":
        return q, k
    keys, values = s["keys"].double(), s["values"].double()
    where, seqs = s["pos"].tolist(), s["seq"].tolist()
    table = s["table"].tolist()
    for r in range(s["rows"]):
        at = table[seqs[r]][where[r] // page], where[r] % page
        if head_first:
            keys[at[0], :, at[1]], values[at[0], :, at[1]] = k[r], v[r]
        else:
            keys[at[0], at[1]], values[at[0], at[1]] = k[r], v[r]
    return q, keys, values
