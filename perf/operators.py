"""Performance cases of the batched operators, through their public entry points.

A batch of sequences decoded together on int8 weights runs, per layer: the
residual normadd and rmsnorm whose rows leave as int8 with a scale each (the
W8A8 GEMM's input), the preparation of q, k and v with the append to a paged
cache, and attention over a prefix that all sequences share and each one's own
pages. Each operator stands here in its plain form too: elementary torch
operations in 32 bits, rounded once at the end.

The shapes are the ones this repository's engine, tests and benchmark use:
hidden 3840; five of six layers attend the last 1024 positions (16 query and 8
KV heads of 256), every sixth attends everything (16 query heads and one k == v
head of 512); two generic grouped layouts stand beside them.

Kinds (``case["kind"]``):

- ``norm``: rows through rmsnorm (``add``: behind the residual normadd) into
  int8 values and row scales.
- ``append``: q/k/v rows of ``seqs`` sequences, ``per`` tokens each, into
  prepared q rows and the paged cache.
- ``attn``: one token of each of ``seqs`` sequences over a shared prefix of
  ``prefix`` tokens and up to ``own`` tokens of its own.
"""
import math

import torch

own = False

H = 3840
EPS = 1e-6
LAYER_SCALE = 0.75
F16, F32, F64, I32 = torch.float16, torch.float32, torch.float64, torch.int32
SLIDING = dict(nH=16, nkv=8, hd=256)
GLOBAL = dict(nH=16, nkv=1, hd=512)
GROUPED = dict(nH=32, nkv=8, hd=128)
SMALL = dict(nH=8, nkv=2, hd=64)


def listed():
    return [
        # one decoded token between two int8 products: launch and latency are most of it
        dict(name="norm_token", kind="norm", M=1, D=H, add=True, half=True),
        # a prefill chunk's rows between the o projection and the gate/up products
        dict(name="norm_chunk_128", kind="norm", M=128, D=H, add=True, half=True),
        # a long batch of rows on the int8 prefill route
        dict(name="norm_rows_2048", kind="norm", M=2048, D=H, add=True, half=True),
        # the first norm of a layer stack alone, rows of an odd length in fp32
        dict(name="norm_odd_first", kind="norm", M=333, D=5001, add=False, half=False),
        # one sequence's token in a sliding layer, fp32 projections as the decode GEMV writes them
        dict(name="append_token", kind="append", seqs=1, per=1, start=400, prefix=0, page=32, keqv=False, half=False,
             pad=0, **SLIDING),
        # a decoded batch behind a shared prompt, its last rows padding
        dict(name="append_batch_61", kind="append", seqs=61, per=1, start=180, prefix=1999, page=32, keqv=False,
             half=True, pad=3, **SLIDING),
        # prompt chunks of several sequences in a k == v layer
        dict(name="append_chunks_global", kind="append", seqs=16, per=128, start=300, prefix=0, page=64, keqv=True,
             half=True, pad=0, **GLOBAL),
        # one sequence alone in a sliding layer, no prefix: latency
        dict(name="attn_single", kind="attn", seqs=1, prefix=0, own=700, window=1024, page=32, pad=0, **SLIDING),
        # a batch behind a common system prompt in a sliding layer, near the prompt's end
        dict(name="attn_batch_sliding", kind="attn", seqs=16, prefix=2000, own=500, window=1024, page=32, pad=2,
             **SLIDING),
        # a full batch in a global layer: a long shared document, answers of ragged length
        dict(name="attn_batch_global", kind="attn", seqs=64, prefix=8192, own=1000, window=0, page=64, pad=0, **GLOBAL),
        # nothing shared: long conversations of ragged length
        dict(name="attn_ragged_own", kind="attn", seqs=32, prefix=0, own=4096, window=0, page=16, pad=0, **GROUPED),
        # a few questions about one very long document
        dict(name="attn_long_prefix", kind="attn", seqs=8, prefix=32001, own=150, window=0, page=128, pad=0,
             **GROUPED),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0), _cost(c))
    kind = rng.choice(["norm", "append", "attn", "attn"])
    while True:
        if kind == "norm":
            add = rng.random() < 0.7
            D = rng.choice([H, _log(rng, 200, 16000), _log(rng, 25, 2000) * 8])
            c = dict(kind=kind, M=_log(rng, 1, 2048), D=D, add=add, half=add and rng.random() < 0.7)
        elif kind == "append":
            heads = rng.choice([SLIDING, GLOBAL, GROUPED, SMALL])
            per = rng.choice([1, 1, _log(rng, 2, 300)])
            c = dict(kind=kind, seqs=_log(rng, 1, 64), per=per, start=_log(rng, 1, 400),
                     prefix=rng.choice([0, _log(rng, 10, 5000)]), page=rng.choice([16, 32, 64, 128]),
                     keqv=rng.random() < 0.3, half=rng.random() < 0.7, pad=rng.choice([0, 0, 5]), **heads)
        else:
            heads = rng.choice([SLIDING, SLIDING, GLOBAL, GLOBAL, GROUPED, SMALL])
            c = dict(kind=kind, seqs=_log(rng, 1, 64), prefix=rng.choice([0, _log(rng, 20, 32000), _log(rng, 500, 32000)]),
                     own=_log(rng, 1, 4096), window=rng.choice([0, 0, 1024]), page=rng.choice([16, 32, 64, 128]),
                     pad=rng.choice([0, 0, 3]), **heads)
        if _cost(c) <= most[kind] and _pool(c) <= 600e6:
            return c


def _spread(n, most):
    """n whole numbers in 1 .. most, spread evenly, the first one the largest."""
    return [max(1, int(round(most * (1.0 - (i * 0.6180339887498949) % 1.0)))) for i in range(n)]


def _pages(case):
    """Own pages of each sequence."""
    if case["kind"] == "append":
        return [-(-(s + case["per"]) // case["page"]) for s in _spread(case["seqs"], case["start"])]
    return [-(-n // case["page"]) for n in _spread(case["seqs"], case["own"])]


def _pool(case):
    """Values of one cache (K or V)."""
    if case["kind"] == "norm":
        return 0
    n = sum(_pages(case)) + (-(-case["prefix"] // case["page"]) if case["kind"] == "attn" else 0)
    return n * case["page"] * case["nkv"] * case["hd"]


def _spans(case):
    """(first key, keys) of each live row of an attention case, and where the rows' prefix keys begin."""
    rows = []
    for n in _spread(case["seqs"], case["own"]):
        pos = case["prefix"] + n - 1
        lo = max(0, pos - case["window"] + 1) if case["window"] else 0
        rows.append((lo, pos + 1 - lo, n))
    return rows, min(min(r[0] for r in rows), case["prefix"])


def work(case):
    if case["kind"] == "norm":
        M, D = case["M"], case["D"]
        e = 2 if case["half"] else 4
        return {"bytes": M * (D * (e + 1 + (8 if case["add"] else 0)) + 4) + D * (8 if case["add"] else 4),
                "flops": M * D * (12 if case["add"] else 7)}
    if case["kind"] == "append":
        T, e = case["seqs"] * case["per"], 2 if case["half"] else 4
        nq, nk = case["nH"] * case["hd"], case["nkv"] * case["hd"]
        rows = T * (e * (nq + nk * (1 if case["keqv"] else 2)) + 2 * (nq + 2 * nk))
        return {"bytes": rows + case["seqs"] * case["per"] * 8 * case["hd"] + 12 * T, "flops": T * (8 * nq + 12 * nk)}
    rows, first = _spans(case)
    nq, nk = case["nH"] * case["hd"], case["nkv"] * case["hd"]
    keys = case["prefix"] - first + sum(min(k, n) for _lo, k, n in rows)
    return {"bytes": 4 * nk * keys + 4 * nq * len(rows), "flops": 4 * nq * sum(k for _lo, k, _n in rows)}


# ---- inputs -----------------------------------------------------------------
def _rand(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _weight(gen, n, scale=1.0):
    return (torch.rand(n, device="cuda", generator=gen) + 0.5) * scale


def _ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def _rope_tables(n, hd):
    ang = torch.arange(n, device="cuda", dtype=F64)[:, None] / 10000.0 ** (
        torch.arange(0, hd, 2, device="cuda", dtype=F64) / hd)[None]
    ang = torch.cat([ang, ang], 1)
    return torch.cos(ang).to(F32).contiguous(), torch.sin(ang).to(F32).contiguous()


def _table(case, gen):
    """Pages dealt at random: (prefix pages, the sequences' tables [seqs][most], pages in the cache)."""
    counts = _pages(case)
    npre = -(-case["prefix"] // case["page"]) if case["kind"] == "attn" else 0
    total = sum(counts) + npre
    deal = torch.randperm(total, device="cuda", generator=gen).to(I32)
    table = torch.full((len(counts), max(counts)), -1, dtype=I32, device="cuda")
    at = npre
    for s, n in enumerate(counts):
        table[s, :n] = deal[at: at + n]
        at += n
    return deal[:npre].contiguous(), table, total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    return globals()["_prepare_" + case["kind"]](case, gen)


def _prepare_norm(case, gen):
    M, D = case["M"], case["D"]
    s = dict(case=case, w=_weight(gen, D, 0.3 if case["add"] else 1.0), x=_rand(gen, M, D) * 2.0)
    # a few loud channels, as residual streams have them
    s["x"][:, :: max(1, D // 7)] *= 8.0
    if case["half"]:
        s["x"] = s["x"].to(F16)
    if case["add"]:
        s.update(h=_rand(gen, M, D), w2=_weight(gen, D))
    s.update(A=torch.empty(M, D, dtype=torch.int8, device="cuda"), sa=torch.empty(M, device="cuda"),
             values=torch.empty(M, D, dtype=F16, device="cuda"))
    return s


def _prepare_append(case, gen):
    nq, nk, hd, per = case["nH"] * case["hd"], case["nkv"] * case["hd"], case["hd"], case["per"]
    starts = _spread(case["seqs"], case["start"])
    _none, table, total = _table(case, gen)
    seq = [s for s in range(case["seqs"]) for _ in range(per)] + [-1] * case["pad"]
    pos = [case["prefix"] + b + i for b in starts for i in range(per)] + [0] * case["pad"]
    T, ld = len(seq), nq + nk * (1 if case["keqv"] else 2)
    cos, sin = _rope_tables(case["prefix"] + max(starts) + per, hd)
    qkv = _rand(gen, T, ld) * 1.7
    shape = (total, case["nkv"], case["page"], hd)
    return dict(case=case, n=case["seqs"] * per, qkv=qkv.to(F16) if case["half"] else qkv,
                qnw=_weight(gen, hd, hd ** -0.5), knw=_weight(gen, hd), cos=cos, sin=sin,
                kc=_rand(gen, *shape).to(F16), vc=_rand(gen, *shape).to(F16), table=table, seq=_ints(seq),
                pos=_ints(pos), prefix_len=_ints([case["prefix"]]), q=torch.zeros(T, nq, dtype=F16, device="cuda"))


def _prepare_attn(case, gen):
    hd = case["hd"]
    lens = _spread(case["seqs"], case["own"])
    prefix_pages, table, total = _table(case, gen)
    T = case["seqs"] + case["pad"]
    shape = (total, case["nkv"], case["page"], hd)
    # prepared q rows: scores of a spread that lets some keys stand out
    q = (_rand(gen, T, case["nH"] * hd) * (1.5 * hd ** -0.5)).to(F16)
    return dict(case=case, n=case["seqs"], q=q, kc=_rand(gen, *shape).to(F16), vc=_rand(gen, *shape).to(F16),
                table=table, prefix_pages=prefix_pages, prefix_len=_ints([case["prefix"]]),
                seq=_ints(list(range(case["seqs"])) + [-1] * case["pad"]),
                pos=_ints([case["prefix"] + n - 1 for n in lens] + [0] * case["pad"]),
                out=torch.zeros(T, case["nH"] * hd, dtype=F16, device="cuda"))


# ---- one pass ---------------------------------------------------------------
def _ops():
    import importlib
    return importlib.import_module("gemma4-12b-snapdragonx2elite_amd.ops")


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "append": _own_append, "attn": _own_attn}[kind](state)
    return {"norm": _plain_norm, "append": _plain_append, "attn": _plain_attn}[kind](state)


def _own_norm(s):
    ops, c = _ops(), s["case"]
    if c["add"]:
        ops.pre_normadd_i8(s["x"], s["w"], s["h"], s["w2"], s["A"], s["sa"], M=c["M"], D=c["D"], scale=LAYER_SCALE)
    else:
        ops.pre_rmsnorm_i8(s["x"], s["w"], s["A"], s["sa"], M=c["M"], D=c["D"])
    torch.mul(s["A"], s["sa"][:, None], out=s["values"])  # what the 8-bit values stand for
    return [s["values"], s["sa"]] + ([s["h"]] if c["add"] else [])


def _own_append(s):
    ops, c = _ops(), s["case"]
    nq, nk = c["nH"] * c["hd"], c["nkv"] * c["hd"]
    ops.paged_prep(s["qkv"], s["qnw"], s["knw"], s["cos"], s["sin"], s["kc"], s["vc"], s["q"], nH=c["nH"], koff=nq,
                   voff=nq if c["keqv"] else nq + nk, table=s["table"], seq=s["seq"], pos=s["pos"],
                   prefix_len=s["prefix_len"])
    return [s["q"], s["kc"], s["vc"]]


def _own_attn(s):
    ops, c = _ops(), s["case"]
    kw = dict(max_prefix=c["prefix"], max_own=c["own"], window=c["window"])
    if "ws" not in s:  # kept for the next pass, as a decode loop keeps it
        s["ws"] = ops.paged_attn_workspace(c["seqs"] + c["pad"], c["nH"], c["nkv"], c["hd"], **kw)
    ops.paged_attn(s["q"], s["kc"], s["vc"], s["out"], nH=c["nH"], table=s["table"], seq=s["seq"], pos=s["pos"],
                   prefix_pages=s["prefix_pages"] if c["prefix"] else None,
                   prefix_len=s["prefix_len"] if c["prefix"] else None, ws=s["ws"], **kw)
    return s["out"]


def _rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _plain_norm(s):
    if s["case"]["add"]:
        s["h"].copy_((s["h"] + _rms(s["x"].float()) * s["w"]) * LAYER_SCALE)
        y = _rms(s["h"]) * s["w2"]
    else:
        y = _rms(s["x"].float()) * s["w"]
    sa = (y.abs().amax(-1) / 127.0).clamp(min=1e-12)
    A = torch.round(y / sa[:, None]).clamp(-127.0, 127.0)
    return [(A * sa[:, None]).to(F16), sa] + ([s["h"]] if s["case"]["add"] else [])


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return x * cos[:, None] + torch.cat([-b, a], -1) * sin[:, None]


def _plain_append(s):
    c, n = s["case"], s["n"]
    hd, nH, nkv, page = c["hd"], c["nH"], c["nkv"], c["page"]
    x = s["qkv"][:n].float().view(n, -1, hd)
    q, k, v = x[:, :nH], x[:, nH: nH + nkv], x[:, nH: nH + nkv] if c["keqv"] else x[:, nH + nkv:]
    pos, seq = s["pos"][:n].long(), s["seq"][:n].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    i = pos - s["prefix_len"].long()
    at = s["table"][seq, i // page].long()
    s["q"][:n] = _rotate(_rms(q) * s["qnw"], cos, sin).to(F16).view(n, -1)
    s["kc"][at, :, i % page] = _rotate(_rms(k) * s["knw"], cos, sin).to(F16)
    s["vc"][at, :, i % page] = _rms(v).to(F16)
    return [s["q"], s["kc"], s["vc"]]


def _plain_attn(s):
    c, n = s["case"], s["n"]
    hd, nkv, P, page = c["hd"], c["nkv"], c["prefix"], c["page"]
    grp = c["nH"] // nkv
    q = s["q"][:n].float().view(n, nkv, grp, hd)
    # the prefix, gathered once: [nkv][P][hd]; every sequence's own pages: [n][nkv][L][hd]
    pre = s["prefix_pages"].long()
    kp = s["kc"][pre].float().transpose(0, 1).reshape(nkv, pre.numel() * page, hd)[:, :P]
    vp = s["vc"][pre].float().transpose(0, 1).reshape(nkv, pre.numel() * page, hd)[:, :P]
    tab = s["table"][s["seq"][:n].long()].clamp(min=0).long()
    ko = s["kc"][tab].float().transpose(1, 2).reshape(n, nkv, -1, hd)
    vo = s["vc"][tab].float().transpose(1, 2).reshape(n, nkv, -1, hd)
    L = ko.shape[2]
    qp = q.transpose(0, 1).reshape(nkv, n * grp, hd)
    sp = torch.matmul(qp, kp.transpose(1, 2).contiguous()).view(nkv, n, grp, P).transpose(0, 1)
    so = torch.matmul(q, ko.transpose(2, 3).contiguous())
    key = torch.cat([torch.arange(P, device="cuda"), P + torch.arange(L, device="cuda")])
    pos = s["pos"][:n, None].long()
    live = key[None] <= pos
    if c["window"]:
        live = live & (key[None] > pos - c["window"])
    sc = torch.cat([sp, so], -1).masked_fill(~live[:, None, None], -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    pp = p[..., :P].transpose(0, 1).reshape(nkv, n * grp, P)
    o = torch.matmul(pp, vp.contiguous()).view(nkv, n, grp, hd).transpose(0, 1) + \
        torch.matmul(p[..., P:].contiguous(), vo)
    s["out"][:n] = o.reshape(n, -1).to(F16)
    return s["out"]


# ---- the definition in 64 bits ----------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attn": _exact_attn}[case["kind"]](case, s)


def _exact_rows(x, w):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w


def _exact_norm(case, s):
    y = _exact_rows(s["x"].double(), s["w"].double())
    h = None
    if case["add"]:
        h = (s["h"].double() + y) * LAYER_SCALE
        y = _exact_rows(h, s["w2"].double())
    sa = torch.clamp(y.abs().max(-1).values / 127.0, min=1e-12)
    values = torch.clamp(torch.round(y / sa[:, None]), -127, 127) * sa[:, None]
    return [values, sa] + ([h] if case["add"] else [])


def _exact_append(case, s):
    hd, nH, nkv, page, n = case["hd"], case["nH"], case["nkv"], case["page"], s["n"]
    x = s["qkv"].double()
    q, kc, vc = s["q"].double(), s["kc"].double(), s["vc"].double()
    half = hd // 2
    pos = s["pos"].tolist()
    seq = s["seq"].tolist()
    table = s["table"].tolist()
    at = [(table[seq[t]][(pos[t] - case["prefix"]) // page], (pos[t] - case["prefix"]) % page) for t in range(n)]
    pages = torch.tensor([a for a, _ in at], device="cuda")
    slots = torch.tensor([b for _, b in at], device="cuda")
    cos, sin = s["cos"].double()[s["pos"][:n].long()], s["sin"].double()[s["pos"][:n].long()]

    def turned(rows):
        out = rows * cos
        out[:, :half] -= rows[:, half:] * sin[:, :half]
        out[:, half:] += rows[:, :half] * sin[:, half:]
        return out

    one = torch.ones(hd, dtype=F64, device="cuda")
    for h in range(nH):
        q[:n, h * hd: (h + 1) * hd] = turned(_exact_rows(x[:n, h * hd: (h + 1) * hd], s["qnw"].double()))
    for h in range(nkv):
        k0 = (nH + h) * hd
        v0 = k0 if case["keqv"] else k0 + nkv * hd
        kc[pages, h, slots] = turned(_exact_rows(x[:n, k0: k0 + hd], s["knw"].double()))
        vc[pages, h, slots] = _exact_rows(x[:n, v0: v0 + hd], one)
    return [q, kc, vc]


def _exact_attn(case, s):
    hd, nkv, grp, P, page = case["hd"], case["nkv"], case["nH"] // case["nkv"], case["prefix"], case["page"]
    out = s["out"].double()
    pre = s["prefix_pages"].long()
    for t, n in enumerate(_spread(case["seqs"], case["own"])):
        pos = P + n - 1
        lo = max(0, pos - case["window"] + 1) if case["window"] else 0
        mine = s["table"][t, : -(-n // page)].long()
        for g in range(nkv):
            def rows(cache):
                shared = cache[pre, g].reshape(-1, hd)[min(lo, P): P]
                return torch.cat([shared, cache[mine, g].reshape(-1, hd)[max(0, lo - P): n]]).double()
            q = s["q"][t].double().view(nkv, grp, hd)[g]
            sc = q @ rows(s["kc"]).T
            e = torch.exp(sc - sc.max(1, keepdim=True).values)
            out[t].view(nkv, grp, hd)[g] = (e @ rows(s["vc"])) / e.sum(1, keepdim=True)
    return out
