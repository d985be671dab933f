"""Paged attention over many tiles per wave: the tile loops in their steady
state, with a page per 16 keys, and the softmax reference moving at every
tile. The launch plan and the walk of each wave are restated here (and the
plan compared with the library's workspace size), so that the sizes below are
known to give what they are meant to.

Tolerance: as in test_gpu_paged_numerics.py, 2 (e + 2^-20 + n 2^-24) max|V|
and half an fp16 step, with n the keys of the longest walk and e the relative
error of an exponential, 1e-5; where scores reach 30 by one product in the last
32 elements, the sum over those is off by 32 * 30 * 2^-24 = 6e-5 more.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F16, PAGE = torch.float16, 16
OWN, SHARED, FEW, STREAM = range(4)
LOG2E, BELOW, MOVE = 1.4426950408889634, 6.0, 14.0


def _ceil(a, b):
    return -(-a // b)


def _plan(T, nH, nkv, hd, P, max_own, window):
    """(mode, prefix splits, own splits) of a launch."""
    grp, per_cu = nH // nkv, 1 if hd == 512 else 2
    places, kt, okt = 256 * per_cu, 32 if hd >= 256 else 64, 16 if hd >= 256 else 32

    def clamp(v, hi):
        return min(max(v, 1), max(min(hi, 256), 1))

    rows, nsp = T * grp, 0
    mode = OWN if not P else STREAM if rows <= 16 else FEW if rows <= 64 else SHARED
    if P:
        span = min(window, P) if window else P
        nrb = _ceil(rows, 128) if mode == SHARED else 1
        even = int(math.sqrt(50.0 * per_cu * span / (T * nH)))
        nsp = clamp(min(places // (nrb * nkv), even), _ceil(span, 2 * kt))
    span = min(window, max_own) if window else max_own
    items = T * nkv * _ceil(grp, 16)
    nso = clamp(min(4 * places // items, max(places // items, _ceil(span, 32 * okt))), _ceil(span, 4 * okt))
    return mode, nsp, nso


def _walks(lo, hi, hd, nsplit, shared):
    """Tiles [(first key, end)] of each wave that walks keys lo .. hi - 1 alone, or of each split of shared tiles."""
    n = (32 if hd >= 256 else 64) if shared else (16 if hd >= 256 else 32)
    waves = 1 if shared else 4
    b16 = lo & ~15
    per = waves * n * max(1, _ceil(hi - b16, waves * n * nsplit))
    out = []
    for split in range(nsplit):
        k0 = b16 + split * per
        k1 = min(k0 + per, hi)
        for w in range(waves):
            out.append([(t, min(t + n, k1)) for t in range(k0 + n * w, k1, waves * n)])
    return [w for w in out if w]


# form: (query heads, KV heads, rows, prefix by head dim, most own keys)
FORMS = {"own": (8, 4, 64, {}, 1300),
         "own_wide": (40, 4, 64, {}, 1300),
         "prefix_stream": (256, 32, 2, {64: 8300, 128: 8300, 256: 4500, 512: 2100}, 40),
         "prefix_64_rows": (128, 16, 8, {64: 9000, 128: 9000, 256: 2500, 512: 2100}, 40),
         "prefix_128_rows": (64, 8, 20, {64: 6000, 128: 6000, 256: 2600, 512: 2100}, 40)}
MODES = dict(prefix_stream=STREAM, prefix_64_rows=FEW, prefix_128_rows=SHARED, own=OWN, own_wide=OWN)


def _case(gpu, form, hd, seed, window, alike):
    """alike: all sequences have the same own pages and lengths."""
    nH, nkv, T, prefixes, most = FORMS[form]
    P = prefixes.get(hd, 0)
    rng = np.random.default_rng(seed)
    lens = [most] * T if alike else [most, *(int(n) for n in rng.integers(most // 2, most + 1, T - 1))]
    own, npre = _ceil(most, PAGE), _ceil(P, PAGE)
    pool = own if alike else max(own, 300 if not P else 40)
    deal = rng.permutation(npre + pool)
    pre, mine = deal[:npre], deal[npre:]
    table = np.stack([mine[:own] if alike else rng.choice(mine, own, replace=False) for _ in range(T)])
    mode, nsp, nso = _plan(T, nH, nkv, hd, P, own * PAGE, window)
    assert mode == MODES[form]
    ws = gpu.paged_attn_workspace(T, nH, nkv, hd, P, own * PAGE, window)
    np_ = nsp + nso
    assert (0 if ws is None else ws.numel()) == (T * nH * np_ * (hd + 2) * 4 if np_ > 1 else 0)
    pos = [P + n - 1 for n in lens]
    los = [max(0, p - window + 1) if window else 0 for p in pos]
    if P:
        walks = _walks(min(los), P, hd, nsp, mode != STREAM)
    else:
        walks = _walks(los[0], lens[0], hd, nso, False)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kc, vc = (torch.randn(npre + pool, nkv, PAGE, hd, device="cuda", generator=gen).to(F16) for _ in range(2))
    q = torch.randn(T, nH * hd, device="cuda", generator=gen) * hd ** -0.5
    return dict(nH=nH, nkv=nkv, hd=hd, T=T, P=P, lens=lens, pos=pos, los=los, window=window, pre=pre, table=table, kc=kc,
                vc=vc, q=q, walks=walks, own=own)


def _i(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _run(gpu, c):
    pre = dict(prefix_pages=_i(c["pre"]), prefix_len=_i([c["P"]]), max_prefix=c["P"]) if c["P"] else {}
    return gpu.paged_attn(c["q"], c["kc"], c["vc"], nH=c["nH"], table=_i(c["table"]), seq=_i(range(c["T"])), pos=_i(c["pos"]),
                          window=c["window"], **pre)


def _rows64(c, cache, t):
    """[nkv][keys][hd] of row t in 64 bits, its keys in order"""
    j = np.arange(c["los"][t], c["pos"][t] + 1)
    i = np.where(j < c["P"], j, j - c["P"])
    pg = np.where(j < c["P"], np.concatenate([c["pre"], [0]])[np.minimum(i // PAGE, len(c["pre"]))],
                  c["table"][t][np.minimum(i // PAGE, c["own"] - 1)])
    return cache[torch.as_tensor(pg, device="cuda"), :, torch.as_tensor(i % PAGE, device="cuda")].double().transpose(0, 1).contiguous()


def _scores64(c, t):
    q = c["q"][t].double().view(c["nkv"], -1, c["hd"])
    return torch.matmul(q, _rows64(c, c["kc"], t).transpose(1, 2).contiguous())


def _check(c, out, e):
    n = max(sum(b - a for a, b in w) for w in c["walks"])
    vmax = float(c["vc"].abs().max())
    bound = 2 * (e + 2.0 ** -20 + n * 2.0 ** -24) * vmax
    for t in range(c["T"]):
        p = torch.softmax(_scores64(c, t), -1)
        ref = torch.matmul(p, _rows64(c, c["vc"], t)).flatten()
        off = (out[t].double() - ref).abs() - (ref.abs() * 2.0 ** -11 + 2.0 ** -25 + bound)
        assert float(off.max()) <= 0, (t, float(off.max()), bound)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("windowed", [False, True])
def test_many_tiles_per_wave(gpu, form, hd, windowed):
    P, most = FORMS[form][3].get(hd, 0), FORMS[form][4]
    # a window that begins inside a tile, near the start
    c = _case(gpu, form, hd, 7 * hd + windowed, P + most - 37 if windowed else 0, False)
    assert max(len(w) for w in c["walks"]) >= 4, [len(w) for w in c["walks"]]
    c["q"] = (c["q"] * 1.5).to(F16)
    _check(c, _run(gpu, c), 1e-5)


def _moves(c, t):
    """Moves of the reference of row t's first head of each KV head behind the first tile of its walks, and walks of
    more than one tile."""
    s = _scores64(c, t)[:, 0].cpu().numpy() * LOG2E
    moves = walks = 0
    for w in c["walks"]:
        ref = np.full(len(s), -np.inf)
        for a, b in w:
            top = s[:, a:b].max(1)
            move = (top > ref + MOVE) | np.isneginf(ref)
            moves += int((move & np.isfinite(ref)).sum())
            ref = np.where(move, top - BELOW, ref)
        walks += len(w) > 1
    return moves, walks


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("form", FORMS)
def test_reference_moves_at_every_tile(gpu, form, hd):
    """Scores rise by 6 from each tile of a wave to its next one: 8.7 in log2
    units, past the 8 at which the reference moves, so that the tile before
    still has 1/400 of the weight; its values are far from this one's."""
    c = _case(gpu, form, hd, 9 * hd, 0, True)
    pages, keys = (c["pre"], c["P"]) if c["P"] else (c["table"][0], c["lens"][0])
    level, side = np.zeros(keys), np.zeros(keys)
    for w in c["walks"]:
        for i, (a, b) in enumerate(w):
            level[a:b], side[a:b] = 6.0 * (i - len(w) // 2), 4.0 * (-1) ** i
    assert np.abs(level).max() <= 30
    pg = torch.as_tensor(pages[np.arange(keys) // PAGE], device="cuda")
    sl = torch.as_tensor(np.arange(keys) % PAGE, device="cuda")
    kc, vc = c["kc"], c["vc"]
    kc[..., -1] = -30.0
    kc[pg, :, sl, -1] = torch.as_tensor(level, device="cuda")[:, None].expand(-1, c["nkv"]).to(F16)
    vc[pg, :, sl] += torch.as_tensor(side, device="cuda")[:, None, None].to(F16)
    q = (c["q"] * 0.1).view(c["T"], c["nH"], hd)
    q[..., -1] = 1.0
    c["q"] = q.view(c["T"], -1).to(F16)
    tiles = sum(len(w) - 1 for w in c["walks"])
    moves, walks = _moves(c, 0)
    assert walks and moves == tiles * c["nkv"], (moves, tiles, c["nkv"])
    _check(c, _run(gpu, c), 1e-5 + 6e-5)
