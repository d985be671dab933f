"""Precision of paged attention (paged_attn), in each of its forms: own pages
with up to 8 query heads per KV head and with more, and a prefix with few,
some and many query rows per KV head.

Tolerances. A softmax weight is held as two fp16 values, to 2^-20 of itself;
the score and its exponential are off by 1e-5 relative of the weight for
|score differences| up to 30; a wave adds n keys' products, and as many
weights, in fp32: n * 2^-24 at most. So the quotient of the two sums is off by
2 (1e-5 + 2^-20 + n 2^-24) max|V| at most, with n up to 128 here 4e-5 max|V|,
before its rounding to fp16, half a step: 2^-11 of the value (2^-25 in the
subnormals).
"""
import numpy as np
import pytest

from oracle import paged_oracle as G
from test_gpu_paged import _attn_case, _i, _np, _run_attn

pytestmark = pytest.mark.gpu

# form: (query heads, KV heads, prefix, own keys of each row)
FORMS = {"own": (8, 4, 0, [1, 5, 40, 200, 33, 64]),
         "own_wide": (20, 1, 0, [1, 5, 40, 200, 33, 64]),
         "prefix_stream": (8, 4, 300, [1, 2, 5]),
         "prefix_64_rows": (16, 2, 300, [1, 2, 5, 30, 7]),
         "prefix_128_rows": (16, 2, 300, [1 + i for i in range(12)])}


def _case(form, hd, seed, **kw):
    nH, nkv, P, lens = FORMS[form]
    return _attn_case(seed + hd, nH, nkv, hd, 32, P, lens, 0, 0, **kw)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("form", FORMS)
def test_equal_values_come_out_unchanged(gpu, form, hd):
    """The output is a mean of V rows under weights that sum to one: where all
    keys have one V row it is that row, whatever the weights, since less than
    2^-12 relative is lost before the rounding to fp16. Scores of a spread
    that leaves most of a row's weight to a few keys."""
    c = _case(form, hd, 40, spread=4.0, poison=False)
    nkv = c["kc"].shape[1]
    v = np.random.default_rng(hd).standard_normal((nkv, hd)).astype(np.float16)
    c["vc"][:] = v[None, :, None, :]
    got = _np(_run_attn(gpu, c)).reshape(len(c["q"]), nkv, c["nH"] // nkv, hd)
    off = got != v[None, :, None, :]
    assert not off.any(), f"{int(off.sum())} of {off.size} values off"


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("spread", [1.5, 4.0])
def test_weights_keep_their_low_bits(gpu, form, hd, spread):
    c = _case(form, hd, 50, spread=spread)
    got = _np(_run_attn(gpu, c)).astype(np.float64)
    ref = np.stack(G.paged_attn_ref(c["q"], c["kc"], c["vc"], nH=c["nH"], table=c["table"], seq=c["seq"], pos=c["pos"],
                                    P=c["P"], prefix_pages=c["pre"]))
    vmax = float(np.abs(c["vc"][np.isfinite(c["vc"])]).max())
    off = np.abs(got - ref) - (np.abs(ref) * 2.0 ** -11 + 2.0 ** -25 + 4e-5 * vmax)
    assert (off <= 0).all(), (int((off > 0).sum()), off.max())


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("P", [0, 200])
def test_positions_far_past_the_own_keys(gpu, hd, P):
    """Windows that begin up to 2^31 - 1, in every split of the own keys: such
    a row has no keys and gives zeros; its neighbours keep theirs."""
    c = _attn_case(hd + P, 8, 4, hd, 16, P, [700, 3, 64, 1, 1, 1], 0, 0, poison=False)
    for window in (1, 64, 1024):
        c.update(window=window, pos=[P + 699, 2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 1500, P, 2 ** 31 - 30000])
        got = _np(_run_attn(gpu, c)).astype(np.float64)
        max_own = 16 * c["table"].shape[1]
        assert not got[[1, 2, 3, 5]].any()
        ref = G.paged_attn_ref(c["q"], c["kc"], c["vc"], nH=8, table=c["table"], seq=c["seq"], pos=c["pos"], P=P,
                               prefix_pages=c["pre"], window=window, max_own=max_own)
        for t in (0, 4):
            off = np.abs(got[t] - ref[t]) - (np.abs(ref[t]) * 2.0 ** -11 + 2.0 ** -25 + 4e-5 * np.abs(c["vc"]).max())
            assert (off <= 0).all(), (t, window, off.max())


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("form", [*FORMS, "own_one_part"])
def test_nonfinite_queries_give_nan(gpu, form, hd):
    """A query head with a NaN or an Inf has no finite score, so that its
    softmax is NaN in fp32 arithmetic, however the keys are split; all others
    keep their bits. An Inf times negative keys alone (all scores -inf) and one
    times a 0 (a NaN score) are among them."""
    if form == "own_one_part":
        c = _attn_case(60 + hd, 8, 4, hd, 32, 0, [1, 5, 30, 64], 0, 0, poison=False)
        assert gpu.paged_attn_workspace(4, 8, 4, hd, 0, 64) is None
    else:
        c = _case(form, hd, 60, poison=False)
    c["kc"][..., 1] = -np.abs(c["kc"][..., 1]) - 1
    c["kc"][..., 2] = 0
    want = _np(_run_attn(gpu, c)).copy()
    T, nH = len(c["q"]), c["nH"]
    hit = np.zeros((T, nH, hd), bool)
    q = c["q"].reshape(T, nH, hd)
    for i, (e, x) in enumerate([(0, np.nan), (hd - 1, np.inf), (hd // 2 + 3, -np.inf), (1, np.inf), (1, -np.inf), (2, np.inf),
                                (hd // 2 + 9, np.nan)]):
        t, h = i * 5 % T, (3 * i + 1) % nH
        q[t, h, e] = x
        hit[t, h] = True
    got = _np(_run_attn(gpu, c))
    hit = hit.reshape(T, -1)
    assert np.isnan(got[hit]).all()
    assert (got[~hit] == want[~hit]).all()


def test_nonfinite_queries_without_keys_give_zeros(gpu):
    c = _attn_case(71, 16, 8, 256, 16, 40, [40, 20, 5], 0, 0, poison=False)
    c["table"][1, :] = -1
    c["pre"][:] = -1
    c["q"][1, 3], c["q"][1, 300] = np.nan, np.inf
    assert not _np(_run_attn(gpu, c))[1].any()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("form", [f for f in FORMS if FORMS[f][2]])
@pytest.mark.parametrize("window", [0, 120])
def test_prefix_longer_than_its_bound(gpu, form, hd, window):
    """prefix_len divides the positions for the append and for attention
    alike: past max_prefix its keys are left out, and own keys stay where
    they are."""
    c = _case(form, hd, 80, poison=False)
    c["window"] = window
    bound = 150     # of 300 positions: the fifth page in part
    got = _np(_run_attn(gpu, dict(c, pre=c["pre"][:5]), max_prefix=bound)).astype(np.float64)
    nkv, page = c["kc"].shape[1:3]
    grp = c["nH"] // nkv
    for t in range(len(c["q"])):
        p = c["pos"][t]
        keys = [j for j in range(max(0, p - window + 1) if window else 0, p + 1) if j < bound or j >= c["P"]]
        pg, sl = np.array([G.slot(j, t, c["P"], c["table"], c["pre"], page, len(c["kc"])) for j in keys]).T
        for h in range(c["nH"]):
            sc = c["kc"][pg, h // grp, sl].astype(np.float64) @ c["q"][t, h * hd:(h + 1) * hd].astype(np.float64)
            e = np.exp(sc - sc.max())
            r = (e @ c["vc"][pg, h // grp, sl].astype(np.float64)) / e.sum()
            off = np.abs(got[t, h * hd:(h + 1) * hd] - r) - (np.abs(r) * 2.0 ** -11 + 2.0 ** -25 +
                                                             4e-5 * np.abs(c["vc"]).max())
            assert (off <= 0).all(), (t, h, off.max())


def test_prefix_length_of_any_value(gpu):
    """Lengths up to 2^31 - 1 with the default bound, the 128 positions that the
    prefix's pages hold: rows inside the prefix keep the keys below it."""
    c = _attn_case(90, 16, 8, 256, 32, 100, [1, 2, 3, 4], 0, 0, poison=False)
    for n in (2 ** 31 - 1, 2 ** 31 - 200, -5):
        for window in (0, 30):
            c.update(window=window, pos=[5, 99, 130, 2 ** 31 - 1])
            got = _np(_run_attn(gpu, c, prefix_len=_i([n]), max_own=32)).astype(np.float64)
            P = max(n, 0)
            for t, p in enumerate(c["pos"]):
                # own keys from P on, of which there are 32
                near = [j for j in range(0, 128) if j < P and j <= p and (not window or j > p - window)]
                near += [j for j in range(P, P + 32) if j <= p and (not window or j > p - window)]
                r = np.zeros(16 * 256)
                if near:
                    pg, sl = np.array([G.slot(j, t, P, c["table"], c["pre"], 32, len(c["kc"])) for j in near]).T
                    for h in range(16):
                        sc = c["kc"][pg, h // 2, sl].astype(np.float64) @ c["q"][t, h * 256:(h + 1) * 256].astype(np.float64)
                        e = np.exp(sc - sc.max())
                        r[h * 256:(h + 1) * 256] = (e @ c["vc"][pg, h // 2, sl].astype(np.float64)) / e.sum()
                off = np.abs(got[t] - r) - (np.abs(r) * 2.0 ** -11 + 2.0 ** -25 + 4e-5 * np.abs(c["vc"]).max())
                assert (off <= 0).all(), (n, window, t, off.max())
