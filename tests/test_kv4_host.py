"""Paged 4-bit KV cache, without a GPU: the oracle's own properties, the rotary
table against its formula, and refusals that need no launch."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import kv4


def test_quantise_holds_values_to_half_a_step():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 128)).astype(np.float32) * np.exp(rng.standard_normal((50, 1)) * 3)
    codes, scales = kv4.quantise(x.astype(np.float32))
    held = kv4.values(codes, scales)
    # half a step, plus what the fp16 scale may fall short of amax / 7 (2^-11 of 7 steps)
    step = np.repeat(scales.astype(np.float64), 32, -1)
    assert (np.abs(held - x) <= step * (0.5 + 7 * 2.0 ** -11)).all()
    again = kv4.quantise(held)
    assert np.array_equal(again[0], codes) and np.array_equal(again[1], scales)


def test_quantise_edges():
    x = np.zeros((4, 64), np.float32)
    x[1, :] = 1e-9            # a scale below fp16's range is 0
    x[2, 3] = np.nan
    x[3, 40] = 1e6            # a scale above it saturates
    codes, scales = kv4.quantise(x)
    assert not codes[0].any() and not scales[0].any()
    assert not codes[1].any() and not scales[1].any()
    assert np.isnan(scales[2, 0]) and scales[2, 1] == 0 and not codes[2].any()
    assert scales[3, 1] == 65504 and codes[3, 40] == 7


@pytest.mark.parametrize("seed", range(4))
def test_bounds_do_not_depend_on_the_split(seed):
    """Folding tokens in one at a time, by shifts of the held int8, gives the page's bounds."""
    rng = np.random.default_rng(seed)
    held = (rng.standard_normal((40, 64)) * np.exp(2 * rng.standard_normal((40, 1)))).astype(np.float32)
    held = kv4.values(*kv4.quantise(held))
    want, e_want = kv4.bounds(held)
    got, e = kv4.bounds(held[:1])
    for t in range(1, len(held)):
        new, e1 = kv4.bounds(held[t:t + 1])
        e2 = max(e, e1)
        x = held[t].astype(np.float64) * 2.0 ** -e2
        lo = np.minimum(got[0].astype(int) >> (e2 - e), np.floor(x))
        hi = np.maximum(-(-got[1].astype(int) >> (e2 - e)), np.ceil(x))
        got, e = np.stack([lo, hi]), e2
    assert e == e_want and np.array_equal(got, want)
    assert (want[0] * 2.0 ** e <= held.min(0)).all() and (want[1] * 2.0 ** e >= held.max(0)).all()


def test_page_score_bounds_every_key():
    rng = np.random.default_rng(1)
    held = kv4.values(*kv4.quantise(rng.standard_normal((16, 64)).astype(np.float32)))
    b, e = kv4.bounds(held)
    q = np.rint(rng.standard_normal((4, 64)) * 30)
    score = np.maximum(q * b[0], q * b[1]).sum() * 2.0 ** e
    assert score >= (held @ q.T).sum(1).max()


@pytest.mark.parametrize("kw", [
    dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
    dict(scaling="llama3", factor=8.0, original_max_positions=512),
    dict(scaling="yarn", factor=4.0, original_max_positions=512)])
def test_rotary_table(kw):
    from flashcodec_b200 import rotary_table
    R, base, n = 64, 10000.0, 3000
    got = rotary_table(n, R, base, device="cpu", **kw).numpy()
    assert got.shape == (n, R) and got.dtype == np.float32
    f, factor, gain = kw.get("scaling"), kw.get("factor", 1.0), 1.0
    freq = []
    for i in range(R // 2):
        w = base ** (-2 * i / R)
        turns = kw.get("original_max_positions", 1) * w / (2 * math.pi)
        if f == "linear":
            w /= factor
        elif f == "ntk":
            w = (base * factor ** (R / (R - 2))) ** (-2 * i / R)
        elif f == "llama3":
            mix = min(1.0, max(0.0, (turns - 1.0) / 3.0))
            w = mix * w + (1 - mix) * w / factor
        elif f == "yarn":
            dim = lambda t: R * math.log(512 / (t * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(dim(32.0)), 0), min(math.ceil(dim(1.0)), R - 1)
            ramp = min(1.0, max(0.0, (i - lo) / (hi - lo)))
            w, gain = w * (1 - ramp) + w / factor * ramp, 0.1 * math.log(factor) + 1
        freq.append(w)
    a = np.arange(n)[:, None] * np.array(freq)
    want = np.concatenate([np.cos(a), np.sin(a)], 1) * gain
    # fp32 rounding of values up to `gain`, and fp64 angles up to n off by an ulp or two
    assert np.abs(got - want).max() <= gain * 2.0 ** -24 + n * 2.0 ** -50


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=63), dict(rotary_dim=0), dict(max_positions=0), dict(factor=0.5),
    dict(scaling="other"), dict(scaling="yarn", factor=2.0), dict(scaling="llama3", factor=2.0)])
def test_rotary_table_refuses(kw):
    from flashcodec_b200 import rotary_table
    a = dict(max_positions=16, rotary_dim=64, device="cpu") | kw
    with pytest.raises(ValueError):
        rotary_table(a.pop("max_positions"), a.pop("rotary_dim"), **a)


def test_no_cpu_cache():
    from flashcodec_b200 import PagedInt4Cache
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedInt4Cache(4, 2, 64, device="cpu")


@pytest.fixture(scope="module")
def lib():
    from flashcodec_b200 import _lib, build
    build.build()
    return _lib.load()


def _append(lib, **kw):
    P = ctypes.c_void_p(0x1000)
    a = dict(q=P, qo=P, Hq=4, k=P, v=P, dtype=1, B=2, S=1, T=2, cu=None, lengths=P, qw=None, kw=None,
             w_dtype=1, rotary=None, rows=0, R=0, pool=P, pages=8, Hk=2, D=64, page=16, table=P,
             max_pages=4, bounds=None, exps=None, status=P) | kw
    return lib.fc_kv4_append(
        a["q"], 256, 256, 64, a["qo"], 256, 256, 64, a["Hq"], a["k"], 128, 128, 64, a["v"], 128, 128, 64,
        a["dtype"], a["B"], a["S"], a["T"], a["cu"], a["lengths"], None, a["qw"], a["kw"], a["w_dtype"],
        1e-6, a["rotary"], a["rows"], a["R"], 0, a["pool"], a["pages"], a["Hk"], a["D"], a["page"],
        a["table"], a["max_pages"], a["max_pages"], a["bounds"], a["exps"], a["status"], None)


ODD = ctypes.c_void_p(0x1004)


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=3), 1), (dict(D=80), 4), (dict(D=512), 4), (dict(page=24), 1), (dict(page=8), 1),
    (dict(page=2048), 1), (dict(T=3), 1), (dict(S=-1), 1), (dict(pages=0), 1), (dict(max_pages=0), 1),
    (dict(max_pages=1 << 30), 1), (dict(pool=None), 1), (dict(pool=ODD), 1), (dict(table=None), 1),
    (dict(status=None), 1), (dict(k=None), 1), (dict(lengths=None), 1), (dict(q=None), 1),
    (dict(bounds=ctypes.c_void_p(0x2000)), 1), (dict(kw=ODD, w_dtype=3), 1),
    (dict(rotary=ctypes.c_void_p(0x2000), rows=4, R=24), 1), (dict(rotary=ODD, rows=4, R=32), 1),
    (dict(rotary=ctypes.c_void_p(0x2000), rows=4, R=128), 1),
    (dict(rotary=ctypes.c_void_p(0x2000), rows=0, R=32), 1), (dict(Hk=0), 1)])
def test_append_refuses(lib, kw, rc):
    assert _append(lib, **kw) == rc
    assert lib.fc_last_error_string()


def test_empty_calls_launch_nothing(lib):
    P = ctypes.c_void_p(0x1000)
    assert _append(lib, B=0, T=0) == 0
    assert _append(lib, S=0, T=0) == 0
    assert lib.fc_kv4_read(P, 8, 2, 64, 16, P, 4, 4, None, 2, 0, 0, None, P, P, 1, 0, 0, 0, P, None) == 0
    assert lib.fc_kv4_attn(P, 1, 0, 1, 4, 256, 256, 64, P, 8, 2, 64, 16, P, 4, 4, P, None, 0, 1.0, P, 256, 256,
                           64, None, P, 4096, P, None) == 0


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=3), 1), (dict(Hq=5), 1), (dict(Hq=0), 1), (dict(D=100), 4), (dict(q=None), 1),
    (dict(lengths=None), 1), (dict(Sq=2, sel=ctypes.c_void_p(0x2000), n=3), 1),
    (dict(sel=ctypes.c_void_p(0x2000), n=-1), 1), (dict(ws=None), 1),
    (dict(ws_bytes=16), 3), (dict(ws=ODD), 1), (dict(B=1 << 25), 1)])
def test_attn_refuses(lib, kw, rc):
    P = ctypes.c_void_p(0x1000)
    a = dict(q=P, dtype=1, B=2, Sq=1, Hq=4, D=64, lengths=P, sel=None, n=0, ws=P, ws_bytes=1 << 30) | kw
    got = lib.fc_kv4_attn(a["q"], a["dtype"], a["B"], a["Sq"], a["Hq"], 256, 256, 64, P, 8, 2, a["D"], 16,
                          P, 4, 4, a["lengths"], a["sel"], a["n"], 1.0, P, 256, 256, 64, None, a["ws"],
                          a["ws_bytes"], P, None)
    assert got == rc and lib.fc_last_error_string()


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=3), 1), (dict(Hq=5), 1), (dict(count=0), 1), (dict(count=2, sink=2), 1), (dict(sink=-1), 1),
    (dict(bounds=None), 1), (dict(exps=None), 1), (dict(ws=None), 1), (dict(ws_bytes=0), 3),
    (dict(Hq=1024), 1)])
def test_select_refuses(lib, kw, rc):
    P = ctypes.c_void_p(0x1000)
    a = dict(q=P, dtype=1, B=2, Hq=4, bounds=P, exps=P, count=4, sink=1, recent=1, ws=P, ws_bytes=1 << 22) | kw
    got = lib.fc_kv4_select(a["q"], a["dtype"], a["B"], a["Hq"], 256, 64, a["bounds"], a["exps"], 8, 2, 64, 16,
                            P, 4, 4, P, a["count"], a["sink"], a["recent"], P, a["ws"], a["ws_bytes"], P, None)
    assert got == rc and lib.fc_last_error_string()


def test_page_bytes(lib):
    # 4.5 bits a value: 16 tokens are 16 * D bytes of K and V codes and 2 * 16 * D / 32 scales
    for D in (64, 96, 128, 192, 256):
        assert lib.fc_kv4_page_bytes(3, D, 64) == 3 * 64 * (D + 2 * 2 * D // 32)
    assert lib.fc_kv4_page_bytes(3, 80, 64) == -1 and lib.fc_kv4_page_bytes(3, 64, 48) == -1
