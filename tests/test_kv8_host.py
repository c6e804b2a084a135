"""Paged 8-bit KV cache and prompt attention, without a GPU: the oracle's own properties, the
rotary axes, arguments and refusals that need no launch."""

import ctypes
import weakref

import numpy as np
import pytest
import torch

from oracle import kv8


def test_quantise_holds_values_to_half_a_step():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 3, 64)) * np.exp(rng.standard_normal((50, 3, 1)) * 3)).astype(np.float32)
    c, s = kv8.quantise(x)
    held = kv8.values(c, s).astype(np.float64)
    step = np.repeat(s.astype(np.float64), 16, 0)[:50, :, None]
    assert (np.abs(held - x) <= step / 2).all()
    for r in range(4):  # a step is 1/128 to 1/64 of the run's largest value
        top = np.abs(x[16 * r: 16 * r + 16]).max((0, 2))
        assert (top < 128 * s[r]).all() and (top >= 64 * s[r]).all()


def test_quantise_edges():
    x = np.zeros((96, 1, 64), np.float32)
    x[16] = 1e-44            # below the least scale
    x[32, 0, 3] = np.nan
    x[48, 0, 5] = np.inf
    x[64, 0, 5], x[65, 0, 6] = -64.0, -1e-30  # a power of two; less than any step
    x[80, 0, 0] = 3.4e38
    c, s = kv8.quantise(x)
    assert s[0, 0] == 0 and s[1, 0] == np.float32(2.0 ** -126) and np.isnan(s[2, 0]) and np.isnan(s[3, 0])
    assert s[4, 0] == 1 and c[64, 0, 5] == -64 and c[65, 0, 6] == -1 and s[5, 0] == np.float32(2.0 ** 121)
    assert c[80, 0, 0] == 127 and not c[:64].any()


@pytest.mark.parametrize("seed", range(4))
def test_stored_codes_do_not_depend_on_the_split(seed):
    """Shifting the codes held when a later token raises the scale gives those of the run at once."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((16, 1, 64)) * np.exp(3 * rng.standard_normal((16, 1, 1)))).astype(np.float32)
    want, s_want = kv8.quantise(x)
    s, c = np.float32(0), np.zeros((0, 64), np.int8)
    for t in range(16):
        new = max(s, kv8.scale(x[t, 0]))
        shift = int(np.log2(new / s)) if s > 0 else 0
        c = np.concatenate([c >> min(shift, 7), kv8.codes(x[t:t + 1, 0], new)])
        s = new
    assert s == s_want[0, 0] and np.array_equal(c, want[:, 0])


def test_rotary_axes():
    from flashcodec_b200 import rotary_axes
    assert rotary_axes((2, 3, 1), device="cpu").tolist() == [0, 0, 1, 1, 1, 2]
    assert rotary_axes((3, 2, 2), alternate=True, device="cpu").tolist() == [0, 1, 2, 0, 1, 2, 0]
    assert rotary_axes((0, 2), device="cpu").dtype == torch.int32
    for bad in ((), (0, 0), (-1, 2)):
        with pytest.raises(ValueError):
            rotary_axes(bad, device="cpu")


def test_no_cpu():
    from flashcodec_b200 import PagedInt8Cache, prompt_attention
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedInt8Cache(4, 2, 64, device="cpu")
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt_attention(q, q, q, torch.tensor([0, 3], dtype=torch.int32))


# ------------------------------------------------------------- arguments, launches stood in for
HK, D, PAGE = 2, 64, 16


@pytest.fixture
def cache():
    from flashcodec_b200 import PagedInt8Cache
    cache = object.__new__(PagedInt8Cache)
    cache.device, cache._index, cache._scale = torch.device("cpu"), -1, 1.0  # a CPU tensor's index
    cache.num_kv_heads, cache.head_dim, cache.page_size = HK, D, PAGE
    cache._codes = cache._scales = cache._status = torch.zeros(1)
    return cache


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("call", ["read", "append", "append_packed", "attend"])
def test_arguments_live_until_the_launch(cache, monkeypatch, call):
    from flashcodec_b200 import _kernels as K
    refs, launched = [], []

    def tmp(t):
        refs.append(weakref.ref(t))
        return t

    def launch(*args):
        assert all(r() is not None for r in refs), "freed before the launch"
        launched.append(args)
    for name in ("kv8_read", "kv8_append", "kv8_attn"):
        monkeypatch.setattr(K, name, launch)
    rows = lambda *lead, heads=HK: tmp(torch.zeros(*lead, heads, D))  # noqa: E731
    table = lambda: tmp(torch.zeros(3, 4, dtype=torch.int32))  # noqa: E731
    if call == "read":
        cache.read(table(), tmp(i32(0, 1, 2)), count=5, cu_seqlens=tmp(i32(0, 1, 3, 5)))
    elif call == "append":
        cache.append(rows(3, 1, heads=4), rows(3, 1), rows(3, 1), table(), tmp(i32(0, 1, 2)),
                     positions=tmp(torch.zeros(2, 3, 1, dtype=torch.int32)), axes=tmp(torch.zeros(32, dtype=torch.int32)),
                     q_weight=tmp(torch.ones(D)), rotary=tmp(torch.ones(8, D)))
    elif call == "append_packed":
        cache.append(rows(5, heads=4), rows(5), rows(5), table(), tmp(i32(0, 1, 2)),
                     positions=tmp(i32(0, 1, 2, 3, 4)), cu_seqlens=tmp(i32(0, 1, 3, 5)))
    else:
        cache.attend(rows(3, heads=4), table(), tmp(i32(1, 1, 2)), return_lse=True)
    assert launched


def test_refused_arguments(cache, monkeypatch):
    from flashcodec_b200 import _kernels as K
    for name in ("kv8_read", "kv8_append", "kv8_attn"):
        monkeypatch.setattr(K, name, lambda *args: None)
    table, lens, kv, q = torch.zeros(3, 4, dtype=torch.int32), i32(0, 1, 2), torch.zeros(3, HK, D), torch.zeros(3, 4, D)
    rotary, axes = torch.ones(8, D), torch.zeros(32, dtype=torch.int32)
    positions = torch.zeros(3, 3, dtype=torch.int32)
    cache.append(q, kv, kv, table, lens, rotary=rotary, positions=positions, axes=axes)
    bad = [dict(axes=axes), dict(axes=axes, rotary=rotary), dict(axes=axes, positions=positions),
           dict(axes=axes[:31], rotary=rotary, positions=positions), dict(axes=axes.long(), rotary=rotary, positions=positions),
           dict(axes=axes, rotary=rotary, positions=i32(0, 0, 0)), dict(axes=axes, rotary=rotary, positions=positions[:0]),
           dict(rotary=rotary, positions=positions), dict(q_out=q.half()), dict(q_weight=torch.ones(D + 1)),
           dict(rotary=rotary.half())]
    for kw in bad:
        with pytest.raises(ValueError):
            cache.append(q, kv, kv, table, lens, **kw)
    for args in ((q, kv[:2], kv, table, lens), (q, kv, kv.half(), table, lens), (q, kv, kv, table.long(), lens),
                 (q, kv, kv, table, lens.long()), (q[:, :, :32], kv, kv, table, lens), (q, kv[:, :1], kv[:, :1], table, lens)):
        with pytest.raises(ValueError):
            cache.append(*args)
    for kw in (dict(count=None), dict(count=-1), dict(count=3, cu_seqlens=i32(0, 3))):
        with pytest.raises(ValueError):
            cache.read(table, **kw)
    for args, kw in (((q[:2], table, lens), {}), ((q, table, lens[:2]), {}), ((q, table, lens), dict(out=q.half()))):
        with pytest.raises(ValueError):
            cache.attend(*args, **kw)
    with pytest.raises(RuntimeError, match="8-bit cache holds rounded values"):
        cache.attend(q.clone().requires_grad_(), table, lens)


@pytest.mark.parametrize("name", ["codes", "scales", "status"])
def test_the_caches_tensors_cannot_be_replaced(cache, name):
    with pytest.raises(AttributeError):
        setattr(cache, name, torch.zeros(1))


# ------------------------------------------------------------- refusals of the C ABI
@pytest.fixture(scope="module")
def lib():
    from flashcodec_b200 import _lib, build
    build.build()
    return _lib.load()


P = ctypes.c_void_p(4096)  # aligned, never read: these calls are refused before a launch


def append(lib, **kw):
    a = dict(q=P, q_sb=128, q_ss=128, q_sh=64, q_out=P, qo_sb=128, qo_ss=128, qo_sh=64, Hq=2, k=ctypes.c_void_p(1 << 20), k_sb=64,
             k_ss=64, k_sh=64, v=ctypes.c_void_p(1 << 21), v_sb=64, v_ss=64, v_sh=64, dtype=1, B=1, S=1, T=1, cu=None,
             lengths=P, positions=None, axes=None, n_axes=0, qw=None, kw=None, w_dtype=0, eps=1e-6, rotary=None, rows=0,
             dim=0, inter=0, codes=P, scales=P, num_pages=4, Hk=1, D=64, page=16, table=P, stride=1, max_pages=1, status=P,
             stream=None) | kw
    return lib.fc_kv8_append(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(D=80), 4), (dict(page=24), 1), (dict(page=8), 1), (dict(scales=None), 1), (dict(codes=None), 1), (dict(status=None), 1),
    (dict(codes=ctypes.c_void_p(4104)), 1), (dict(dtype=3), 1), (dict(T=2), 1), (dict(k=None), 1), (dict(lengths=None), 1),
    (dict(q_out=None), 1), (dict(rotary=P, rows=4, dim=24), 1), (dict(rotary=P, rows=4, dim=80), 1),
    (dict(rotary=P, rows=0, dim=64), 1), (dict(rotary=ctypes.c_void_p(4100), rows=4, dim=64), 1),
    (dict(axes=P, n_axes=3), 1), (dict(axes=P, n_axes=3, positions=P), 1),
    (dict(axes=P, n_axes=0, positions=P, rotary=P, rows=4, dim=64), 1), (dict(q_out=ctypes.c_void_p(4224)), 1),
    (dict(k=P), 1), (dict(qo_sh=0), 1), (dict(qw=P, w_dtype=3), 1)])
def test_append_refuses(lib, kw, code):
    assert append(lib, **kw) == code


def test_append_of_nothing(lib):
    assert append(lib, T=0, S=0) == 0 and append(lib, B=0, T=0) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(D=48), 4), (dict(dtype=3), 1), (dict(Hq=3), 1), (dict(Hq=0), 1), (dict(scale=float("nan")), 1),
    (dict(scale=float("inf")), 1), (dict(ws=None), 1), (dict(ws=ctypes.c_void_p(4100)), 1), (dict(bytes=1024), 3), (dict(q=None), 1),
    (dict(out=ctypes.c_void_p(4096 + 128)), 1), (dict(o_sh=0), 1), (dict(B=1 << 20), 4), (dict(scales=None), 1)])
def test_attend_refuses(lib, kw, code):
    a = dict(q=P, dtype=1, B=1, Sq=1, Hq=4, q_sb=256, q_ss=256, q_sh=64, codes=P, scales=P, num_pages=4, Hk=2, D=64, page=16,
             table=P, stride=1, max_pages=4, lengths=P, scale=0.1, out=ctypes.c_void_p(1 << 30), o_sb=256, o_ss=256, o_sh=64, lse=None, ws=P,
             bytes=1 << 40, status=P, stream=None) | kw
    assert lib.fc_kv8_attn(*a.values()) == code


@pytest.mark.parametrize("kw,code", [(dict(dtype=3), 1), (dict(T=3), 1), (dict(k=None), 1), (dict(D=100), 4)])
def test_read_refuses(lib, kw, code):
    a = dict(codes=P, scales=P, num_pages=4, Hk=2, D=64, page=16, table=P, stride=1, max_pages=4, starts=None, B=1, S=2, T=2, cu=None,
             k=P, v=P, dtype=1, o_sb=256, o_ss=128, o_sh=64, status=P, stream=None) | kw
    assert lib.fc_kv8_read(*a.values()) == code


@pytest.mark.parametrize("kw,code", [
    (dict(D=80), 4), (dict(dtype=0), 4), (dict(Hq=3), 1), (dict(Hq=512), 4), (dict(scale=float("nan")), 1), (dict(Tq=9), 1),
    (dict(cu_q=P), 1), (dict(q=None), 1), (dict(k=None), 1), (dict(out=ctypes.c_void_p(4096 + 128)), 1), (dict(o_sh=0), 1),
    (dict(out=ctypes.c_void_p(1 << 24)), 1), (dict(ws=None), 1), (dict(bytes=64), 3), (dict(q=ctypes.c_void_p(4098)), 1),
    (dict(k_ss=132), 1), (dict(k_sh=0), 1)])
def test_prompt_refuses(lib, kw, code):
    a = dict(q=P, q_sb=2048, q_ss=256, q_sh=64, k=ctypes.c_void_p(1 << 24), k_sb=1024, k_ss=128, k_sh=64,
             v=ctypes.c_void_p(1 << 26), v_sb=1024, v_ss=128, v_sh=64, dtype=1, B=1, Sq=8, Sk=8, Tq=8, Tk=8, Hq=4, Hk=2, D=64,
             cu_q=None, cu_k=None, causal=1, scale=0.1, out=ctypes.c_void_p(1 << 30), o_sb=2048, o_ss=256, o_sh=64, lse=None, ws=P,
             bytes=1 << 40, stream=None) | kw
    assert lib.fc_prompt_attn(*a.values()) == code
