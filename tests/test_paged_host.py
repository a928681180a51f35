"""What the launchers of rotary positions, the paged cache and its attention refuse before
anything is launched, their workspaces, the frequencies, and the tests' own oracle (host
logic, no GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import _paged as O
from pico_amd import kernels as K
from pico_amd._lib import hip_lib

PTR = 256  # never read: every call here is refused on its arguments
EINVAL = -1


@pytest.fixture(scope="module")
def L():
    return hip_lib()


def _refused(L, status, word):
    assert status == EINVAL
    assert word in L.pk_last_error().decode()


def _rope(rot=8, freqs=PTR):
    return ctypes.byref(K.PkRope(freqs, rot, 0, 1.0))


def _cache(**kw):
    f = dict(k=PTR, v=PTR, k_exp=PTR, v_exp=PTR, table=PTR, lens=PTR, offsets=PTR, pages=8, kv_heads=2,
             hd=64, page=16, B=3, width=4)
    f.update(kw)
    return ctypes.byref(K.PkKvCache(*[f[n] for n, _ in K.PkKvCache._fields_]))


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "parts"])
@pytest.mark.parametrize("rot", [0, 2, 10, 64])
def test_frequencies(scaling, rot):
    base, factor, length, low, high = 10000.0, 8.0, 2048.0, 1.0, 32.0
    got = K.rope_freqs(rot, base, scaling, factor, length, low, high, device="cpu").numpy()
    want = []
    for i in range(rot // 2):
        b = base * factor ** (rot / (rot - 2)) if scaling == "ntk" and rot > 2 else base
        f = b ** (-2 * i / rot)
        if scaling == "linear":
            f /= factor
        if scaling == "parts":
            r = length * f / (2 * math.pi)
            g = min(1.0, max(0.0, (r - low) / (high - low)))
            f = f * (g + (1 - g) / factor)
        want.append(f)
    assert got.dtype == np.float64 and got.shape == (rot // 2,)
    np.testing.assert_allclose(got, want, rtol=1e-14)


def test_frequencies_refused(L):
    buf = (ctypes.c_double * 8)()
    for rot in (-2, 3, 2048):
        _refused(L, L.pk_rope_freqs(rot, 1e4, 0, 1.0, 0.0, 1.0, 2.0, buf), "rot")
    _refused(L, L.pk_rope_freqs(4, 1e4, 0, 1.0, 0.0, 1.0, 2.0, None), "NULL")
    _refused(L, L.pk_rope_freqs(4, 1e4, 4, 1.0, 0.0, 1.0, 2.0, buf), "scaling")
    for base, factor in ((0.0, 2.0), (math.nan, 2.0), (math.inf, 2.0), (1e4, 0.0), (1e4, -1.0), (1e4, math.inf)):
        _refused(L, L.pk_rope_freqs(4, base, 1, factor, 0.0, 1.0, 2.0, buf), "positive")
    for length, low, high in ((0.0, 1.0, 2.0), (math.nan, 1.0, 2.0), (9.0, 2.0, 2.0), (9.0, math.nan, 2.0)):
        _refused(L, L.pk_rope_freqs(4, 1e4, 3, 2.0, length, low, high, buf), "parts")


def test_rope_refused(L):
    f = L.pk_rope_f32
    for N, H, hd in ((-1, 1, 8), (1 << 24, 1, 8), (4, 0, 8), (4, 1, 0), (4, 1, 1025), (4, 1 << 17, 16)):
        _refused(L, f(N, H, hd, _rope(2), PTR, PTR, 1 << 30, PTR, 1 << 30, 0, None), "pk_rope_f32")
    for rope in (None, _rope(10), _rope(3), _rope(-2), _rope(8, None)):
        _refused(L, f(4, 2, 8, rope, PTR, PTR, 16, PTR, 16, 0, None), "rot")
    for p, x, y in ((None, PTR, PTR), (PTR, None, PTR), (PTR, PTR, None)):
        _refused(L, f(4, 2, 8, _rope(), p, x, 16, y, 16, 0, None), "NULL")
    for ldx, ldy in ((15, 16), (16, 15)):
        _refused(L, f(4, 2, 8, _rope(), PTR, PTR, ldx, PTR, ldy, 0, None), "stride")
    assert f(0, 2, 8, _rope(), None, None, 16, None, 16, 0, None) == 0


BAD_CACHE = [(dict(hd=0), "head size"), (dict(hd=257), "head size"), (dict(page=8), "page"),
             (dict(page=48), "page"), (dict(page=256), "page"), (dict(kv_heads=0), "kv_heads"),
             (dict(kv_heads=4097), "kv_heads"), (dict(pages=0), "pages"), (dict(pages=1 << 31), "pages"),
             (dict(B=-1), "B"), (dict(B=(1 << 20) + 1), "B"), (dict(width=0), "width"),
             (dict(width=1 << 26), "width"), (dict(k=None), "NULL"), (dict(v=None), "NULL"),
             (dict(k_exp=None), "NULL"), (dict(v_exp=None), "NULL"), (dict(table=None), "NULL"),
             (dict(lens=None), "NULL"), (dict(offsets=None), "NULL"), (dict(k=264), "aligned"),
             (dict(v=264), "aligned"), (dict(k_exp=257), "aligned"), (dict(v_exp=258), "aligned")]


@pytest.mark.parametrize("bad,word", BAD_CACHE)
def test_bad_caches_refused(L, bad, word):
    c = _cache(**bad)
    _refused(L, L.pk_kv_append_f32(c, 4, PTR, 1 << 20, PTR, 1 << 20, None, 0, None, 0, None, 0, None), word)
    _refused(L, L.pk_attn_paged_f32(c, 4, 4096, 1.0, PTR, 1 << 20, PTR, 1 << 20, PTR, 1 << 40, None), word)
    assert L.pk_attn_paged_workspace(c, 4, 4096) == 0


def test_append_refused(L):
    f = L.pk_kv_append_f32
    _refused(L, f(None, 4, PTR, 128, PTR, 128, None, 0, None, 0, None, 0, None), "NULL")
    for N in (-1, 1 << 24):
        _refused(L, f(_cache(), N, PTR, 128, PTR, 128, None, 0, None, 0, None, 0, None), "rows")
    for rope in (_rope(66), _rope(5), _rope(8, None)):
        _refused(L, f(_cache(), 4, PTR, 128, PTR, 128, rope, 0, None, 0, None, 0, None), "rot")
    for k, v in ((None, PTR), (PTR, None)):
        _refused(L, f(_cache(), 4, k, 128, v, 128, None, 0, None, 0, None, 0, None), "NULL")
    for ldk, ldv in ((127, 128), (128, 127)):
        _refused(L, f(_cache(), 4, PTR, ldk, PTR, ldv, None, 0, None, 0, None, 0, None), "stride")
    for H, ldq, out, ldo in ((0, 256, PTR, 256), (1 << 15, 1 << 30, PTR, 1 << 30), (4, 255, PTR, 256),
                             (4, 256, PTR, 255), (4, 256, None, 256)):
        _refused(L, f(_cache(), 4, PTR, 128, PTR, 128, None, H, PTR, ldq, out, ldo, None), "q")
    # nothing to write
    assert f(_cache(), 0, None, 128, None, 128, None, 0, None, 0, None, 0, None) == 0
    assert f(_cache(B=0), 4, None, 128, None, 128, None, 0, None, 0, None, 0, None) == 0
    # more workgroups than a launch has
    _refused(L, f(_cache(kv_heads=4096, B=1 << 20), 1 << 23, PTR, 1 << 20, PTR, 1 << 20, None, 0, None, 0, None, 0,
                  None), "launch")


def test_attention_refused(L):
    f = L.pk_attn_paged_f32
    _refused(L, f(None, 4, 4, 1.0, PTR, 256, PTR, 256, PTR, 1 << 40, None), "NULL")
    for H in (0, 3, 1 << 15):
        _refused(L, f(_cache(), 4, H, 1.0, PTR, 1 << 30, PTR, 1 << 30, PTR, 1 << 40, None), "heads")
    _refused(L, f(_cache(), 1 << 20, 4096, 1.0, PTR, 1 << 20, PTR, 1 << 20, PTR, 1 << 40, None), "N*H")
    for q, o in ((None, PTR), (PTR, None)):
        _refused(L, f(_cache(), 4, 4, 1.0, q, 256, o, 256, PTR, 1 << 40, None), "NULL")
    for ldq, ldo in ((255, 256), (256, 255)):
        _refused(L, f(_cache(), 4, 4, 1.0, PTR, ldq, PTR, ldo, PTR, 1 << 40, None), "stride")
    need = L.pk_attn_paged_workspace(_cache(width=4096), 3, 4)
    assert need > 0
    for ws, size in ((None, need), (PTR, need - 1), (PTR + 4, need)):
        _refused(L, f(_cache(width=4096), 3, 4, 1.0, PTR, 256, PTR, 256, ws, size, None), "workspace")
    assert f(_cache(), 0, 4, 1.0, None, 256, None, 256, None, 0, None) == 0
    assert f(_cache(B=0), 4, 4, 1.0, None, 256, None, 256, None, 0, None) == 0
    assert L.pk_attn_paged_workspace(_cache(), 0, 4) == 0


def test_no_sequences_need_no_arrays(L):
    c = _cache(B=0, table=None, lens=None, offsets=None)
    assert L.pk_kv_append_f32(c, 4, PTR, 128, PTR, 128, None, 0, None, 0, None, 0, None) == 0
    assert L.pk_attn_paged_f32(c, 4, 4, 1.0, PTR, 256, PTR, 256, None, 0, None) == 0
    assert L.pk_attn_paged_workspace(c, 4, 4) == 0
    assert L.pk_kv_append_f32(_cache(B=0, k=None), 4, PTR, 128, PTR, 128, None, 0, None, 0, None, 0, None) == EINVAL


def test_head_sizes():
    assert [K.kv_head_size(h) for h in (0, -1, 1, 32, 33, 64, 65, 96, 97, 128, 129, 256, 257)] == \
        [0, 0, 32, 32, 64, 64, 96, 96, 128, 128, 256, 256, 0]
    assert all(K.kv_head_size(h) == O.head_size(h) for h in range(1, 257))


def test_bindings_refuse():
    cpu = torch.zeros(4, 16)
    with pytest.raises(TypeError):
        K.Rope(torch.zeros(4))  # not float64
    with pytest.raises((TypeError, ValueError)):
        K.PagedKV(*[torch.zeros(1, dtype=torch.uint8)] * 4, *[torch.zeros(1, dtype=torch.int32)] * 3, 64)
    del cpu


# ------------------------------------------------------- the oracle's own rounding
def test_the_oracle_rounds_to_nearest_even():
    x = np.concatenate([np.linspace(-500, 500, 4001), np.linspace(-0.02, 0.02, 4001), [np.inf, -np.inf]])
    want = torch.tensor(x).clamp(-448, 448).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(O.CODES[O.encode(x)], O.CODES[want])
    every = np.array([c for c in range(256) if c & 127 != 127])
    np.testing.assert_array_equal(O.encode(O.CODES[every]), every)
    assert np.isnan(O.CODES[O.encode([np.nan])]).all()


def test_the_oracle_finds_the_exponent():
    for top, e in ((448.0, 0), (448.1, 1), (224.0, -1), (0.0, -40), (1e-30, -40), (1e30, 40), (1.0, -8)):
        assert O.exponent(np.array([top, -top / 2, np.nan, np.inf])) == e


# --------------------------------------------------------------- pico's API
@pytest.fixture(scope="module")
def A():
    from pico_amd import pico

    lib = pico.amd_lib()
    for name, (res, args) in pico._GPU_SIGS.items():
        if "rope" in name or "kv_" in name or "cached" in name:
            f = getattr(lib, name)
            f.restype, f.argtypes = res, args
    return lib


@pytest.mark.parametrize("bad", [dict(rot=0), dict(rot=-2), dict(rot=7), dict(rot=1026), dict(base=0.0),
                                 dict(scaling=9), dict(scaling=1, factor=0.0), dict(scaling=3, length=0.0),
                                 dict(scaling=3, low=2.0, high=2.0), dict(magnitude=math.inf)])
def test_pico_rope_init_refuses(A, bad):
    from pico_amd.pico import PicoRopeConfig

    f = dict(rot=8, interleaved=0, base=1e4, scaling=0, factor=2.0, length=9.0, low=1.0, high=32.0, magnitude=0.0)
    f.update(bad)
    c = PicoRopeConfig(*[f[n] for n, _ in PicoRopeConfig._fields_])
    assert not A.pico_rope_init(ctypes.byref(c))
    assert not A.pico_rope_init(None)
    A.pico_rope_free(None)


@pytest.mark.parametrize("bad", [dict(layers=0), dict(kv_heads=0), dict(kv_heads=4097), dict(head_dim=0),
                                 dict(head_dim=257), dict(page=24), dict(pages=0), dict(sequences=0),
                                 dict(sequences=(1 << 20) + 1), dict(max_length=0), dict(max_length=1 << 30)])
def test_pico_kv_init_refuses(A, bad):
    from pico_amd.pico import PicoKVConfig

    f = dict(layers=1, kv_heads=2, head_dim=64, page=16, pages=4, sequences=2, max_length=64)
    f.update(bad)
    c = PicoKVConfig(*[f[n] for n, _ in PicoKVConfig._fields_])
    assert not A.pico_kv_init(ctypes.byref(c))
    assert not A.pico_kv_init(None)


def test_pico_without_a_cache(A):
    assert A.pico_kv_begin(None, None) == -1
    assert A.pico_kv_length(None, 0) == -1
    assert A.pico_kv_drop(None, 0) != 0
    assert not A.pico_attention_cached(None, 0, None, None, None, 1, None)
    assert not A.pico_rope(None, None, None, 1)
    A.pico_kv_free(None)
