"""The 8-bit operators' refusals and the product's rule: host code, no GPU.  Every call here is answered before it would
touch a device (the pointers are small numbers that nothing dereferences)."""
import ctypes

import pytest

import warpc_public_release_b200 as w
from warpc_public_release_b200 import _lib
from warpc_public_release_b200._lib import WG_E_ARG, WG_E_LIMIT, WarpcError

P = 4096  # an aligned address that no refused call reads


def refused(code, f, *a, **kw):
    with pytest.raises(WarpcError) as e:
        f(*a, **kw)
    assert e.value.code == code


@pytest.mark.parametrize("change", [
    dict(dX=None), dict(dQ=None), dict(dScale=None), dict(k=0), dict(m=-1), dict(ldx=63), dict(ldq=63), dict(dX=P + 1), dict(dScale=P + 2),
    dict(dtype="fp32", dX=P + 2)])
def test_quantise_refuses(change):
    kw = {**dict(m=2, k=64, dX=P, dQ=P, dScale=P), **change}
    refused(WG_E_ARG, w.quantise_rows, **kw)


@pytest.mark.parametrize("change", [
    dict(dX=None), dict(dW=None), dict(dQ=None), dict(dScale=None), dict(eps=-1.0), dict(eps=float("nan")), dict(dR=P), dict(dH=P),
    dict(dR=P, dH=P, ldr=63), dict(dR=P, dH=P, ldh=63), dict(dR=P + 1, dH=P), dict(dR=P, dH=P + 1), dict(dW=P + 1), dict(ldx=63), dict(ldq=63),
    dict(dR=2 * P, dH=P, ldh=80), dict(dR=P, dH=P, dX=2 * P, ldh=80), dict(k=0), dict(m=-1), dict(dScale=P + 1)])
def test_norm_refuses(change):
    kw = {**dict(m=2, k=64, dX=P, dW=P, eps=1e-6, dQ=P, dScale=P), **change}
    refused(WG_E_ARG, w.norm_quantise_rows, **kw)


def test_rows_too_long():
    refused(WG_E_LIMIT, w.quantise_rows, 1, 2 ** 30 + 1, P, P, P)
    refused(WG_E_LIMIT, w.norm_quantise_rows, 1, 2 ** 30 + 1, P, P, 1e-6, P, P)


def test_no_rows_is_no_work():
    w.quantise_rows(0, 64, None, None, None)
    w.norm_quantise_rows(0, 64, None, None, 1e-6, None, None)


def test_unknown_type():
    with pytest.raises(ValueError):
        w.quantise_rows(1, 64, P, P, P, dtype="int8")
    with pytest.raises(ValueError):
        w.Int8Plan(64, 64, P, P, out="fp64")
    assert _lib.lib().wg_quantise_rows(0, 1, 64, 3, P, 64, P, 64, P, None) == WG_E_ARG


@pytest.mark.parametrize("change,code", [
    (dict(dBt=None), WG_E_ARG), (dict(dScaleB=None), WG_E_ARG), (dict(dBt=P + 8), WG_E_ARG), (dict(dScaleB=P + 4), WG_E_ARG), (dict(dBias=P + 4), WG_E_ARG),
    (dict(n=0), WG_E_ARG), (dict(k=0), WG_E_ARG), (dict(ldb=48), WG_E_ARG), (dict(ldb=72), WG_E_ARG), (dict(k=65), WG_E_ARG),
    (dict(k=131072), WG_E_LIMIT), (dict(n=2 ** 30 + 1), WG_E_LIMIT)])
def test_plan_refuses(change, code):
    kw = {**dict(n=64, k=64, dBt=P, dScaleB=P), **change}
    refused(code, w.Int8Plan, **kw)


def test_null_plans():
    l = _lib.lib()
    assert l.wg_int8_launch(None, 1, P, 64, P, P, 64, None) == WG_E_ARG
    assert l.wg_int8_plan_set_program(None, None) == WG_E_ARG
    assert l.wg_int8_plan_set_timeout_ms(None, 1) == WG_E_ARG
    assert l.wg_int8_last_device_status(None, None) == WG_E_ARG
    assert l.wg_int8_plan_reset(None) == WG_E_ARG
    assert l.wg_int8_plan_destroy(None) == 0
    assert l.wg_int8_plan_create(0, 64, 64, P, 64, P, None, 0, None) == WG_E_ARG


@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 17, 33, 64, 65, 128, 129, 300, 1000, 4096, 70000, 2 ** 30])
@pytest.mark.parametrize("n", [1, 48, 1003, 4096, 16384, 100000])
@pytest.mark.parametrize("k", [1, 100, 1111, 4096, 131071])
def test_rule_covers_every_shape(m, n, k):
    """The rule's launch covers the output, fits the machine, and shares K only where there is some for everyone."""
    if m * n > 2 ** 40:  # more values than any memory holds: may be refused
        try:
            w.int8_choose(m, n, k)
        except WarpcError as e:
            assert e.code == WG_E_LIMIT
            return
    i = w.int8_choose(m, n, k)
    up = lambda a, b: -(-a // b)  # noqa: E731
    assert i.threads in (256, 384) and 0 <= i.dynsmem <= 232448 and 1 <= i.cluster <= 8 and i.grid % i.cluster == 0 and 0 < i.grid < 2 ** 31
    if i.kernel == _lib.INT8_GEMV:
        assert m <= i.tile_m and i.tile_n * i.split == 32 and i.tiles == i.grid == up(n, i.tile_n)
    else:
        assert i.tiles == up(m, i.tile_m) * up(n, i.tile_n) and i.depth >= 2
        if i.kernel == _lib.INT8_FEW:
            assert i.split <= up(k, 128) and i.cluster == i.split and i.grid == i.tiles * i.split
        else:
            assert i.split == 1 and i.cluster == i.tile_m // 128 and i.grid <= 148 and i.grid <= i.tiles * i.cluster


def test_rule_refuses():
    for a in ((0, 64, 64), (64, 0, 64), (64, 64, 0)):
        refused(WG_E_ARG, w.int8_choose, *a)
    refused(WG_E_LIMIT, w.int8_choose, 64, 64, 131072)
    refused(WG_E_LIMIT, w.int8_choose, 2 ** 30 + 1, 64, 64)
    refused(WG_E_LIMIT, w.int8_choose, 64, 2 ** 30 + 1, 64)
    assert _lib.lib().wg_int8_choose(1, 1, 1, None) == WG_E_ARG


def test_info_layout():
    assert ctypes.sizeof(w.Int8Info) == 40


def test_the_commands(capsys):
    from warpc_public_release_b200 import gemm, run_int8
    assert gemm.main(["int8", "512", "4096", "4096"]) == 0
    line = capsys.readouterr().out
    assert line.startswith("# int8 kernel=") and " grid=" in line
    assert gemm.main(["int8", "0", "4096", "4096"]) == 1 and gemm.main(["int8", "5"]) == 2
    for bad in ([], ["1", "2"], ["1", "2", "x"], ["0", "2", "3"], ["1", "2", "3", "0"], ["1", "2", "3", "--out", "int8"], ["1", "2", "3", "--out"]):
        assert run_int8.main(bad) == 2
