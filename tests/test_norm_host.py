"""The norms' backward entry points without a GPU: what they refuse before they touch a device."""
import pytest


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as entry

    entry.build()
    from qwen3_moe_fused import _lib

    return _lib.load()


ARGS = dict(dnormed=64, dsum=64, base=64, rstd=64, gamma=64, y=64, inv=64, weights=64, scale=1.0, dresidual=64, dy=64, dweights=64,
            dgamma=None, T=4, k=2, H=8, dtype=1, ws=None, ws_bytes=0, stream=None)


def call(fn, **changed):
    return fn(*{**ARGS, **changed}.values())


def test_refusals(lib):
    inputs, stored = lib.moe_combine_add_rms_norm_bwd_inputs, lib.moe_combine_add_rms_norm_bwd
    for fn in (inputs, stored):
        assert call(fn, dtype=9) == -1
        assert call(fn, H=24577) == -2 and call(fn, H=0) == -2 and call(fn, T=-1) == -2 and call(fn, T=1 << 31) == -2
        assert call(fn, inv=None) == -2  # k = 2 without an index
        assert call(fn, inv=None, k=1) == -3  # gradients of weights that there are not
        assert call(fn, rstd=None) == -3 and call(fn, gamma=None) == -3 and call(fn, weights=None) == -3
        assert call(fn, y=None) == -3
        assert call(fn, dgamma=64) == -4 and call(fn, dgamma=64, ws=72, ws_bytes=1 << 20) == -4
        assert call(fn, T=0) == 0 and call(fn, dresidual=None, dy=None, dweights=None) == 0
    # the sum from the inputs: a residual may be missing, the rows may not; the stored sum the other way round
    add = dict(inv=None, k=1, weights=None, dweights=None, dgamma=64)
    assert call(inputs, **add, y=None) == -3 and call(inputs, **add, base=None) == -4
    assert call(stored, **add, base=None) == -3 and call(stored, **add, y=None) == -4


def test_longest_rows_are_taken(lib):
    longest = 1 << 24
    assert lib.moe_fp8_quantize_rows(None, 1, 4, longest, None, None, None) == -3  # (of the arguments only the addresses are missing)
    assert lib.moe_fp8_silu_quantize(None, None, 4, longest, None, None, None, None, 1, None) == -3
    assert lib.moe_fp8_silu_quantize(None, None, 4, longest + 1, None, None, None, None, 1, None) == -2
    assert lib.moe_fp8_silu_bwd_quantize(None, None, None, 4, longest + 1, None, None, None, None, 1, None) == -2
