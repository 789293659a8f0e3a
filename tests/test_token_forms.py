"""CPU tests that the sizes of token_forms.py take the forms of the kernels that they are there for, so that none goes untested."""
import ctypes

import pytest

import token_forms as F

F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    import protein_clip_amd  # noqa: F401
    from protein_clip_amd import _lib
    return _lib.load()


def _aligned(rows, width, out, dtype):
    step = 4 if dtype == F32 else 8
    return width % step == 0 and out % step == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_sizes_take_their_tiles(lib, dtype):
    seen = set()
    for rows, width, out, _, _, _, tiles, aligned in F.LINEAR:
        assert _aligned(rows, width, out, dtype) == aligned
        got = [lib.pclip_linear_tile(rows, width, out, dtype, p, aligned) for p in range(3)]
        assert tuple(got[:2]) == tiles
        seen |= {(p, aligned, tile) for p, tile in enumerate(got)}
    # dW has 64 x 64 tiles in the small cases of test_gpu_token_ops.py
    assert seen >= {(p, True, tile) for p in (0, 1) for tile in (64, 128, 256)} | {(p, False, tile) for p in (0, 1) for tile in (64, 128)} | {(2, True, 128), (2, False, 128)}


def test_linear_sizes_take_their_tiles_in_f32(lib):
    seen = {(p, _aligned(*c[:3], F32), lib.pclip_linear_tile(*c[:3], F32, p, _aligned(*c[:3], F32))) for c in F.LINEAR for p in range(3)}
    assert seen >= {(p, a, 64) for p in range(3) for a in (True, False)} | {(2, True, 128)}


def test_split_sizes_split(lib):
    """dx is the product of dy with the weight, its contraction the layer's width out: a forward of these sizes."""
    for rows, width, out, _, _, _, splits in F.SPLIT:
        assert (lib.pclip_linear_fwd_workspace_bytes(rows, width, out, F32) > 0, lib.pclip_linear_fwd_workspace_bytes(rows, out, width, F32) > 0) == splits
        assert lib.pclip_linear_fwd_workspace_bytes(rows, width, out, BF16) == lib.pclip_linear_fwd_workspace_bytes(rows, width, out, F16) == 0
    assert lib.pclip_linear_fwd_workspace_bytes(300, 320, 320, F32) == lib.pclip_linear_fwd_workspace_bytes(16384, 1280, 1280, F32) == 0


def test_scratch_of_the_forward_is_checked(lib):
    one, err = ctypes.c_void_p(64), lambda: lib.pclip_last_error().decode()
    need = lib.pclip_linear_fwd_workspace_bytes(60, 2560, 2560, F32)

    def call(ws=one, n=need):
        return lib.pclip_linear_fwd_ws(one, one, None, None, 60, 2560, 2560, F32, 0, one, None, ws, n, None)

    assert call(n=need - 1) == -1 and "workspace too small" in err()
    assert call(ws=ctypes.c_void_p(72)) == -1 and "16-byte aligned" in err()
    assert lib.pclip_linear_fwd_ws(None, one, None, None, 60, 2560, 2560, F32, 0, one, None, one, need, None) == -1 and "null pointer" in err()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_norm_widths_reach_every_form(lib, dtype):
    def form(d):
        v = [ctypes.c_int() for _ in range(3)]
        assert lib.pclip_norm_gate_row(d, dtype, *map(ctypes.byref, v)) == 0
        return tuple(x.value for x in v)

    assert {form(c[2]) for c in F.NORM} == {form(d) for d in range(1, 4097)}


def test_queries_refuse_bad_sizes(lib):
    n = ctypes.c_int()
    assert lib.pclip_linear_tile(0, 8, 8, BF16, 0, 1) == 0 and lib.pclip_linear_tile(8, 8, 8, 7, 0, 1) == 0
    assert lib.pclip_norm_gate_row(4097, F32, ctypes.byref(n), ctypes.byref(n), ctypes.byref(n)) == -1
    assert lib.pclip_norm_gate_row(8, F32, None, ctypes.byref(n), ctypes.byref(n)) == -1
