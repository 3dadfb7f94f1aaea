"""Host side of the pre-norm block's operators: the generator's published vectors, formulas against differences, workspace sizes,
and every refusal of the C ABI and of the Python layer. No kernel is launched: each call below is refused before it would."""
import ctypes
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import prenorm_oracle as P
from cgpt_b200 import _lib, ops
from cgpt_b200._lib import lib

OK, NULL, DTYPE, SHAPE, OPTION, ALIGN = 0, 1, 2, 3, 4, 5
A, B, C, D, E, F, G, H = (0x10000 * (i + 1) for i in range(8))     # aligned addresses that nothing reads
BF16, F32 = _lib.BF16, _lib.F32


def test_philox_published_vectors():
    hexes = lambda c, k: [f"{int(w):08x}" for w in P.philox4x32_10(c, k)]
    assert hexes([0] * 4, [0, 0]) == "6627e8d5 e169c58d bc57ac4c 9b00dbd8".split()
    assert hexes([0xffffffff] * 4, [0xffffffff] * 2) == "408f276d 41c83b0e a20bc7c6 6d5451fd".split()
    assert hexes([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == "d16cfe09 94fdcceb 5001e420 24126ea1".split()


def test_decisions_do_not_depend_on_where_a_count_starts():
    whole = P.keep(100, 0.3, 7, 9, 2)
    for first in (0, 1, 7, 8, 13):
        assert np.array_equal(P.keep(40, 0.3, 7, 9, 2, first), whole[first:first + 40])


def test_layernorm_gradient_against_differences():
    """Central differences in 64 bits: the truncation error is h^2 / 6 times third derivatives of order one, the rounding error
    2^-53 / h times the loss of order ten; both are below 1e-8 at h = 1e-5."""
    r = np.random.default_rng(0)
    x, w, b, dy = r.standard_normal((3, 7)), r.standard_normal(7), r.standard_normal(7), r.standard_normal((3, 7))
    dx, dw, db = P.layernorm_backward(dy, x, w, 1e-5)
    loss = lambda x, w, b: float((dy * P.layernorm(x, w, b, 1e-5)).sum())
    h = 1e-5
    for _ in range(5):
        vx, vw, vb = r.standard_normal(x.shape), r.standard_normal(7), r.standard_normal(7)
        num = (loss(x + h * vx, w + h * vw, b + h * vb) - loss(x - h * vx, w - h * vw, b - h * vb)) / (2 * h)
        assert abs(num - ((dx * vx).sum() + (dw * vw).sum() + (db * vb).sum())) < 1e-7


def test_workspace_sizes():
    assert lib.cgpt_layernorm_backward_workspace_bytes(0, 8) == 0 and lib.cgpt_layernorm_backward_workspace_bytes(8, 0) == 0
    assert lib.cgpt_layernorm_backward_workspace_bytes(1 << 40, 1 << 20) == 0
    assert lib.cgpt_layernorm_backward_workspace_bytes(1, 1) >= 8
    size = lib.cgpt_scaled_embedding_backward_workspace_bytes
    assert size(0, 8) == size(8, 0) == size(1 << 31, 8) == 0
    assert size(1, 1) >= 16


@pytest.mark.parametrize("size", [lib.cgpt_layernorm_backward_workspace_bytes, lib.cgpt_scaled_embedding_backward_workspace_bytes])
@pytest.mark.parametrize("hidden", [1, 64, 250, 256, 511, 1000, 1024, 2048, 2056, 4099, 8192, 12008, 16384])
def test_a_workspace_for_many_rows_serves_fewer(size, hidden):
    """Rows a CTA takes, and CTAs, change with the row count; what is asked for may not fall at any of these changes."""
    sizes = [size(n, hidden) for n in (*range(1, 12000), *range(12000, 80000, 37))]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))


def dropout_forward(out=A, x=B, residual=None, count=8, p=0.5, state=C, site=0, dtype=BF16):
    return lib.cgpt_dropout_forward(out, x, residual, count, p, state, site, dtype, None)


def dropout_backward(dx=A, dy=B, count=8, p=0.5, state=C, site=0, accumulate=0, dtype=BF16):
    return lib.cgpt_dropout_backward(dx, dy, count, p, state, site, accumulate, dtype, None)


def norm_forward(y=A, x=B, w=C, b=D, rows=4, hidden=8, eps=1e-5, dtype=BF16):
    return lib.cgpt_layernorm_forward(y, x, w, b, rows, hidden, eps, dtype, None)


def norm_backward(dx=A, dw=B, db=C, dy=D, x=E, w=F, residual=None, ws=G, size=1 << 20, rows=4, hidden=8, eps=1e-5, dtype=BF16):
    return lib.cgpt_layernorm_backward(dx, dw, db, dy, x, w, residual, ws, size, rows, hidden, eps, dtype, None)


def fused_forward(y=A, total=B, x=C, residual=D, w=E, b=F, rows=4, hidden=8, eps=1e-5, p=0.5, state=G, dtype=BF16):
    return lib.cgpt_dropout_add_layernorm_forward(y, total, x, residual, w, b, rows, hidden, eps, p, state, 0, dtype, None)


def fused_backward(dx=A, dr=B, dw=C, db=D, dy=E, dsum=F, total=G, w=H, ws=9 * A, size=1 << 20, rows=4, hidden=8, eps=1e-5, p=0.5,
                   state=10 * A, dtype=BF16):
    return lib.cgpt_dropout_add_layernorm_backward(dx, dr, dw, db, dy, dsum, total, w, ws, size, rows, hidden, eps, p, state, 0, dtype, None)


def embed_forward(out=A, ids=B, w=C, tokens=4, vocab=10, hidden=8, scale=1.0, p=0.5, state=D, dtype=BF16):
    return lib.cgpt_scaled_embedding_forward(out, ids, w, tokens, vocab, hidden, scale, p, state, 0, dtype, None)


def embed_backward(dw=A, dy=B, ids=C, ws=D, size=1 << 24, tokens=4, vocab=10, hidden=8, scale=1.0, pad=0xffffffff, p=0.5, state=E, dtype=BF16):
    return lib.cgpt_scaled_embedding_backward(dw, dy, ids, ws, size, tokens, vocab, hidden, scale, pad, p, state, 0, 0, dtype, None)


CALLS = [dropout_forward, dropout_backward, norm_forward, norm_backward, fused_forward, fused_backward, embed_forward, embed_backward]
WITH_DROPOUT = [dropout_forward, dropout_backward, fused_forward, fused_backward, embed_forward, embed_backward]
REQUIRED = {dropout_forward: "out x state", dropout_backward: "dx dy state", norm_forward: "y x w", norm_backward: "dx dw dy x w ws",
            fused_forward: "y total x residual w state", fused_backward: "dx dr dw dy total w ws state", embed_forward: "out ids w state",
            embed_backward: "dw dy ids ws state"}


@pytest.mark.parametrize("call", CALLS)
def test_refuses_null_and_dtype(call):
    for name in REQUIRED[call].split():
        assert call(**{name: None}) == NULL, name
    assert call(dtype=3) == DTYPE and call(dtype=-1) == DTYPE


@pytest.mark.parametrize("call", CALLS)
def test_refuses_empty_and_oversized(call):
    sizes = {dropout_forward: ["count"], dropout_backward: ["count"], embed_forward: ["tokens", "vocab", "hidden"],
             embed_backward: ["tokens", "vocab", "hidden"]}.get(call, ["rows", "hidden"])
    for name in sizes:
        assert call(**{name: 0}) == SHAPE, name
        assert call(**{name: 1 << 50}) == SHAPE, name


@pytest.mark.parametrize("call", WITH_DROPOUT)
def test_refuses_bad_dropout_options(call):
    for p in (-0.1, 1.0, 1.5, float("nan"), float("inf")):
        assert call(p=p) == OPTION, p
    assert call(state=0x10004) == ALIGN
    if call in (dropout_forward, dropout_backward):
        assert call(count=(1 << 35) + 1) == SHAPE      # the block counter would wrap
    else:
        rows = "tokens" if call in (embed_forward, embed_backward) else "rows"
        assert call(**{rows: (1 << 25) + 1, "hidden": 1 << 10, **({"size": 1 << 60} if "size" in call.__code__.co_varnames else {})}) == SHAPE


@pytest.mark.parametrize("call", CALLS)
def test_refuses_misaligned_pointers(call):
    for name in call.__code__.co_varnames[:call.__code__.co_argcount]:
        default = dict(zip(call.__code__.co_varnames, call.__defaults__))[name]
        if isinstance(default, int) and default >= A and name not in ("state", "size", "pad"):
            assert call(**{name: default + 1}) == ALIGN, name
    if "ws" in call.__code__.co_varnames:
        assert call(ws=9 * A + 8) == ALIGN
    if "ids" in call.__code__.co_varnames:
        assert call(ids=B + 2) == ALIGN


@pytest.mark.parametrize("call", [norm_forward, norm_backward, fused_forward, fused_backward])
def test_refuses_bad_epsilon(call):
    for eps in (0.0, -1.0, float("nan")):
        assert call(eps=eps) == OPTION


def test_refuses_aliases_and_small_workspaces():
    assert norm_forward(y=B) == OPTION
    assert norm_backward(dx=D) == OPTION and norm_backward(dx=E) == OPTION
    assert all(fused_forward(y=v) == OPTION for v in (B, C, D))
    assert all(fused_backward(dx=v) == OPTION for v in (B, E, F, G)) and all(fused_backward(dr=v) == OPTION for v in (E, G))
    assert dropout_backward(dx=B, accumulate=1) == OPTION
    assert embed_backward(dw=B) == OPTION and embed_backward(scale=float("inf")) == OPTION and embed_forward(scale=float("nan")) == OPTION
    need = lib.cgpt_layernorm_backward_workspace_bytes(4, 8)
    assert norm_backward(size=need - 1) == SHAPE and fused_backward(size=need - 1) == SHAPE
    assert embed_backward(size=lib.cgpt_scaled_embedding_backward_workspace_bytes(4, 8) - 1) == SHAPE
    assert lib.cgpt_dropout_advance(None, 1, None) == NULL and lib.cgpt_dropout_advance(A + 4, 1, None) == ALIGN


def test_refuses_a_scale_that_overflows_with_dropout():
    # kept elements are multiplied by scale * 65536 / (65536 - t): infinite here, and 0 * inf in dropped places
    assert embed_forward(scale=3e38, p=0.5) == OPTION and embed_backward(scale=-3e38, p=0.5) == OPTION


def test_python_layer_refuses_host_tensors_and_options():
    x, w, ids = torch.zeros(4, 8), torch.zeros(8), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.dropout_forward(x, x, None)
    with pytest.raises(ValueError):
        ops.layernorm_forward(x, x.clone(), w, w, 1e-5)
    with pytest.raises(ValueError):
        ops.layernorm_backward(x, w, w, x, x, w, 1e-5)
    with pytest.raises(ValueError):
        ops.dropout_add_layernorm_forward(x, x, x, x, w, w, 1e-5, None)
    with pytest.raises(ValueError):
        ops.scaled_embedding_forward(x, ids, 4, torch.zeros(10, 8))
    with pytest.raises(ValueError):
        ops.scaled_embedding_backward(torch.zeros(10, 8), x, ids, 4)
    with pytest.raises(ValueError):
        ops.dropout_advance(torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.dropout_advance(None, -1)


def test_state_holds_any_64_bit_words():
    s = ops.make_dropout_state(0xffffffffffffffff, 1 << 63, device="cpu")
    assert [ctypes.c_uint64(v).value for v in s.tolist()] == [0xffffffffffffffff, 1 << 63]


def test_the_module_is_imported_without_cuda_functions_in_torch():
    """What a torch built without CUDA lacks is taken away in a fresh process before the import."""
    code = ("import torch\nfor name in dir(torch._C):\n    if name.startswith('_cuda_'): delattr(torch._C, name)\n"
            "import cgpt_b200.ops as ops\n"
            "try: ops.layernorm_forward(*(torch.zeros(4, 8) for _ in range(2)), torch.zeros(8), None, 1e-5)\n"
            "except ValueError: print('refused')\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True)
    assert done.stdout == "refused\n", done.stderr
