"""CPU: what the attention path's entry points refuse before any launch, the
records they take, the shares of work, and the plans made on the host."""
from __future__ import annotations

import ctypes
import math
import shutil
import subprocess
from fractions import Fraction

import attention_oracle as oracle
import pytest
import torch

from conftest import ROOT
from losslessly_compressed_tensors_amd.components import attention
from losslessly_compressed_tensors_amd.components.dropout import dropout_add
from losslessly_compressed_tensors_amd.kernels import attention as kernels
from losslessly_compressed_tensors_amd.kernels import hip

LCT_E_NULL, LCT_E_SIZE, LCT_E_ARG = -1, -3, -4
FAKE = 1 << 20                     # never dereferenced: the checks fail first


@pytest.fixture(scope="module")
def lib():
    if not hip.LIBRARY_PATH.exists():
        pytest.skip("liblct_hip.so not built (python -m losslessly_compressed_tensors_amd.build)")
    return hip.load_library()


def _attention(pointers=(FAKE,) * 4, lse=FAKE, lengths=0, strides=((512, 64, 128),) * 4, batch=1,
               heads=2, kv_heads=1, queries=4, keys=4, dim=64, window=0, sinks=0, scale=0.1):
    return hip.ATTENTION.pack(*pointers, lse, lengths, *(s for t in strides for s in t), batch,
                              heads, kv_heads, queries, keys, dim, window, sinks, 0, scale)


BAD_ATTENTION = [
    (dict(pointers=(FAKE, 0, FAKE, FAKE)), LCT_E_NULL),
    (dict(batch=0), LCT_E_SIZE), (dict(heads=3, kv_heads=2), LCT_E_SIZE),
    (dict(queries=0), LCT_E_SIZE), (dict(keys=0), LCT_E_SIZE), (dict(keys=2 ** 30 + 1), LCT_E_SIZE),
    (dict(dim=12), LCT_E_SIZE), (dict(dim=136), LCT_E_SIZE), (dict(dim=0), LCT_E_SIZE),
    (dict(batch=2 ** 15, heads=2 ** 9), LCT_E_SIZE),
    (dict(window=-1), LCT_E_ARG), (dict(sinks=-1), LCT_E_ARG), (dict(scale=0.0), LCT_E_ARG),
    (dict(scale=-1.0), LCT_E_ARG), (dict(scale=math.nan), LCT_E_ARG),
    (dict(scale=math.inf), LCT_E_ARG), (dict(pointers=(FAKE + 8,) + (FAKE,) * 3), LCT_E_ARG),
    (dict(strides=((512, 64, 4),) + ((512, 64, 128),) * 3), LCT_E_ARG),
    (dict(strides=((512, 64, 128),) * 3 + ((512, 64, 1 << 24),)), LCT_E_ARG),
    (dict(strides=((-512, 64, 128),) + ((512, 64, 128),) * 3), LCT_E_ARG),
]


@pytest.mark.parametrize("change,code", BAD_ATTENTION, ids=lambda c: str(c)[:60])
def test_attention_rejects_bad_records_before_launch(lib, change, code):
    record = _attention(**change)
    gradients = hip.ATTENTION_GRADIENTS.pack(*(FAKE,) * 5, *(512, 64, 128) * 4)
    assert lib.lct_attention_forward(record, 1, None, 0, None) == code
    assert lib.lct_attention_backward(record, gradients, 1, 1, None, 0, None) == code
    assert lib.lct_attention_decode(record, 1, None, 0, None) == code


def test_attention_rejects_bad_parts_and_workspaces_before_launch(lib):
    record = _attention()
    for splits in (0, 65, -1):
        assert lib.lct_attention_forward(record, splits, None, 0, None) == LCT_E_ARG
    assert lib.lct_attention_forward(record, 2, None, 1 << 20, None) == LCT_E_NULL
    need = 2 * 2 * 4 * 66
    assert lib.lct_attention_forward(record, 2, ctypes.c_void_p(FAKE), need - 1, None) == LCT_E_SIZE
    assert lib.lct_attention_forward(record, 2, ctypes.c_void_p(FAKE + 4), need, None) == LCT_E_ARG

    gradients = hip.ATTENTION_GRADIENTS.pack(*(FAKE,) * 5, *(512, 64, 128) * 4)
    call = lib.lct_attention_backward
    assert call(record, None, 1, 1, None, 0, None) == LCT_E_NULL
    assert call(_attention(lse=0), gradients, 1, 1, None, 0, None) == LCT_E_NULL
    missing = hip.ATTENTION_GRADIENTS.pack(FAKE, FAKE, 0, FAKE, FAKE, *(512, 64, 128) * 4)
    assert call(record, missing, 1, 1, None, 0, None) == LCT_E_NULL
    odd = hip.ATTENTION_GRADIENTS.pack(*(FAKE,) * 5, *(512, 64, 129), *(512, 64, 128) * 3)
    assert call(record, odd, 1, 1, None, 0, None) == LCT_E_ARG
    assert call(record, gradients, 0, 1, None, 0, None) == LCT_E_ARG
    assert call(record, gradients, 1, 65, None, 0, None) == LCT_E_ARG
    assert call(record, gradients, 2, 1, None, 0, None) == LCT_E_NULL
    need = 2 * 2 * 128 * 64          # one block of 128 keys in two parts, dk and dv
    assert call(record, gradients, 2, 1, ctypes.c_void_p(FAKE), need - 1, None) == LCT_E_SIZE

    one = _attention(queries=1, lse=0)
    assert lib.lct_attention_decode(record, 1, None, 0, None) == LCT_E_ARG       # four queries
    assert lib.lct_attention_decode(_attention(queries=1), 1, None, 0, None) == LCT_E_ARG   # lse
    assert lib.lct_attention_decode(one, 65, None, 0, None) == LCT_E_ARG
    assert lib.lct_attention_decode(one, 2, None, 1 << 20, None) == LCT_E_NULL
    assert lib.lct_attention_decode(one, 2, ctypes.c_void_p(FAKE), 2 * 2 * 66 - 1,
                                    None) == LCT_E_SIZE


def _rotary(pointers=(FAKE, FAKE, 0, FAKE, FAKE, 0), turns=FAKE, strides=(512, 128, 64) * 6, batch=1,
            tokens=4, heads=2, kv_heads=1, dim=64, turned=64, kind=0, capacity=0):
    return hip.ROTARY.pack(*pointers, turns, 0, *strides, 0, 0, 0, batch, tokens, heads, kv_heads,
                           dim, turned, 0, 0, kind, capacity, 1.0)


@pytest.mark.parametrize("change,code", [
    (dict(pointers=(0, FAKE, 0, FAKE, FAKE, 0)), LCT_E_NULL), (dict(turns=0), LCT_E_NULL),
    (dict(pointers=(FAKE, FAKE, 0, FAKE, 0, 0)), LCT_E_NULL),
    (dict(pointers=(FAKE, 0, FAKE, FAKE, 0, FAKE)), LCT_E_NULL),      # v without k
    (dict(batch=0), LCT_E_SIZE), (dict(tokens=0), LCT_E_SIZE), (dict(heads=0), LCT_E_SIZE),
    (dict(kv_heads=0), LCT_E_SIZE), (dict(heads=4097), LCT_E_SIZE), (dict(dim=257), LCT_E_SIZE),
    (dict(turned=63), LCT_E_SIZE), (dict(turned=66), LCT_E_SIZE), (dict(turned=0), LCT_E_SIZE),
    (dict(capacity=-1), LCT_E_SIZE), (dict(kind=3), LCT_E_ARG),
    (dict(pointers=(FAKE + 1, FAKE, 0, FAKE, FAKE, 0)), LCT_E_ARG),
    (dict(pointers=(FAKE,) * 6), LCT_E_ARG),                          # v without a cache
    (dict(strides=(512, 128, 1 << 31) + (512, 128, 64) * 5), LCT_E_ARG),
], ids=lambda c: str(c)[:60])
def test_rotate_rejects_bad_records_before_launch(lib, change, code):
    assert lib.lct_rotate(_rotary(**change), None) == code


def test_dropout_rejects_bad_arguments_before_launch(lib):
    fake = ctypes.c_void_p(FAKE)

    def call(x=fake, residual=fake, out=fake, n=8, kind=0, below=0, more=None):
        return lib.lct_dropout(x, residual, out, n, kind, below, 0, 0, more, None)

    assert call(x=None) == LCT_E_NULL and call(out=None) == LCT_E_NULL
    assert call(n=0) == LCT_E_SIZE and call(n=2 ** 35 - 2047) == LCT_E_SIZE
    assert call(kind=3) == LCT_E_ARG
    assert call(below=-1) == LCT_E_ARG and call(below=65537) == LCT_E_ARG
    assert call(x=ctypes.c_void_p(FAKE + 8)) == LCT_E_ARG
    assert call(residual=ctypes.c_void_p(FAKE + 2)) == LCT_E_ARG
    assert call(more=ctypes.c_void_p(FAKE + 4)) == LCT_E_ARG


def test_records_have_the_headers_layout(tmp_path):
    """Sizes and the last fields' places, from a C compiler."""
    include = "/opt/rocm/include"
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    source = tmp_path / "sizes.c"
    source.write_text(f'''#include <stdio.h>
#include <stddef.h>
#include "{ROOT}/include/lct.h"
int main(void) {{
    printf("%zu %zu %zu %zu %zu\\n", sizeof(lct_attention), offsetof(lct_attention, scale),
           sizeof(lct_attention_gradients), sizeof(lct_rotary), offsetof(lct_rotary, magnitude));
    return 0;
}}''')
    program = tmp_path / "sizes"
    built = subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", "-I", include, str(source), "-o",
                            str(program)], capture_output=True, text=True)
    if built.returncode:
        pytest.skip(f"the HIP headers do not compile here: {built.stderr[-200:]}")
    sizes = [int(n) for n in subprocess.run([str(program)], capture_output=True, text=True,
                                            check=True).stdout.split()]
    assert sizes == [hip.ATTENTION.size, hip.ATTENTION.size - 4, hip.ATTENTION_GRADIENTS.size,
                     hip.ROTARY.size, hip.ROTARY.size - 8]


def test_shares_of_work():
    """Parts lie within the entry points' limits, small calls are whole, and what
    few workgroups would do is shared."""
    for batch, heads, kv, queries, keys, dim, window, sinks in (
            (1, 1, 1, 1, 1, 8, 0, 0), (8, 12, 12, 1024, 1024, 64, 256, 4),
            (1, 16, 4, 16384, 16384, 128, 4096, 4), (1, 32, 8, 8191, 16383, 128, 0, 0),
            (1, 8, 1, 16, 100000, 128, 0, 0), (1, 1, 1, 2 ** 20, 2 ** 20, 64, 5, 2 ** 20)):
        forward = kernels.forward_splits(batch, heads, queries, keys, window, sinks)
        assert 1 <= forward <= 64
        for n in kernels.backward_splits(batch, heads, kv, queries, keys, dim, window, sinks):
            assert 1 <= n <= 64
        assert 1 <= kernels.decode_splits(batch, heads, kv, keys, window, sinks) <= 64
    assert kernels.forward_splits(8, 12, 1024, 1024, 256, 4) == 1
    assert kernels.forward_splits(1, 8, 16, 100000, 0, 0) == 64
    assert kernels.backward_splits(1, 16, 4, 16384, 16384, 128, 0, 7)[1] == 1    # no window
    # Both sides of the lines that decode_splits states.
    assert kernels.decode_splits(1, 12, 12, 1024, 0, 0) == 1
    assert kernels.decode_splits(1, 12, 12, 1100, 0, 0) > 1
    assert kernels.decode_splits(1, 12, 12, 100000, 256, 4) == 1
    assert kernels.decode_splits(64, 32, 8, 8192, 4096, 4) == 1
    assert kernels.decode_splits(16, 32, 8, 4096, 0, 0) == 6


def test_plans():
    plan = attention.Rotary([0.0, math.pi, -math.pi / 2, 2 * math.pi], device="cpu")
    # 0, a half (the sign bit), minus a quarter, a whole turn (none).
    assert plan.turns.tolist() == [0, -2 ** 63, -2 ** 62, 0] and plan.dim == 8
    trainer = attention.trainer_frequencies(64)
    assert trainer.shape == (32,) and float(trainer[0]) == -1.0
    assert abs(float(trainer[15]) + 1 / 1024) < 1e-15 and bool((trainer[16:] == 0).all())
    with pytest.raises(ValueError, match="factor"):
        attention.rotary_frequencies(8, factor=0.5)
    with pytest.raises(ValueError, match="fast_turns"):
        attention.rotary_frequencies(8, scaling="ramp", factor=2.0, slow_turns=4, fast_turns=4)


def test_host_tensors_are_refused():
    q = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        attention.window_attention(q, q, q)
    with pytest.raises(ValueError, match="GPU"):
        attention.apply_rotary(attention.Rotary([1.0], device="cpu"), q)
    with pytest.raises(ValueError, match="GPU"):
        dropout_add(q, None, 0.1, 1)
    with pytest.raises(TypeError):
        attention.window_attention(None, q, q)


def test_the_oracle_itself():
    """The 64-bit forms against torch's own: attention without a window, its
    gradients, the generator's published words."""
    gen = torch.Generator().manual_seed(3)
    q, k, v, g = (torch.randn(2, 4, 9, 16, generator=gen, dtype=torch.float64) for _ in range(4))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.nn.functional.scaled_dot_product_attention(*leaves, is_causal=True, scale=0.3)
    want.backward(g)
    seen = oracle.sees(9, 9, None, 0, None, 2)
    # The bounds' type: any; only the exact values are looked at.
    got = oracle.attention_with_bounds(*(t.to(torch.bfloat16) for t in (q, k, v)), seen, 0.3,
                                       g.to(torch.bfloat16))
    rounded = [t.to(torch.bfloat16).double().requires_grad_() for t in (q, k, v)]
    out = torch.nn.functional.scaled_dot_product_attention(*rounded, is_causal=True, scale=0.3)
    out.backward(g.to(torch.bfloat16).double())
    for name, value in zip(("out", "dq", "dk", "dv"), (out, *(t.grad for t in rounded))):
        assert float((got[name][0] - value.detach()).abs().amax()) < 1e-12
    assert int(oracle.sees(5, 3).sum()) == 6 and int(oracle.sees(4, 4, 1, 2).sum()) == 1 + 2 + 3 + 3
    assert [hex(int(w)) for w in oracle.philox_words(1, 0, 0)[0]] == [
        "0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


@pytest.mark.parametrize("dim,block", [(64, 128), (128, 256)])
def test_the_workspace_holds_parts_of_blocks_that_have_several(lib, dim, block):
    """1000 keys of 2 key heads, 300 sinks: no more is asked than parts that are
    written, by the entry point and by its caller."""
    blocks, sink_blocks = -(-1000 // block), -(-300 // block)
    gradients = hip.ATTENTION_GRADIENTS.pack(*(FAKE,) * 5, *(512, 64, 128) * 4)
    fake = ctypes.c_void_p(FAKE)
    for window, sinks, splits, sink_splits, parts in (
            (50, 300, 1, 5, sink_blocks * 5), (50, 300, 3, 1, (blocks - sink_blocks) * 3),
            (50, 300, 3, 5, sink_blocks * 5 + (blocks - sink_blocks) * 3), (0, 300, 1, 5, 0),
            (0, 300, 3, 5, blocks * 3), (50, 1000, 3, 1, 0), (50, 300, 1, 1, 0)):
        floats = 2 * parts * (2 * block * dim + 64)
        assert kernels.backward_workspace(1, 2, 1000, dim, window, sinks, splits,
                                          sink_splits) == floats
        record = _attention(heads=4, kv_heads=2, queries=1000, keys=1000, dim=dim, window=window,
                            sinks=sinks)
        if parts:
            assert lib.lct_attention_backward(record, gradients, splits, sink_splits, fake,
                                              floats - 1, None) == LCT_E_SIZE
            assert lib.lct_attention_backward(record, gradients, splits, sink_splits, None, floats,
                                              None) == LCT_E_NULL
    # One long sequence under a window: its blocks without sinks are stored whole.
    splits, sink_splits = kernels.backward_splits(1, 16, 4, 16384, 16384, 128, 4096, 4)
    assert splits == 1 and sink_splits > 1
    assert kernels.backward_workspace(1, 4, 16384, 128, 4096, 4, splits, sink_splits) == (
        4 * sink_splits * (2 * 256 * 128 + 64))


def test_long_caches_are_only_bound_by_what_is_launched(lib):
    """2^28 keys: the launch that adds parts is as large as the blocks that have any."""
    gradients = hip.ATTENTION_GRADIENTS.pack(*(FAKE,) * 5, *(512, 64, 128) * 4)
    long = _attention(keys=2 ** 28, window=5, sinks=3)
    call = lib.lct_attention_backward
    assert call(long, gradients, 1, 2, None, 0, None) == LCT_E_NULL      # the workspace
    assert call(long, gradients, 2, 1, None, 0, None) == LCT_E_SIZE      # parts of all keys


# To 60 digits.
PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494")


@pytest.mark.parametrize("frequency", [1.0, 0.01, 1e-6, -0.3333333333333333, 5e-324, 1e300,
                                       12345.678, *attention.rotary_frequencies(16).tolist()])
def test_frequencies_are_the_nearest_fractions_of_a_turn(frequency):
    """Half of the last place, and the 2^-54 that FP64's turn is off."""
    turns, = attention.Rotary([frequency], device="cpu").turns.tolist()
    exact = Fraction(frequency) * 2 ** 64 / (2 * PI)
    off = (turns - exact) % 2 ** 64
    assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + abs(exact) / 2 ** 54


def test_positions_are_held_to_where_angles_are_right():
    for position in (2 ** 31, -2 ** 31, 0):
        assert attention._first_position(position) == position
    for position in (2 ** 31 + 1, -2 ** 31 - 1, 2 ** 62):
        with pytest.raises(ValueError, match="positions"):
            attention._first_position(position)
    # The fastest pair there: less than FP32's 2^-26 of a turn off.
    turns, = attention.Rotary([1.0], device="cpu").turns.tolist()
    off = (Fraction(turns, 2 ** 64) - 1 / (2 * PI)) * 2 ** 31 % 1
    assert min(off, 1 - off) < Fraction(1, 2 ** 26)
