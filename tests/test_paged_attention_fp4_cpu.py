"""What the descriptors of attention over a 4-bit pool refuse, without a GPU."""
import ctypes

import pytest
import torch

from capi import describe

_POOL = ("k_codes", "v_codes", "k_scales", "v_scales")
_ORDER = {"": ("out", "q", *_POOL, "table", "lens", "alibi"), "Prefill": ("out", "q", *_POOL, "table", "lens", "cum", "alibi")}


def _operands(which, n=3, heads=8, kv=2, d=128, page=16, dtype=torch.bfloat16, index=torch.int64, alibi=False):
    u8 = torch.uint8
    rows = n if which == "" else 2 * n
    o = dict(out=torch.zeros((rows, heads, d), dtype=dtype), q=torch.zeros((rows, heads, d), dtype=dtype),
             table=torch.zeros((n, 4), dtype=index), lens=torch.zeros(n, dtype=index), cum=torch.zeros(n + 1, dtype=index),
             alibi=torch.zeros(heads) if alibi else None)
    for name in _POOL:
        o[name] = torch.zeros((6, kv, page, d // (2 if "codes" in name else 32)), dtype=u8)
    return o


def _create(lib, handle, which, operands, absent=None):
    descs = [lib.infiniopTensorDescriptor_t() if name == absent or operands[name] is None else describe(operands[name])
             for name in _ORDER[which]]
    op = lib.infiniopOperatorDescriptor_t()
    status = getattr(lib.LIBINFINIOP, f"infiniopCreatePagedAttention{which}Fp4Descriptor")(
        handle, ctypes.byref(op), *descs, ctypes.c_float(0.1))
    for d in descs:
        if d:
            lib.destroy_tensor_descriptor(d)
    if status == 0:
        size = ctypes.c_size_t(77)
        assert getattr(lib.LIBINFINIOP, f"infiniopGetPagedAttention{which}Fp4WorkspaceSize")(op, ctypes.byref(size)) == 0
        assert size.value != 77
        assert getattr(lib.LIBINFINIOP, f"infiniopDestroyPagedAttention{which}Fp4Descriptor")(op) == 0
    return status


@pytest.mark.parametrize("which", ["", "Prefill"])
def test_descriptors_accept(lib, host_amd_handle, which):
    for d in (64, 128, 192, 256):
        for dtype in (torch.float16, torch.bfloat16):
            for index in (torch.int64, torch.int32, torch.uint32):
                for n, page, alibi in ((0, 16, False), (1, 1, True), (70, 24, False)):
                    assert _create(lib, host_amd_handle, which, _operands(which, n, 8, 2, d, page, dtype, index, alibi)) == 0
    o = _operands(which)
    for name in _POOL:  # pages stored [rows, heads]
        o[name] = o[name].transpose(1, 2).contiguous().transpose(1, 2)
    o["q"] = torch.zeros((1, 1, 128), dtype=torch.bfloat16).expand(o["q"].shape)  # a query for all
    assert _create(lib, host_amd_handle, which, o) == 0
    o["out"] = torch.zeros((o["q"].shape[0], 9, 131), dtype=torch.bfloat16)[:, 1:, 2:130]
    assert _create(lib, host_amd_handle, which, o) == 0


@pytest.mark.parametrize("which", ["", "Prefill"])
def test_descriptors_refuse(lib, host_amd_handle, which):
    S = lib.InfiniStatus

    def status(**changed):
        return _create(lib, host_amd_handle, which, {**_operands(which), **changed})

    o = _operands(which)
    rows, bf16 = o["q"].shape[0], torch.bfloat16
    for name in _ORDER[which][:-1]:
        assert _create(lib, host_amd_handle, which, o, absent=name) == S.NULL_POINTER
    for name in _POOL:
        assert status(**{name: o[name].to(torch.int8)}) == S.BAD_TENSOR_DTYPE
        assert status(**{name: o[name][0]}) == S.BAD_TENSOR_SHAPE
        for short in (o[name][:-1], o[name][:, :-1], o[name][:, :, :-1], o[name][..., :-1]):
            assert status(**{name: short}) == S.BAD_TENSOR_SHAPE
        wide = torch.zeros((*o[name].shape[:3], 2 * o[name].shape[3]), dtype=torch.uint8)
        assert status(**{name: wide[..., ::2]}) == S.BAD_TENSOR_STRIDES
        # rows that do not all begin where 16 bytes of codes, or four scales, are loaded at once
        odd = torch.zeros((*o[name].shape[:3], o[name].shape[3] + (8 if "codes" in name else 2)), dtype=torch.uint8)
        assert status(**{name: odd[..., :o[name].shape[3]]}) == S.BAD_TENSOR_STRIDES
        # a page of more than 2^31 bytes
        far = torch.empty_strided((6, 2, 1 << 12, o[name].shape[3]), (1 << 40, 1 << 38, 1 << 20, 1), dtype=torch.uint8, device="meta")
        pages = {n: torch.empty((6, 2, 1 << 12, o[n].shape[3]), dtype=torch.uint8, device="meta") for n in _POOL}
        assert status(**pages) == 0 and status(**{**pages, name: far}) == S.BAD_TENSOR_STRIDES
    assert status(q=o["q"].float(), out=o["out"].float()) == S.BAD_TENSOR_DTYPE
    assert status(out=o["out"].half()) == S.BAD_TENSOR_DTYPE
    for name in ("q", "out"):
        for short in (o[name][0], o[name][:-1], o[name][:, :-1], o[name][..., :64]):
            assert status(**{name: short}) == S.BAD_TENSOR_SHAPE
        assert status(**{name: torch.zeros((rows, 8, 256), dtype=bf16)[..., ::2]}) == S.BAD_TENSOR_STRIDES
    for shape in ((1, 8, 128), (rows, 1, 128)):  # two results in one place
        assert status(out=torch.zeros(shape, dtype=bf16).expand(o["out"].shape)) == S.BAD_TENSOR_STRIDES
    assert _create(lib, host_amd_handle, which, _operands(which, d=96)) == S.BAD_TENSOR_SHAPE
    assert _create(lib, host_amd_handle, which, _operands(which, d=512)) == S.BAD_TENSOR_SHAPE
    assert _create(lib, host_amd_handle, which, _operands(which, heads=7)) == S.BAD_TENSOR_SHAPE
    assert status(table=o["table"].int()) == S.BAD_TENSOR_DTYPE
    assert status(table=o["table"].float(), lens=o["lens"].float()) == S.BAD_TENSOR_DTYPE
    assert status(table=o["table"][0]) == S.BAD_TENSOR_SHAPE
    assert status(table=o["table"][:-1]) == S.BAD_TENSOR_SHAPE
    assert status(table=torch.zeros((3, 8), dtype=torch.int64)[:, ::2]) == S.BAD_TENSOR_STRIDES
    assert status(lens=torch.zeros(6, dtype=torch.int64)[::2]) == S.BAD_TENSOR_STRIDES
    assert status(lens=o["lens"][:, None]) == S.BAD_TENSOR_SHAPE
    assert status(alibi=torch.zeros(8, dtype=torch.bfloat16)) == S.BAD_TENSOR_DTYPE
    assert status(alibi=torch.zeros(7)) == S.BAD_TENSOR_SHAPE
    assert status(alibi=torch.zeros((8, 1))) == S.BAD_TENSOR_SHAPE
    assert status(alibi=torch.zeros(16)[::2]) == S.BAD_TENSOR_STRIDES
    if which == "":
        assert status(lens=o["lens"][:-1]) != 0
    else:
        assert status(cum=o["cum"].int()) == S.BAD_TENSOR_DTYPE
        assert status(cum=o["cum"][:, None]) == S.BAD_TENSOR_SHAPE
        assert status(cum=o["cum"][:-1]) == S.BAD_PARAM
        assert status(cum=torch.zeros(8, dtype=torch.int64)[::2]) == S.BAD_TENSOR_STRIDES
        for rows, expected in ((1 << 24, 0), (1 << 28, S.BAD_TENSOR_SHAPE)):  # more rows than are counted
            q = torch.empty((rows, 8, 128), dtype=bf16, device="meta")
            assert status(q=q, out=q) == expected
        n = 65000  # more workgroups than a grid has
        heads = torch.empty((n, 260, 128), dtype=bf16, device="meta")
        pool = {name: torch.empty((6, 260, 16, o[name].shape[3]), dtype=torch.uint8, device="meta") for name in _POOL}
        rest = {name: torch.empty(size, dtype=torch.int64, device="meta") for name, size in (("table", (n, 4)), ("lens", n), ("cum", n + 1))}
        assert status(q=heads, out=heads, **pool, **rest) == S.BAD_TENSOR_SHAPE
    cpu = ctypes.pointer(lib.Handle(lib.InfiniDevice.CPU, 0))
    assert _create(lib, cpu, which, o) == S.DEVICE_TYPE_NOT_SUPPORTED
    assert _create(lib, None, which, o) == S.NULL_POINTER


def test_python_operators_refuse_host_tensors():
    from infinicore_amd import ops

    for which, run in (("", ops.paged_attention_fp4), ("Prefill", ops.paged_attention_prefill_fp4)):
        o = _operands(which)
        with pytest.raises(ValueError):
            run(*(o[name] for name in _ORDER[which][1:]), 0.1)
