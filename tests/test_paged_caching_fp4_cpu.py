"""The 4-bit pool without a GPU: the 64-bit restatement the GPU tests compare with, pinned by the format's own arithmetic, and
what the writer's and the reader's descriptors refuse."""
import ctypes
import itertools

import pytest
import torch

import fp4_reference as fp4
from capi import describe


def test_every_code_and_tie():
    # one group: 6 fixes the scale at 2^0, then every magnitude, every middle between two and its neighbourhood
    middles = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    to_even = [0, 2, 2, 4, 4, 6, 6]
    for m, code in zip(middles, to_even):
        x = torch.zeros(32, dtype=torch.float64)
        x[0], x[1], x[2], x[3], x[4] = 6.0, m, -m, m * (1 - 1e-6), m * (1 + 1e-6)
        codes, scales = fp4.quantise(x)
        assert scales.tolist() == [127]
        got = [int(c) for b in codes.tolist() for c in (b & 15, b >> 4)]
        lower = middles.index(m)
        assert got[:5] == [7, code, code + 8, lower, lower + 1]


def test_scale_rule():
    x = torch.zeros((8, 32), dtype=torch.float64)
    for i, top in enumerate([1.0, 1.99, 2.0, 7.99, 2.0 ** -30, 2.0 ** 20, 0.0, float("inf")]):
        x[i, 5] = top
    codes, scales = fp4.quantise(x)
    assert scales[:, 0].tolist() == [125, 125, 126, 127, 104, 140, 104, 255]
    back = fp4.values(codes, scales)
    assert back[0, 5] == 1.0 and back[1, 5] == 1.5 and back[2, 5] == 2.0 and back[3, 5] == 6.0  # (1.99 = 7.96 / 4: held at 6 / 4)
    assert back[4].abs().max() == 0 and back[5, 5] == 49152.0 and back[6].abs().max() == 0 and back[7].isnan().all()


def test_written_values_are_exact_in_16_bits():
    codes = torch.arange(256, dtype=torch.uint8).repeat(37, 1)[:, :, None].expand(-1, -1, 16)
    scales = torch.arange(104, 141, dtype=torch.uint8)[:, None, None].expand(-1, 256, 1)
    v = fp4.values(codes, scales)
    assert torch.equal(v.to(torch.float16).double(), v) and torch.equal(v.to(torch.bfloat16).double(), v)


def test_error_of_a_group():
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((500, 32), generator=gen, dtype=torch.float64)
    codes, scales = fp4.quantise(x)
    unit = torch.pow(2.0, scales.double() - 127)
    # inside 6 units half a step of at most 2; between 6 and 8 units held at 6
    assert ((fp4.values(codes, scales) - x).abs() <= torch.where(x.abs() <= 6 * unit, 1.0, 2.0) * unit).all()


# ---- descriptors ----

def _operands(n=5, heads=4, d=64, dv=64, blocks=6, page=16, dtype=torch.bfloat16):
    u8 = torch.uint8
    return dict(k_codes=torch.zeros((blocks, heads, page, d // 2), dtype=u8), v_codes=torch.zeros((blocks, heads, page, dv // 2), dtype=u8),
                k_scales=torch.zeros((blocks, heads, page, d // 32), dtype=u8), v_scales=torch.zeros((blocks, heads, page, dv // 32), dtype=u8),
                k=torch.zeros((n, heads, d), dtype=dtype), v=torch.zeros((n, heads, dv), dtype=dtype), slots=torch.zeros(n, dtype=torch.int64))


_POOL = ("k_codes", "v_codes", "k_scales", "v_scales")
_ORDER = {"Caching": (*_POOL, "k", "v", "slots"), "Reading": ("k", "v", *_POOL, "slots")}


def _create(lib, handle, which, operands, absent=None):
    descs = [lib.infiniopTensorDescriptor_t() if name == absent else describe(operands[name]) for name in _ORDER[which]]
    op = lib.infiniopOperatorDescriptor_t()
    status = getattr(lib.LIBINFINIOP, f"infiniopCreatePaged{which}Fp4Descriptor")(handle, ctypes.byref(op), *descs)
    for d in descs:
        if d:
            lib.destroy_tensor_descriptor(d)
    if status == 0:
        size = ctypes.c_size_t(77)
        assert getattr(lib.LIBINFINIOP, f"infiniopGetPaged{which}Fp4WorkspaceSize")(op, ctypes.byref(size)) == 0 and size.value == 0
        assert getattr(lib.LIBINFINIOP, f"infiniopDestroyPaged{which}Fp4Descriptor")(op) == 0
    return status


@pytest.mark.parametrize("which", ["Caching", "Reading"])
def test_descriptors_accept(lib, host_amd_handle, which):
    for dtype, d, page, n in itertools.product((torch.bfloat16, torch.float16, torch.float32), (32, 64, 96, 256, 576), (1, 7, 16), (0, 1, 5)):
        assert _create(lib, host_amd_handle, which, _operands(n=n, d=d, page=page, dtype=dtype)) == 0
    o = _operands(d=576, dv=512)
    assert _create(lib, host_amd_handle, which, o) == 0
    o = _operands()
    for name in _POOL:  # pages stored [rows, heads]
        o[name] = o[name].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros((5, 12, 64), dtype=torch.bfloat16)
    o["k"], o["v"] = wide[:, :4], wide[:, 4:8]
    assert _create(lib, host_amd_handle, which, o) == 0


@pytest.mark.parametrize("which", ["Caching", "Reading"])
def test_descriptors_refuse(lib, host_amd_handle, which):
    S = lib.InfiniStatus

    def status(**changed):
        return _create(lib, host_amd_handle, which, {**_operands(), **changed})

    o = _operands()
    for name in _ORDER[which]:
        assert _create(lib, host_amd_handle, which, o, absent=name) == S.NULL_POINTER
    for name in _POOL:
        assert status(**{name: o[name].to(torch.int8)}) == S.BAD_TENSOR_DTYPE
        assert status(**{name: o[name][0]}) == S.BAD_TENSOR_SHAPE
        assert status(**{name: o[name][:-1]}) == S.BAD_TENSOR_SHAPE
        assert status(**{name: o[name][:, :-1]}) == S.BAD_TENSOR_SHAPE
        assert status(**{name: o[name][:, :, :-1]}) == S.BAD_TENSOR_SHAPE
        assert status(**{name: o[name][..., :-1]}) == S.BAD_TENSOR_SHAPE
        wide = torch.zeros((*o[name].shape[:3], 2 * o[name].shape[3]), dtype=torch.uint8)
        assert status(**{name: wide[..., ::2]}) == S.BAD_TENSOR_STRIDES
    for name in ("k", "v"):
        assert status(**{name: o[name].to(torch.float16)}) == S.BAD_TENSOR_DTYPE
        assert status(**{name: o[name][0]}) == S.BAD_TENSOR_SHAPE
        assert status(**{name: o[name][:-1]}) == S.BAD_TENSOR_SHAPE
        assert status(**{name: o[name][:, :-1]}) == S.BAD_TENSOR_SHAPE
        assert status(**{name: o[name][..., :32]}) == S.BAD_TENSOR_SHAPE
        assert status(**{name: torch.zeros((5, 4, 128), dtype=torch.bfloat16)[..., ::2]}) == S.BAD_TENSOR_STRIDES
        broadcast = torch.zeros((1, 4, 64), dtype=torch.bfloat16).expand(5, -1, -1)
        assert status(**{name: broadcast}) == (0 if which == "Caching" else S.BAD_TENSOR_STRIDES)
    assert status(k=o["k"].to(torch.int16), v=o["v"].to(torch.int16)) == S.BAD_TENSOR_DTYPE
    assert status(slots=o["slots"].int()) == S.BAD_TENSOR_DTYPE
    assert status(slots=o["slots"][:-1]) == S.BAD_TENSOR_SHAPE
    assert status(slots=torch.zeros(10, dtype=torch.int64)[::2]) == S.BAD_TENSOR_STRIDES
    tokens = 1 << 30  # counted in 32 bits
    many = {name: torch.empty((tokens, *o[name].shape[1:]), dtype=o[name].dtype, device="meta") for name in ("k", "v", "slots")}
    assert status(**many) == S.BAD_TENSOR_SHAPE
    wide = {name: torch.empty((*o[name].shape[:-1], o[name].shape[-1] << 22), dtype=o[name].dtype, device="meta") for name in (*_POOL, "k", "v")}
    assert status(**wide) == S.BAD_TENSOR_SHAPE
    cpu = ctypes.pointer(lib.Handle(lib.InfiniDevice.CPU, 0))
    assert _create(lib, cpu, which, o) == S.DEVICE_TYPE_NOT_SUPPORTED
    assert _create(lib, None, which, o) == S.NULL_POINTER


def test_python_operators_refuse_host_tensors():
    from infinicore_amd import ops

    o = _operands()
    pool = [o[name] for name in _POOL]
    with pytest.raises(ValueError):
        ops.paged_caching_fp4(*pool, o["k"], o["v"], o["slots"])
    with pytest.raises(ValueError):
        ops.paged_reading_fp4(*pool, o["slots"])
    with pytest.raises(ValueError):
        ops.paged_reading_fp4(*pool, o["slots"], dtype=torch.float64)
