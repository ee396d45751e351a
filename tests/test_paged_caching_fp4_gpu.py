"""GPU parity of infiniopPagedCachingFp4 and infiniopPagedReadingFp4: codes, scales and values against the 64-bit
restatement, all equal (scales are powers of two, so every code and every value has one right answer)."""
import ctypes

import pytest
import torch

import fp4_reference as fp4
from capi import describe, ptr
from infinicore_amd import libinfiniop as L
from infinicore_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
POOL = ("k_codes", "v_codes", "k_scales", "v_scales")


def empty_pool(blocks, heads, page, d, dv, layout="packed"):
    made = []
    for width in (d // 2, dv // 2, d // 32, dv // 32):
        if layout == "packed":
            t = torch.full((blocks, heads, page, width), 0x5A, dtype=torch.uint8)
        elif layout == "rows":  # stored [pages, rows, heads]
            t = torch.full((blocks, page, heads, width), 0x5A, dtype=torch.uint8).transpose(1, 2)
        else:  # rows at odd distances: nothing is aligned
            t = torch.full((blocks, heads, page, width + 3), 0x5A, dtype=torch.uint8)[..., 1:1 + width]
        made.append(t)
    return made


def to_device(t):
    """With the strides it has on the host."""
    base = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=DEV)
    return base.copy_(t)


def run_c(which, tensors, stream=0):
    """The C entry points, as capi.py drives the others."""
    L.set_device(L.InfiniDevice.AMD, 0)
    handle = L.create_handle()
    descs = [describe(t) for t in tensors]
    op = L.infiniopOperatorDescriptor_t()
    L.check_error(getattr(L.LIBINFINIOP, f"infiniopCreatePaged{which}Fp4Descriptor")(handle, ctypes.byref(op), *descs))
    for d in descs:
        L.destroy_tensor_descriptor(d)
    torch.cuda.synchronize()
    L.check_error(getattr(L.LIBINFINIOP, f"infiniopPaged{which}Fp4")(op, None, 0, *[ptr(t) for t in tensors], ctypes.c_void_p(stream)))
    torch.cuda.synchronize()
    L.check_error(getattr(L.LIBINFINIOP, f"infiniopDestroyPaged{which}Fp4Descriptor")(op))
    L.destroy_handle(handle)


def written(pool, k, v, slots):
    """The host pool after the write."""
    pool = [t.clone() for t in pool]
    page = pool[0].shape[2]
    for x, codes, scales in ((k, pool[0], pool[2]), (v, pool[1], pool[3])):
        c, s = fp4.quantise(x)
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < codes.shape[0] * page:
                codes[slot // page, :, slot % page] = c[i]
                scales[slot // page, :, slot % page] = s[i]
    return pool


def check(k, v, slots, blocks, page, layout="packed", source="packed"):
    print("case", tuple(k.shape), tuple(v.shape), k.dtype, page, layout, source, flush=True)
    heads, d, dv = k.shape[1], k.shape[2], v.shape[2]
    pool = empty_pool(blocks, heads, page, d, dv, layout)
    want = written(pool, k, v, slots)
    got = [to_device(t) for t in pool]
    if source == "slices":  # of one projection output
        both = torch.cat((k, v), dim=-1).to(DEV)
        kd, vd = both[..., :d], both[..., d:]
    elif source == "odd":
        kd = torch.empty((k.shape[0], heads, d + 1), dtype=k.dtype, device=DEV)[..., 1:].copy_(k)
        vd = torch.empty((v.shape[0], heads, dv + 1), dtype=v.dtype, device=DEV)[..., 1:].copy_(v)
    else:
        kd, vd = k.to(DEV), v.to(DEV)
    run_c("Caching", (*got, kd, vd, slots.to(DEV)))
    for name, g, w in zip(POOL, got, want):
        assert torch.equal(g.cpu(), w), name

    held = ((slots >= 0) & (slots < blocks * page))[:, None, None]
    at = slots.clamp(0, blocks * page - 1)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        ko, vo = torch.full(k.shape, 7.0, dtype=dtype, device=DEV), torch.full(v.shape, 7.0, dtype=dtype, device=DEV)
        if source == "odd":
            ko = torch.full((k.shape[0], heads, d + 3), 7.0, dtype=dtype, device=DEV)[..., 1:1 + d]
        run_c("Reading", (ko, vo, *got, slots.to(DEV)))
        for o, codes, scales in ((ko, want[0], want[2]), (vo, want[1], want[3])):
            x = fp4.values(codes[at // page, :, at % page], scales[at // page, :, at % page])
            x = torch.where(held, x, 0.0)
            torch.testing.assert_close(o.cpu().double(), x, rtol=0, atol=0, equal_nan=True)
        if source == "odd":
            assert (ko.as_strided((k.shape[0], heads), (ko.stride(0), ko.stride(1)), ko.storage_offset() + d) == 7.0).all()


def random_tokens(seed, n, heads, d, dv, dtype):
    gen = torch.Generator().manual_seed(seed)
    size = torch.exp(3 * torch.randn((1, heads, d), generator=gen))
    return (torch.randn((n, heads, d), generator=gen) * size).to(dtype), torch.randn((n, heads, dv), generator=gen).to(dtype)


def random_slots(seed, n, room, padding=0):
    slots = torch.randperm(room, generator=torch.Generator().manual_seed(seed))[:n]
    slots[:padding] = torch.tensor([-1, -5, room, 1 << 40])[torch.arange(padding) % 4]
    return slots


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,heads,d,dv,page", [
    (1, 8, 128, 128, 16), (300, 8, 128, 128, 16), (37, 16, 64, 64, 32), (9, 5, 192, 192, 24), (11, 1, 256, 256, 7),
    (6, 3, 32, 32, 1), (5, 1, 576, 512, 16), (7, 2, 96, 32, 8), (3, 40, 256, 256, 128)])
def test_shapes(dtype, n, heads, d, dv, page):
    k, v = random_tokens(n + d, n, heads, d, dv, dtype)
    blocks = -(-2 * n // page) + 2
    check(k, v, random_slots(n, n, blocks * page, padding=min(n // 2, 5)), blocks, page)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout,source", [("rows", "packed"), ("packed", "slices"), ("odd", "packed"), ("packed", "odd"),
                                           ("odd", "odd")])
def test_layouts(dtype, layout, source):
    k, v = random_tokens(5, 21, 4, 128, 64, dtype)
    check(k, v, random_slots(2, 21, 4 * 16, padding=3), 4, 16, layout, source)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value_as_the_largest_and_below(dtype):
    """Each of the 65 536 bit patterns heads a group with smaller ones of both signs; infinities and NaN among them."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    scaled = [x.float() * f for f in (1.0, -0.9, 0.77, 0.5, -0.3, 0.126, 0.0, -0.0)]
    k = torch.stack([s.to(dtype) for s in scaled], dim=-1).repeat(1, 4)[:, None, :]  # [65536, 1, 32]
    v = x.view(-1, 32)[torch.arange(65536) // 32 % 2048][:, None, :].contiguous()
    check(k, v, torch.arange(65536), 4096, 16)


def test_fp32_extremes():
    tops = torch.tensor([0.0, 1e-45, 1e-38, 2.0 ** -25, 2.0 ** -24, 2.0 ** -21, 1.0, 49151.9, 49152.0, 65504.0, 3e38, float("inf"),
                         float("-inf"), float("nan")])
    k = torch.randn((len(tops), 1, 32), generator=torch.Generator().manual_seed(0)).sign() * tops[:, None, None]
    k[:, 0, 1:] *= torch.linspace(1, 0, 31)
    k = torch.where(torch.isnan(k) & ~torch.isnan(tops)[:, None, None], 0.0, k)
    check(k, k.flip(0), torch.arange(len(tops)), 1, 16)


def test_scales_that_were_not_written_here():
    """A pool from elsewhere: every scale byte reads as 2^(s - 127), rounded once."""
    codes = torch.arange(16, dtype=torch.uint8) * 17
    codes = codes.expand(256, 1, 1, 16).contiguous()
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1, 1, 1)
    want = fp4.values(codes, scales)[:, :, 0]
    pool = [t.to(DEV) for t in (codes, codes, scales, scales)]
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        k, v = ops.paged_reading_fp4(*pool, torch.arange(256, device=DEV), dtype=dtype)
        assert k.dtype == dtype
        torch.testing.assert_close(k.cpu(), want.to(dtype), rtol=0, atol=0, equal_nan=True)
        torch.testing.assert_close(v.cpu(), want.to(dtype), rtol=0, atol=0, equal_nan=True)


def test_offsets_past_32_bits():
    heads, page, d = 8, 16, 128
    blocks = (9 << 29) // (heads * page * d // 2)  # 4.8e9 bytes of codes
    pool = [torch.zeros((blocks, heads, page, w), dtype=torch.uint8, device=DEV) for w in (64, 64, 4, 4)]
    k, v = random_tokens(1, 40, heads, d, d, torch.bfloat16)
    slots = torch.cat((torch.arange(20), blocks * page - 1 - torch.arange(20)))
    ops.paged_caching_fp4(*pool, k.to(DEV), v.to(DEV), slots.to(DEV))
    got = ops.paged_reading_fp4(*pool, slots.to(DEV), dtype=torch.float32)
    for g, x in zip(got, (k, v)):
        assert torch.equal(g.cpu().double(), fp4.values(*fp4.quantise(x)))


def test_nothing_to_do():
    pool = [t.to(DEV) for t in empty_pool(3, 2, 16, 64, 64)]
    before = [t.clone() for t in pool]
    none = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device=DEV)
    ops.paged_caching_fp4(*pool, none, none, torch.zeros(0, dtype=torch.int64, device=DEV))
    k, v = ops.paged_reading_fp4(*pool, torch.zeros(0, dtype=torch.int64, device=DEV))
    assert k.shape == v.shape == (0, 2, 64)
    away = torch.tensor([-1, 48, -9223372036854775808, 9223372036854775807], device=DEV)
    ops.paged_caching_fp4(*pool, *(torch.ones((4, 2, 64), dtype=torch.bfloat16, device=DEV),) * 2, away)
    assert all(torch.equal(a, b) for a, b in zip(pool, before))
    k, v = ops.paged_reading_fp4(*pool, away)
    assert not k.any() and not v.any()
    hollow = [t[:0] for t in pool]
    k, v = ops.paged_reading_fp4(*hollow, away)
    assert not k.any() and not v.any()


def test_python_operators_streams_and_graphs():
    pool = [t.to(DEV) for t in empty_pool(64, 4, 16, 128, 128)]
    k, v = random_tokens(8, 100, 4, 128, 128, torch.float16)
    slots = random_slots(3, 100, 1024, padding=4)
    want = written([t.cpu() for t in pool], k, v, slots)
    kd, vd, sd = k.to(DEV), v.to(DEV), slots.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        same = ops.paged_caching_fp4(*pool, kd, vd, sd)
        ko, vo = ops.paged_reading_fp4(*pool, sd, dtype=torch.float16)
    side.synchronize()
    assert all(a is b for a, b in zip(same, pool))
    assert all(torch.equal(g.cpu(), w) for g, w in zip(pool, want))
    eager = (ko.clone(), vo.clone())

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_caching_fp4(*pool, kd, vd, sd)
        gk, gv = ops.paged_reading_fp4(*pool, sd, dtype=torch.float16)
    for turn in range(3):
        for t in pool:
            t.fill_(0x5A)
        gk.fill_(3)
        kd.copy_((k * (turn + 1)).to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        again = written([torch.full_like(t, 0x5A) for t in want], k * (turn + 1), v, slots)
        assert all(torch.equal(g.cpu(), w) for g, w in zip(pool, again))
        assert torch.equal(gv, eager[1]) and (turn or torch.equal(gk, eager[0]))
        ops.paged_reading_fp4(*pool, sd)  # eager work between the replays

    out = torch.empty_like(kd)
    k2, v2 = ops.paged_reading_fp4(*pool, sd, k=out)
    assert k2 is out and v2.dtype == torch.float16
    torch.testing.assert_close(k2, gk, rtol=0, atol=0, equal_nan=True)


def test_python_operators_refuse():
    pool = [t.to(DEV) for t in empty_pool(4, 4, 16, 128, 128)]
    k, v = (t.to(DEV) for t in random_tokens(8, 10, 4, 128, 128, torch.float16))
    slots = torch.arange(10, device=DEV)
    with pytest.raises(ValueError):
        ops.paged_caching_fp4(*pool, k, v, slots.cpu())
    with pytest.raises(ValueError):
        ops.paged_reading_fp4(*pool[:3], pool[3].cpu(), slots)
    with pytest.raises(L.InfiniStatusError):
        ops.paged_caching_fp4(*pool, k, v.float(), slots)
    with pytest.raises(L.InfiniStatusError):
        ops.paged_caching_fp4(*pool, k[:, :2], v[:, :2], slots)
    with pytest.raises(IndexError):
        ops.paged_reading_fp4(pool[0][0], *pool[1:], slots)
