"""GPU parity of infiniopPagedAttentionFp4 with the 64-bit restatement (tests/fp4_reference.py, where the allowance is
derived): lengths around the tile, step and page borders, head layouts and sizes, strides, poisoned rows behind the sequences."""
import ctypes
import math

import pytest
import torch

import fp4_reference as fp4
from capi import describe, ptr
from infinicore_amd import libinfiniop as L
from infinicore_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN_BYTE = fp4.NAN_BYTE


def reference(b, lens, slopes=None, scale=None):
    """(outputs, allowed), rows of empty sequences NaN."""
    q, pool = b["q"], b["pool"]
    scale = b["scale"] if scale is None else scale
    outs, allows = [], []
    for i, n in enumerate(lens):
        if n <= 0:
            outs.append(torch.full_like(q[i:i + 1], math.nan, dtype=torch.float64))
            allows.append(torch.zeros_like(outs[-1]))
            continue
        pages = b["table"][i, :b["needed"][i]].long()
        k, v = fp4.sequence(pool[0], pool[2], pages, n), fp4.sequence(pool[1], pool[3], pages, n)
        o, w = fp4.attention(q[i:i + 1], k, v, scale, [n - 1], slopes)
        outs.append(o)
        allows.append(w)
    return torch.cat(outs), torch.cat(allows)


def check(b, lens, slopes=None, out=None, scale=None):
    want, allowed = reference(b, lens, slopes, scale)
    if out is None:
        out = torch.full_like(b["q"], 7.0)
    got = ops.paged_attention_fp4(b["q"], *b["pool"], b["table"], b["lens"], slopes, b["scale"] if scale is None else scale, out=out)
    assert got is out
    torch.cuda.synchronize()
    empty = torch.tensor([n <= 0 for n in lens], device=DEV)
    assert (got[empty] == 7.0).all(), "a sequence without tokens"
    off = fp4.off_by(got[~empty], want[~empty], allowed[~empty])
    print("off by", off, flush=True)
    assert off <= 1.0, off
    return got


BORDERS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 127, 129, -3, 500, 777]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 32, 8, 24, 1, 7, 48])
def test_lengths_sizes_pages(dtype, d, page):
    print("case", dtype, d, page, flush=True)
    check(fp4.make_batch(d + page, BORDERS, 8, 2, d, page, dtype), BORDERS)


# A table that could hold far more tokens than the sequences have: their steps are cut into equal runs.
WIDE = 1 << 16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 32, 8, 24, 1, 7, 48])
def test_cut_lengths_sizes_pages(dtype, d, page):
    print("case", dtype, d, page, flush=True)
    check(fp4.widen(fp4.make_batch(d + page, BORDERS, 8, 2, d, page, dtype), WIDE), BORDERS)


@pytest.mark.parametrize("sequences", [1, 3, 65, 200])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (40, 1), (3, 3), (34, 2)])
def test_cut_parts_of_a_row(sequences, heads, kv_heads):
    """Joined by one wavefront, by four and by sixteen; more sequences than lanes; pairs of KV heads and single ones."""
    lens = [(137 * i) % 400 + (3000 if i == 0 else 0) for i in range(sequences)]
    slopes = torch.tensor([2.0 ** (-h / 4) for h in range(heads)], device=DEV)
    for index in (torch.int64, torch.int32, torch.uint32):
        b = fp4.widen(fp4.make_batch(21, lens, heads, kv_heads, 128, 16, torch.bfloat16, index=index, layout="padded"), WIDE)
        check(b, lens)
        check(b, lens, slopes)


def test_cut_and_whole_agree_on_a_nan():
    lens = [70, 1000, 129]
    b = fp4.widen(fp4.make_batch(11, lens, 8, 2, 128, 16, torch.bfloat16), WIDE)
    clean = check(b, lens)
    b["pool"][3][int(b["table"][1, 17]), 1, 5, 2] = NAN_BYTE
    got = ops.paged_attention_fp4(b["q"], *b["pool"], b["table"], b["lens"], None, b["scale"])
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[1, 4:, 64:96] = True
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean[~nan])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (32, 8), (40, 8), (28, 4), (48, 8), (16, 1), (17, 1), (64, 2), (40, 1), (3, 3)])
def test_head_layouts(dtype, heads, kv_heads):
    print("case", dtype, heads, kv_heads, flush=True)
    lens = [1, 70, 333, 0, 1025]
    check(fp4.make_batch(heads, lens, heads, kv_heads, 128, 16, dtype), lens)


@pytest.mark.parametrize("index", [torch.int64, torch.int32, torch.uint32])
@pytest.mark.parametrize("layout", ["packed", "rows", "padded"])
def test_indices_and_layouts(index, layout):
    lens = [5, 0, 200, 64, 1]
    check(fp4.make_batch(3, lens, 16, 4, 128, 16, torch.bfloat16, index=index, layout=layout), lens)


@pytest.mark.parametrize("d,page", [(64, 16), (128, 8), (192, 16), (256, 5)])
def test_query_and_output_strides(d, page):
    lens = [40, 3, 0, 130]
    b = fp4.make_batch(9, lens, 12, 4, d, page, torch.float16)
    fused = torch.zeros((4, 20, d), dtype=torch.float16, device=DEV)  # q as a slice of a projection
    fused[:, 3:15] = b["q"]
    odd = torch.zeros((4, 12, d + 1), dtype=torch.float16, device=DEV)
    odd[..., 1:] = b["q"]
    for q in (fused[:, 3:15], odd[..., 1:], b["q"].transpose(0, 1).contiguous().transpose(0, 1)):
        b["q"] = q
        check(b, lens)
        wide = torch.full((4, 13, d + 3), 7.0, dtype=torch.float16, device=DEV)
        check(b, lens, out=wide[:, 1:, 1:d + 1])
        assert (wide[:, 0] == 7.0).all() and (wide[..., 0] == 7.0).all() and (wide[..., d + 1:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_alibi(dtype, d):
    lens = [1, 100, 0, 1531, 64]
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / 16) for h in range(16)], device=DEV)
    check(fp4.make_batch(4, lens, 16, 16, d, 32, dtype, index=torch.int32), lens, slopes)
    slopes = torch.cat((-slopes[:6], torch.zeros(6, device=DEV)))  # rising with the distance, and none
    check(fp4.make_batch(5, lens, 10, 2, d, 16, dtype), lens, slopes)


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
def test_scales(scale):
    lens = [1, 90, 300]
    check(fp4.make_batch(6, lens, 8, 2, 128, 16, torch.bfloat16), lens, scale=scale)


@pytest.mark.parametrize("page", [16, 7])
def test_one_long_sequence_and_many_short(page):
    check(fp4.make_batch(7, [40001], 16, 2, 128, page, torch.bfloat16), [40001])
    lens = [(37 * i) % 90 for i in range(333)]
    check(fp4.make_batch(8, lens, 8, 2, 64, page, torch.float16), lens)
    lens = [3, 9000, 1, 0, 5000, 2]
    check(fp4.make_batch(8, lens, 32, 8, 128, page, torch.float16), lens)


def test_climbing_scores():
    """The maximum moves in every tile, below and above the threshold for moving the reference point."""
    lens = [900, 2100]
    for hot in (1.0, 30.0, 300.0):
        b = fp4.make_batch(10, lens, 8, 2, 128, 16, torch.bfloat16, hot=hot)
        for i, n in enumerate(lens):  # later rows hold larger keys along the query
            pages = b["table"][i, :b["needed"][i]].long()
            order = torch.arange(len(pages) * 16, device=DEV).view(-1, 1, 16, 1)
            scales = b["pool"][2][pages]
            b["pool"][2][pages] = torch.where(scales == 255, 255, (110 + order * 14 // (len(pages) * 16)).to(torch.uint8))
        check(b, lens)


def test_a_visible_nan_stays_in_its_sequence_and_head():
    lens = [70, 300, 129]
    b = fp4.make_batch(11, lens, 8, 2, 128, 16, torch.bfloat16)
    clean = check(b, lens)
    page = int(b["table"][1, 17])
    b["pool"][2][page, 1, 5, 2] = NAN_BYTE  # a key of sequence 1, KV head 1
    got = ops.paged_attention_fp4(b["q"], *b["pool"], b["table"], b["lens"], None, b["scale"])
    assert got[1, 4:].isnan().all() and torch.equal(got[1, :4], clean[1, :4])
    assert torch.equal(got[[0, 2]], clean[[0, 2]])
    b["pool"][2][page, 1, 5, 2] = 120
    clean = check(b, lens)
    b["pool"][3][page, 1, 5, 2] = NAN_BYTE  # a group of a value: columns 64 .. 95
    got = ops.paged_attention_fp4(b["q"], *b["pool"], b["table"], b["lens"], None, b["scale"])
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[1, 4:, 64:96] = True
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean[~nan])


def test_products_that_overflow():
    """Queries so large that products with keys are infinite in 32 bits: -inf has no weight, +inf and NaN reach the output."""
    lens = [100]
    b = fp4.make_batch(12, lens, 1, 1, 64, 16, torch.bfloat16)
    codes = torch.zeros_like(b["pool"][0])
    codes[..., 0] = 0x0F  # -6 in the first element of every key
    pages = b["table"][0, :7].long()
    codes[pages[2], 0, 3, 0] = 0x00  # but of one token, whose score is 0
    b["pool"][0], b["pool"][2] = codes, torch.where(b["pool"][2] == 255, 255, 140).to(torch.uint8)
    b["q"][:] = 0
    b["q"][..., 0] = 3e38
    got = ops.paged_attention_fp4(b["q"], *b["pool"], b["table"], b["lens"], None, 1.0)
    v = fp4.sequence(b["pool"][1], b["pool"][3], pages, 100)[0, 35]
    torch.testing.assert_close(got[0, 0].double(), v, rtol=2 ** -8, atol=0)
    b["q"][..., 0] = -3e38
    assert ops.paged_attention_fp4(b["q"], *b["pool"], b["table"], b["lens"], None, 1.0).isnan().all()


def test_page_order_repeats_and_lengths_beyond_the_table():
    lens = [333, 1000, 17]
    b = fp4.make_batch(13, lens, 8, 2, 128, 16, torch.float16)
    first = check(b, lens)
    assert torch.equal(check(b, lens), first)
    blocks = b["pool"][0].shape[0]
    perm = torch.randperm(blocks, device=DEV)
    moved = dict(b, pool=[t[perm] for t in b["pool"]])
    back = torch.argsort(perm)
    table = b["table"].clone()
    for i, n in enumerate(b["needed"]):
        table[i, :n] = back[table[i, :n]]
    moved["table"] = table
    assert torch.equal(check(moved, lens), first)
    # one page for two sequences, and twice in one
    table = b["table"].clone()
    table[2, :2] = table[0, :2]
    table[0, 3] = table[0, 0]
    check(dict(b, table=table), lens)
    # longer than the table: cut to it, its entries forced into the pool
    short = dict(b, table=b["table"][:, :20], needed=[20, 20, 2], lens=torch.tensor([320, 1 << 40, 17], device=DEV))
    check(short, [320, 320, 17])


def test_offsets_past_32_bits():
    d, page, kv = 128, 16, 8
    blocks = (9 << 29) // (kv * page * d // 2)  # 4.8e9 bytes of codes
    pool = [torch.zeros((blocks, kv, page, w), dtype=torch.uint8, device=DEV) for w in (64, 64, 4, 4)]
    table = torch.stack((torch.arange(5), blocks - 1 - torch.arange(5))).to(DEV)
    small = fp4.make_pool(1, 10, kv, page, d)
    for big, t in zip(pool, small):
        big[table.flatten()] = t.to(DEV)
    b = dict(q=torch.randn((2, 32, d), generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV), pool=pool, table=table,
             lens=torch.tensor([77, 80], device=DEV), needed=[5, 5], scale=0.1)
    check(b, [77, 80])


def test_streams_and_graphs():
    lens = [300, 40, 1200]
    b = fp4.make_batch(14, lens, 32, 8, 128, 16, torch.bfloat16, poison=False)
    args = (b["q"], *b["pool"], b["table"], b["lens"], None, b["scale"])
    eager = ops.paged_attention_fp4(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.paged_attention_fp4(*args)
    side.synchronize()
    assert torch.equal(eager, other)
    graphs = []
    for _ in range(2):  # two graphs of one call have scratch of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_attention_fp4(*args)
        graphs.append((graph, out))
    ops.clear_plan_cache()
    for turn, now in enumerate(([300, 40, 1200], [16, 2, 1199], [0, 41, 700])):
        b["lens"].copy_(torch.tensor(now))
        want = ops.paged_attention_fp4(*args, out=torch.zeros_like(eager))
        for graph, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):  # both at once
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want), turn


def test_c_entry_points():
    lens = [100, 2000]
    b = fp4.make_batch(15, lens, 16, 4, 128, 16, torch.bfloat16)
    out = torch.full_like(b["q"], 7.0)
    tensors = [out, b["q"], *b["pool"], b["table"], b["lens"]]
    L.set_device(L.InfiniDevice.AMD, 0)
    handle = L.create_handle()
    descs = [describe(t) for t in tensors]
    op = L.infiniopOperatorDescriptor_t()
    L.check_error(L.LIBINFINIOP.infiniopCreatePagedAttentionFp4Descriptor(handle, ctypes.byref(op), *descs,
                                                                          L.infiniopTensorDescriptor_t(), b["scale"]))
    for d in descs:
        L.destroy_tensor_descriptor(d)
    size = ctypes.c_size_t(0)
    L.check_error(L.LIBINFINIOP.infiniopGetPagedAttentionFp4WorkspaceSize(op, ctypes.byref(size)))
    want, allowed = reference(b, lens)
    run = lambda ws, n, *p: L.LIBINFINIOP.infiniopPagedAttentionFp4(op, ws, n, *p, None, None)  # noqa: E731
    pointers = [ptr(t) for t in tensors]
    for fill in (0, 255, 77):
        workspace = torch.full((size.value + 1,), fill, dtype=torch.uint8, device=DEV)
        torch.cuda.synchronize()
        for offset in (0, 1):
            L.check_error(run(ctypes.c_void_p(workspace.data_ptr() + offset), size.value, *pointers))
            torch.cuda.synchronize()
            assert fp4.off_by(out, want, allowed) <= 1.0
    S = L.InfiniStatus
    assert run(ptr(workspace), size.value - 1, *pointers) == S.INSUFFICIENT_WORKSPACE
    assert run(None, size.value, *pointers) == S.INSUFFICIENT_WORKSPACE
    for i in range(len(pointers)):
        assert run(ptr(workspace), size.value, *pointers[:i], None, *pointers[i + 1:]) == S.NULL_POINTER
    for i in (2, 3):
        assert run(ptr(workspace), size.value, *pointers[:i], ctypes.c_void_p(pointers[i].value + 8), *pointers[i + 1:]) == S.BAD_PARAM
    L.check_error(L.LIBINFINIOP.infiniopDestroyPagedAttentionFp4Descriptor(op))
    L.destroy_handle(handle)
