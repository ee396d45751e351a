"""GPU parity of infiniopPagedAttentionPrefillFp4 with the 64-bit restatement (tests/fp4_reference.py, where the allowance is
derived): runs and histories around the tile, step and row-block borders, head layouts and sizes, strides, masks that leave a
row nothing, values that are not finite behind what a row sees."""
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


def make_runs(seed, runs, heads, kv_heads, d, page, dtype, *, lead=0, behind=0, **more):
    """runs: (new tokens, history) of each sequence; `lead` and `behind` rows of q belong to nobody."""
    lens = [n + h for n, h in runs]
    total = sum(n for n, _ in runs)
    b = fp4.make_batch(seed, lens, heads, kv_heads, d, page, dtype, rows=lead + total + behind, **more)
    cum = [lead]
    for n, _ in runs:
        cum.append(cum[-1] + n)
    b.update(runs=runs, cum=torch.tensor(cum).to(b["table"].dtype).to(DEV), starts=cum)
    return b


def reference(b, slopes=None):
    """(outputs, allowed, rows that are written)."""
    q, pool = b["q"], b["pool"]
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=DEV)
    allowed = torch.zeros_like(out)
    rows = torch.zeros(q.shape[0], dtype=torch.bool, device=DEV)
    for i, (n, h) in enumerate(b["runs"]):
        if n <= 0 or n + h <= 0:
            continue
        at = slice(b["starts"][i], b["starts"][i] + n)
        pages = b["table"][i, :b["needed"][i]].long()
        k, v = fp4.sequence(pool[0], pool[2], pages, n + h), fp4.sequence(pool[1], pool[3], pages, n + h)
        last = [h + j for j in range(n)]
        out[at], allowed[at] = fp4.attention(q[at], k, v, b["scale"], last, slopes, terms=True)
        rows[at] = torch.tensor([x >= 0 for x in last], device=DEV)
    return out, allowed, rows


def check(b, slopes=None, out=None):
    want, allowed, rows = reference(b, slopes)
    if out is None:
        out = torch.full_like(b["q"], 7.0)
    got = ops.paged_attention_prefill_fp4(b["q"], *b["pool"], b["table"], b["lens"], b["cum"], slopes, b["scale"], out=out)
    assert got is out
    torch.cuda.synchronize()
    assert (got[~rows] == 7.0).all(), "rows of nobody, or that see nothing"
    assert torch.equal(got[rows].isnan(), want[rows].isnan()), "not finite"
    off = fp4.off_by(got[rows].nan_to_num(), want[rows].nan_to_num(), allowed[rows].nan_to_num())
    print("off by", off, flush=True)
    assert off <= 1.0, off
    return got


RUNS = [(1, 0), (0, 5), (2, 0), (17, 0), (64, 0), (5, 59), (3, 61), (1, 300), (65, 64), (0, 0), (130, 7), (33, 511), (4, -2), (3, -3)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 32, 8, 24, 1, 7, 48])
def test_runs_sizes_pages(dtype, d, page):
    print("case", dtype, d, page, flush=True)
    check(make_runs(d + page, RUNS, 8, 2, d, page, dtype, lead=3, behind=5))


# A table that could hold far more tokens than the sequences have: their few rows go to the wavefronts of the whole device, 16 at
# a time, whatever the lengths are.
WIDE = 1 << 16
FEW = [(1, 0), (2, 0), (0, 7), (5, 59), (3, 61), (1, 300), (4, 28), (0, 0), (4, 640), (3, 509), (4, -2), (3, -3), (9, 33)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 32, 8, 24, 1, 7, 48])
def test_few_rows_sizes_pages(dtype, d, page):
    print("case", dtype, d, page, flush=True)
    check(fp4.widen(make_runs(d + page, FEW, 8, 2, d, page, dtype, lead=3, behind=5), WIDE))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (32, 8), (40, 8), (28, 4), (48, 8), (16, 1), (17, 1), (64, 2), (3, 3)])
def test_few_rows_head_layouts(dtype, heads, kv_heads):
    check(fp4.widen(make_runs(heads, [(3, 700), (1, 40), (4, 0), (2, 333)], heads, kv_heads, 128, 16, dtype), WIDE))


@pytest.mark.parametrize("sequences", [1, 3, 65, 200])
def test_few_rows_parts_of_a_row(sequences):
    """Joined by one wavefront, by four and by sixteen; more sequences than lanes."""
    runs = [(1 + i % 4, (137 * i) % 400 + (3000 if i == 0 else 0)) for i in range(sequences)]
    slopes = torch.tensor([2.0 ** -h for h in range(8)], device=DEV)
    for index in (torch.int64, torch.int32, torch.uint32):
        b = fp4.widen(make_runs(21, runs, 8, 2, 64, 16, torch.float16, index=index, layout="rows"), WIDE)
        check(b)
        check(b, slopes)
        check(dict(b, scale=-0.1))


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 8, 7])
def test_few_rows_and_values_that_are_not_finite(d, page):
    runs = [(4, 190), (5, 66), (7, 28), (1, 5)]
    b = fp4.widen(make_runs(11, runs, 8, 2, d, page, torch.bfloat16), WIDE)
    for i, (n, h) in enumerate(runs):
        for pool, back, group in ((2, 1, 0), (3, 2, 1), (3, n - 1, d // 32 - 1)):
            t = h + max(n - back, 0)
            if t < h + n:
                b["pool"][pool][int(b["table"][i, t // page]), 1, t % page, group] = fp4.NAN_BYTE
    got = check(b)
    assert got.isnan().any() and not got[:, :4].isnan().any()


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("slopes", [False, True])
def test_values_that_are_not_finite_in_the_history(d, slopes):
    """Keys and values in steps that every row of a block sees to the end: they reach all of them, in their columns."""
    runs = [(90, 300), (40, 129), (66, 64)]
    slopes = torch.tensor([2.0 ** -h for h in range(8)], device=DEV) if slopes else None
    b = make_runs(12, runs, 8, 2, d, 16, torch.bfloat16)
    for i, pool, t in ((0, 3, 0), (0, 3, 63), (0, 3, 200), (0, 3, 299), (1, 3, 127), (2, 2, 10)):
        b["pool"][pool][int(b["table"][i, t // 16]), 1, t % 16, t % (d // 32)] = fp4.NAN_BYTE
    got = check(b, slopes)
    assert not got[:, :4].isnan().any() and got[130:, 4:].isnan().all() and not got[:130, 4:].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_queries_of_every_size(dtype, d):
    """Elements of one group from the type's largest to its smallest, groups of zeros, and queries that are not finite."""
    runs = [(40, 30)]
    b = make_runs(13, runs, 8, 2, d, 16, dtype)
    gen = torch.Generator().manual_seed(5)
    q = torch.randn(b["q"].shape, generator=gen).double()
    q[:20] *= torch.exp2(torch.randint(-16, 3, q[:20].shape, generator=gen).double())
    q[3] = 0
    q[4, :, 32:] = 0
    q[5] *= 2.0 ** -20
    b["q"] = q.to(dtype).to(DEV)
    check(b)
    big = 300.0
    b["q"] = (q * big).to(dtype).to(DEV)
    check(b)
    clean = check(b)
    b["q"] = b["q"].clone()
    b["q"][7, 1, d - 1] = math.inf
    b["q"][8, 2, 0] = math.nan
    got = ops.paged_attention_prefill_fp4(b["q"], *b["pool"], b["table"], b["lens"], b["cum"], None, b["scale"])
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[7, 1] = nan[8, 2] = True
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean[~nan])


def test_blocks_in_both_orders():
    """More row blocks than compute units: by length up to 64 sequences, as the sequences come beyond."""
    runs = [((53 * i) % 90, (37 * i) % 130) for i in range(64)]
    check(make_runs(31, runs, 32, 8, 64, 16, torch.bfloat16))
    check(make_runs(32, runs + [(5, 0), (40, 3)], 32, 8, 64, 16, torch.bfloat16))
    check(make_runs(33, [(1, -5), (600, -590), (700, 0), (3, -1), (300, 40)], 16, 4, 64, 16, torch.float16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_blocks_of_128_rows(dtype, d):
    """Rows enough for the larger row blocks on every device; they are found by the number of rows alone."""
    runs = [(1100, 100), (700, 0), (900, 37), (1, 900)]
    check(make_runs(d, runs, 32, 4, d, 16, dtype))
    check(make_runs(d, [(1500, 3)], 48, 6, d, 7, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (32, 8), (40, 8), (28, 4), (48, 8), (16, 1), (17, 1), (64, 2), (40, 1), (3, 3)])
@pytest.mark.parametrize("runs", [[(70, 30), (3, 400), (1, 0)], [(3, 1500), (1, 40), (4, 0), (2, 777)]])
def test_head_layouts(dtype, heads, kv_heads, runs):
    print("case", dtype, heads, kv_heads, runs, flush=True)
    check(make_runs(heads, runs, heads, kv_heads, 128, 16, dtype))


@pytest.mark.parametrize("index", [torch.int64, torch.int32, torch.uint32])
@pytest.mark.parametrize("layout", ["packed", "rows", "padded"])
@pytest.mark.parametrize("runs", [[(5, 0), (40, 200), (1, 64)], [(2, 100), (1, 200)]])
def test_indices_and_layouts(index, layout, runs):
    check(make_runs(3, runs, 16, 4, 128, 16, torch.bfloat16, index=index, layout=layout))


@pytest.mark.parametrize("d,page", [(64, 16), (128, 8), (192, 16), (256, 5)])
@pytest.mark.parametrize("runs", [[(40, 0), (3, 90)], [(2, 90), (1, 130)]])
def test_query_and_output_strides(d, page, runs):
    b = make_runs(9, runs, 12, 4, d, page, torch.float16)
    n = b["q"].shape[0]
    fused = torch.zeros((n, 20, d), dtype=torch.float16, device=DEV)
    fused[:, 3:15] = b["q"]
    odd = torch.zeros((n, 12, d + 1), dtype=torch.float16, device=DEV)
    odd[..., 1:] = b["q"]
    for q in (fused[:, 3:15], odd[..., 1:], b["q"].transpose(0, 1).contiguous().transpose(0, 1)):
        b["q"] = q
        check(b)
        wide = torch.full((n, 13, d + 3), 7.0, dtype=torch.float16, device=DEV)
        check(b, out=wide[:, 1:, 1:d + 1])
        assert (wide[:, 0] == 7.0).all() and (wide[..., 0] == 7.0).all() and (wide[..., d + 1:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("runs", [[(100, 0), (33, 700)], [(3, 100), (2, 700), (1, 5)]])
def test_alibi_and_scales(dtype, runs):
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / 16) for h in range(16)], device=DEV)
    check(make_runs(4, runs, 16, 16, 64, 32, dtype, index=torch.int32), slopes)
    slopes = torch.cat((-slopes[:6], torch.zeros(6, device=DEV)))
    check(make_runs(5, runs, 10, 2, 128, 16, dtype), slopes)
    for scale in (0.0, -0.125, 1.0):
        b = make_runs(6, runs, 8, 2, 128, 16, dtype)
        b["scale"] = scale
        check(b)


def test_one_long_sequence_and_many_short():
    check(make_runs(7, [(5, 20001)], 16, 2, 128, 16, torch.bfloat16))
    check(make_runs(7, [(90, 9001)], 16, 2, 128, 16, torch.bfloat16))
    check(make_runs(8, [((7 * i) % 23, (37 * i) % 90) for i in range(333)], 8, 2, 64, 16, torch.float16))
    check(make_runs(8, [(1 + i % 3, (37 * i) % 190) for i in range(200)], 8, 2, 128, 16, torch.float16))


@pytest.mark.parametrize("runs", [[(300, 600)], [(3, 800), (2, 600)]])
def test_climbing_scores(runs):
    for hot in (1.0, 30.0, 300.0):
        b = make_runs(10, runs, 8, 2, 128, 16, torch.bfloat16, hot=hot)
        for i in range(len(runs)):
            pages = b["table"][i, :b["needed"][i]].long()
            order = torch.arange(len(pages) * 16, device=DEV).view(-1, 1, 16, 1)
            scales = b["pool"][2][pages]
            b["pool"][2][pages] = torch.where(scales == 255, 255, (110 + order * 14 // (len(pages) * 16)).to(torch.uint8))
        check(b)


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("runs", [[(150, 40), (1, 70)], [(4, 190), (5, 66), (7, 28)]])
def test_nothing_passes_from_tokens_that_a_row_does_not_see(runs, d, page):
    """Keys and values of new tokens that are not finite: they reach the rows from their own on, in their columns, and no other."""
    b = make_runs(11, runs, 8, 2, d, page, torch.bfloat16)
    for i, (n, h) in enumerate(runs):
        for pool, back, group in ((2, 1, 0), (3, 2, 1), (3, n - 1, d // 32 - 1)):
            t = h + max(n - back, 0)
            if t < h + n:
                b["pool"][pool][int(b["table"][i, t // page]), 1, t % page, group] = fp4.NAN_BYTE
    got = check(b)
    assert got.isnan().any() and not got[:, :4].isnan().any()


def test_page_order_repeats_and_lengths_beyond_the_table():
    for runs in ([(100, 200), (64, 0), (5, 900)], [(3, 300), (2, 1000)]):
        b = make_runs(13, runs, 8, 2, 128, 16, torch.float16)
        first = check(b)
        assert torch.equal(check(b), first)
        perm = torch.randperm(b["pool"][0].shape[0], device=DEV)
        back = torch.argsort(perm)
        table = b["table"].clone()
        for i, n in enumerate(b["needed"]):
            table[i, :n] = back[table[i, :n]]
        assert torch.equal(check(dict(b, pool=[t[perm] for t in b["pool"]], table=table)), first)
    # positions behind the table: what it holds is seen by all of them
    b = make_runs(14, [(100, 200)], 8, 2, 128, 16, torch.float16, poison=False)
    b["table"], b["needed"] = b["table"][:, :10], [10]
    want = torch.full_like(b["q"], 7.0, dtype=torch.float64)
    pages = b["table"][0].long()
    k, v = (fp4.sequence(b["pool"][x], b["pool"][x + 2], pages, 160) for x in (0, 1))
    want, allowed = fp4.attention(b["q"], k, v, b["scale"], [159] * 100, terms=True)
    got = ops.paged_attention_prefill_fp4(b["q"], *b["pool"], b["table"], b["lens"], b["cum"], None, b["scale"])
    assert fp4.off_by(got, want, allowed) <= 1.0
    # prefix sums beyond the query: clipped
    got2 = ops.paged_attention_prefill_fp4(b["q"][:50].contiguous(), *b["pool"], b["table"], b["lens"], b["cum"], None, b["scale"])
    assert torch.equal(got2, got[:50])


def test_offsets_past_32_bits():
    d, page, kv = 128, 16, 8
    blocks = (9 << 29) // (kv * page * d // 2)  # 4.8e9 bytes of codes
    pool = [torch.zeros((blocks, kv, page, w), dtype=torch.uint8, device=DEV) for w in (64, 64, 4, 4)]
    table = torch.stack((torch.arange(5), blocks - 1 - torch.arange(5))).to(DEV)
    small = fp4.make_pool(1, 10, kv, page, d)
    for big, t in zip(pool, small):
        big[table.flatten()] = t.to(DEV)
    for runs in ([(60, 17), (70, 10)], [(2, 70), (3, 77)]):
        n = sum(x for x, _ in runs)
        b = dict(q=torch.randn((n, 32, d), generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV), pool=pool, table=table,
                 lens=torch.tensor([x + h for x, h in runs], device=DEV), needed=[5, 5], scale=0.1, runs=runs,
                 cum=torch.tensor([0, runs[0][0], n], device=DEV), starts=[0, runs[0][0], n])
        check(b)


@pytest.mark.parametrize("runs", [[(100, 200), (33, 0), (1, 700)], [(2, 200), (3, 900)]])
def test_streams_and_graphs(runs):
    b = make_runs(14, runs, 32, 8, 128, 16, torch.bfloat16, poison=False)
    args = (b["q"], *b["pool"], b["table"], b["lens"], b["cum"], None, b["scale"])
    eager = ops.paged_attention_prefill_fp4(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.paged_attention_prefill_fp4(*args)
    side.synchronize()
    assert torch.equal(eager, other)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_attention_prefill_fp4(*args)
        graphs.append((graph, out))
    ops.clear_plan_cache()
    lens = b["lens"].clone()
    for turn, less in enumerate((0, 1, 17)):
        b["lens"].copy_(lens - less)
        want = ops.paged_attention_prefill_fp4(*args, out=torch.zeros_like(eager))
        for graph, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want), turn


def test_one_new_token_is_decode():
    lens = [1, 30, 500, 64]
    b = make_runs(15, [(1, n - 1) for n in lens], 8, 2, 128, 16, torch.bfloat16)
    got = check(b)
    decode = ops.paged_attention_fp4(b["q"], *b["pool"], b["table"], b["lens"], None, b["scale"])
    want, allowed, _ = reference(b)
    assert fp4.off_by(decode, want, allowed) <= 1.0 and fp4.off_by(got, want, allowed) <= 1.0


def test_chunks_through_the_whole_family():
    """A prompt in chunks, then single tokens, as a server runs them: written, attended over, read back; against the 16-bit
    operators on the values that were read back."""
    kv, heads, d, page, dtype = 4, 16, 128, 16, torch.bfloat16
    gen = torch.Generator().manual_seed(3)
    pool = [torch.zeros((40, kv, page, w), dtype=torch.uint8, device=DEV) for w in (d // 2, d // 2, d // 32, d // 32)]
    table = torch.randperm(40, generator=gen)[:20].view(1, 20).to(DEV)
    total = 0
    for n in (100, 57, 1, 3, 1):
        k, v = (torch.randn((n, kv, d), generator=gen).to(dtype).to(DEV) for _ in range(2))
        q = torch.randn((n, heads, d), generator=gen).to(dtype).to(DEV)
        at = torch.arange(total, total + n, device=DEV)
        ops.paged_caching_fp4(*pool, k, v, table[0, at // page] * page + at % page)
        total += n
        lens, cum = torch.tensor([total], device=DEV), torch.tensor([0, n], device=DEV)
        if n == 1:
            got = ops.paged_attention_fp4(q, *pool, table, lens, None, d ** -0.5)
        else:
            got = ops.paged_attention_prefill_fp4(q, *pool, table, lens, cum, None, d ** -0.5)
        every = torch.arange(20 * page, device=DEV)
        ko, vo = ops.paged_reading_fp4(*pool, table[0, every // page] * page + every % page)
        as_pool = [x.view(20, page, kv, d).transpose(1, 2) for x in (ko, vo)]
        rows = torch.arange(20, device=DEV).view(1, 20)
        wide = ops.paged_attention_prefill(q, *as_pool, rows, lens, cum, None, d ** -0.5)
        exact, allowed = fp4.attention(q, ko[:total].transpose(0, 1).double(), vo[:total].transpose(0, 1).double(), d ** -0.5,
                                       list(range(total - n, total)), terms=n > 1)
        assert fp4.off_by(got, exact, allowed) <= 1.0
        # the 16-bit operator rounds its probabilities to bf16: 2^-8 of every weight, twice (numerator and denominator)
        assert fp4.off_by(wide, exact, allowed + 2 ** -7 * vo[:total].abs().amax().double()) <= 1.0
        assert torch.equal(ko[:total].cpu().double()[-n:], fp4.values(*fp4.quantise(k.cpu())))


@pytest.mark.parametrize("wide", [0, WIDE])
def test_prefix_sums_that_fall(wide):
    """Rows claimed by several sequences, all of them alike: written once or more, with what one of them gives them; nothing
    outside q, the output and the workspace is reached (the workspace has a border that has to stay)."""
    b = make_runs(41, [(4, 60)] * 70, 8, 2, 128, 16, torch.bfloat16, poison=False)
    b["table"][:] = b["table"][:1].clone()
    b = fp4.widen(b, wide)
    b["q"] = b["q"][:8].contiguous()
    b["q"][4:] = b["q"][:4].clone()
    cum = torch.tensor([(0, 4, 8)[i % 3] for i in range(71)], device=DEV)
    want, allowed, _ = reference(dict(b, runs=b["runs"][:2], starts=[0, 4, 8]))
    L.set_device(L.InfiniDevice.AMD, 0)
    handle = L.create_handle()
    out = torch.zeros_like(b["q"])
    tensors = [out, b["q"], *b["pool"], b["table"], b["lens"], cum]
    descs = [describe(t) for t in tensors]
    op, size = L.infiniopOperatorDescriptor_t(), ctypes.c_size_t(0)
    L.check_error(L.LIBINFINIOP.infiniopCreatePagedAttentionPrefillFp4Descriptor(handle, ctypes.byref(op), *descs,
                                                                                 L.infiniopTensorDescriptor_t(), b["scale"]))
    L.check_error(L.LIBINFINIOP.infiniopGetPagedAttentionPrefillFp4WorkspaceSize(op, ctypes.byref(size)))
    assert (size.value > 0) == (wide > 0)
    workspace = torch.full((size.value + 4096,), 77, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    L.check_error(L.LIBINFINIOP.infiniopPagedAttentionPrefillFp4(op, ptr(workspace), size.value, *(ptr(t) for t in tensors), None, None))
    torch.cuda.synchronize()
    assert (workspace[size.value:] == 77).all()
    assert fp4.off_by(out, want, allowed) <= 1.0
    for d in descs:
        L.destroy_tensor_descriptor(d)
    L.check_error(L.LIBINFINIOP.infiniopDestroyPagedAttentionPrefillFp4Descriptor(op))
    L.destroy_handle(handle)


@pytest.mark.parametrize("wide", [0, WIDE])
def test_c_entry_points(wide):
    runs = [(7, 30), (2, 500)] if wide else [(70, 30), (2, 500)]
    b = fp4.widen(make_runs(15, runs, 16, 4, 128, 16, torch.bfloat16), wide)
    out = torch.full_like(b["q"], 7.0)
    tensors = [out, b["q"], *b["pool"], b["table"], b["lens"], b["cum"]]
    L.set_device(L.InfiniDevice.AMD, 0)
    handle = L.create_handle()
    descs = [describe(t) for t in tensors]
    op = L.infiniopOperatorDescriptor_t()
    L.check_error(L.LIBINFINIOP.infiniopCreatePagedAttentionPrefillFp4Descriptor(handle, ctypes.byref(op), *descs,
                                                                                 L.infiniopTensorDescriptor_t(), b["scale"]))
    for d in descs:
        L.destroy_tensor_descriptor(d)
    size = ctypes.c_size_t(0)
    L.check_error(L.LIBINFINIOP.infiniopGetPagedAttentionPrefillFp4WorkspaceSize(op, ctypes.byref(size)))
    want, allowed, _ = reference(b)
    run = lambda ws, n, *p: L.LIBINFINIOP.infiniopPagedAttentionPrefillFp4(op, ws, n, *p, None, None)  # noqa: E731
    pointers = [ptr(t) for t in tensors]
    for fill in (0, 255, 77):
        workspace = torch.full((size.value + 1,), fill, dtype=torch.uint8, device=DEV)
        torch.cuda.synchronize()
        for offset in (0, 1):
            out.fill_(7.0)
            torch.cuda.synchronize()
            L.check_error(run(ctypes.c_void_p(workspace.data_ptr() + offset), size.value, *pointers))
            torch.cuda.synchronize()
            assert fp4.off_by(out, want, allowed) <= 1.0
    S = L.InfiniStatus
    assert (size.value > 0) == (wide > 0)
    if size.value:
        assert run(ptr(workspace), size.value - 1, *pointers) == S.INSUFFICIENT_WORKSPACE
        assert run(None, size.value, *pointers) == S.INSUFFICIENT_WORKSPACE
    for i in range(len(pointers)):
        assert run(ptr(workspace), size.value, *pointers[:i], None, *pointers[i + 1:]) == S.NULL_POINTER
    for i in (2, 3):
        assert run(ptr(workspace), size.value, *pointers[:i], ctypes.c_void_p(pointers[i].value + 8), *pointers[i + 1:]) == S.BAD_PARAM
    L.check_error(L.LIBINFINIOP.infiniopDestroyPagedAttentionPrefillFp4Descriptor(op))
    L.destroy_handle(handle)
