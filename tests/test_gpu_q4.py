"""Products with weights stored in 4 bits against the matrix their blocks stand for, in 64 bits."""
import numpy as np
import pytest
import torch

import cortexsdr_b200 as cs
from cortexsdr_b200 import _lib
from tests import operator_refs as ref
from tests import synth

pytestmark = pytest.mark.gpu
DTYPES = {"f32": (torch.float32, 0), "bf16": (torch.bfloat16, 1), "f16": (torch.float16, 2)}


def run(w, x, layout, rows, ctx, bias=None, y_layout=None):
    tdtype = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[x.dtype]
    batch = x.shape[0]
    y_layout = layout if y_layout is None else y_layout
    xd = (x if layout else x.t()).contiguous().cuda()
    y = torch.full((batch, rows) if y_layout else (rows, batch), 7.0, device="cuda")
    torch.cuda.synchronize()
    w.matmul_device(xd.data_ptr(), tdtype, layout, batch, y.data_ptr(), y_layout, bias.data_ptr() if bias is not None else 0)
    ctx.synchronize()
    return (y if y_layout else y.t()).to(torch.float64).cpu().numpy()


def check(y, x, dense):
    """Each product of fp32 values carries at most 2^-22 (two 11-bit halves of x) + 2^-23 (the step), sums fp32: 2^-19
    of sum |x w| covers widths to 2^14 summed in any order with room; on the whole fp32's own error."""
    x = x.to(torch.float64).numpy()
    want, room = x @ dense.T, np.abs(x) @ np.abs(dense).T
    assert (np.abs(y - want) <= 2.0 ** -19 * room + 1e-30).all()
    assert np.linalg.norm(y - want) <= 2e-6 * np.linalg.norm(want) + 1e-30


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,batch", [(1, 32, 1), (16, 128, 1), (17, 160, 2), (100, 896, 1), (333, 1056, 3), (64, 4096, 4),
                                             (130, 2080, 5), (48, 96, 8), (1000, 512, 16), (33, 1280, 17), (50, 352, 40), (20, 64, 130)])
def test_q4_0(ctx, rows, cols, batch, dtype):
    rng = np.random.default_rng(rows)
    payload, dense = ref.q4_weight(rng, rows, cols, "q4_0")
    w = cs.Q4Weight.from_payload(payload, "q4_0", rows, cols, ctx)
    x = torch.tensor(rng.normal(0, 1, (batch, cols)), dtype=torch.float32).to(DTYPES[dtype][0])
    for layout in (0, 1):
        check(run(w, x, layout, rows, ctx), x, dense)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,batch", [(1, 256, 1), (40, 256, 2), (129, 1024, 1), (31, 2304, 7), (512, 768, 16), (70, 512, 33),
                                             (24, 4096, 3), (3, 11008, 9)])
def test_q4_k(ctx, rows, cols, batch, dtype):
    rng = np.random.default_rng(rows + 1)
    payload, dense = ref.q4_weight(rng, rows, cols, "q4_k")
    w = cs.Q4Weight.from_payload(payload, "q4_k", rows, cols, ctx)
    x = torch.tensor(rng.normal(0, 1, (batch, cols)), dtype=torch.float32).to(DTYPES[dtype][0])
    for layout in (0, 1):
        check(run(w, x, layout, rows, ctx), x, dense)


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
def test_the_matrix_is_what_dequantisation_gives(ctx, fmt):
    # one column at a time: the product is the stored weight itself, to fp32
    rng = np.random.default_rng(5)
    payload, dense = ref.q4_weight(rng, 37, 512, fmt)
    w = cs.Q4Weight.from_payload(payload, fmt, 37, 512, ctx)
    wide = cs.dequantize_inference(payload, fmt, ctx=ctx).astype(np.float64).reshape(37, 512)
    for c0 in range(0, 512, 64):
        eye = torch.zeros(64, 512)
        eye[torch.arange(64), c0 + torch.arange(64)] = 1.0
        y = run(w, eye, 1, 37, ctx)
        # q4_k: minimum and step times code are one rounding each, as large as the larger of them
        bound = 2.0 ** -22 * (np.abs(dense[:, c0:c0 + 64]).T + (0.2 if fmt == "q4_k" else 0.0))
        assert (np.abs(y - wide[:, c0:c0 + 64].T) <= bound).all()


def test_bias_layouts_and_untouched_rows(ctx):
    rng = np.random.default_rng(6)
    rows, cols, batch = 45, 224, 5
    payload, dense = ref.q4_weight(rng, rows, cols, "q4_0")
    w = cs.Q4Weight.from_payload(payload, "q4_0", rows, cols, ctx)
    x = torch.tensor(rng.normal(0, 1, (batch, cols)), dtype=torch.float32)
    bias = torch.tensor(rng.normal(0, 1, rows), dtype=torch.float32).cuda()
    want = x.to(torch.float64).numpy() @ dense.T + bias.cpu().numpy()
    for lx in (0, 1):
        for ly in (0, 1):
            np.testing.assert_allclose(run(w, x, lx, rows, ctx, bias, ly), want, rtol=0, atol=1e-5)
    # the buffer around the result stays as it was, and operands need not start on 16 bytes
    room = torch.full((rows * batch + 2,), 7.0, device="cuda")
    xr = torch.zeros(batch * cols + 1, device="cuda")
    xr[1:] = x.reshape(-1).cuda()
    torch.cuda.synchronize()
    w.matmul_device(xr.data_ptr() + 4, 0, 1, batch, room.data_ptr() + 4, 1)
    ctx.synchronize()
    assert room[0] == 7 and room[-1] == 7
    np.testing.assert_allclose(room[1:-1].view(batch, rows).cpu().numpy(), want - bias.cpu().numpy(), rtol=0, atol=1e-5)


@pytest.mark.parametrize("scale", [1e-20, 1e-6, 1e5, 1e20])
def test_activations_of_any_magnitude(ctx, scale):
    rng = np.random.default_rng(7)
    payload, dense = ref.q4_weight(rng, 64, 768, "q4_k")
    w = cs.Q4Weight.from_payload(payload, "q4_k", 64, 768, ctx)
    for dtype in (torch.float32, torch.bfloat16):
        x = (torch.tensor(rng.normal(0, 1, (3, 768))) * scale).to(dtype)
        x[1] = x[1] * 1e-3                   # rows of one call differ in magnitude
        check(run(w, x, 1, 64, ctx), x, dense)
    x = torch.zeros(2, 768)
    assert (run(w, x, 1, 64, ctx) == 0).all()


def test_what_is_not_finite_stays_with_its_token(ctx):
    rng = np.random.default_rng(8)
    payload, dense = ref.q4_weight(rng, 40, 512, "q4_0")
    w = cs.Q4Weight.from_payload(payload, "q4_0", 40, 512, ctx)
    x = torch.tensor(rng.normal(0, 1, (6, 512)), dtype=torch.float32)
    clean = run(w, x, 1, 40, ctx)
    x[2, 7], x[4, 300] = float("nan"), float("inf")
    y = run(w, x, 1, 40, ctx)
    keep = [0, 1, 3, 5]
    np.testing.assert_array_equal(y[keep], clean[keep])
    assert not np.isfinite(y[2]).any() and not np.isfinite(y[4][dense[:, 300] != 0]).any()


def test_repeats_itself_and_captures(ctx):
    rng = np.random.default_rng(9)
    payload, dense = ref.q4_weight(rng, 4096, 4096, "q4_k")
    side = torch.cuda.Stream()
    own = cs.Context(0, side.cuda_stream)
    w = cs.Q4Weight.from_payload(payload, "q4_k", 4096, 4096, own)
    x = torch.tensor(rng.normal(0, 1, (2, 4096)), dtype=torch.float32).cuda()
    y = torch.zeros(2, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        w.matmul_device(x.data_ptr(), 0, 1, 2, y.data_ptr(), 1)
        side.synchronize()
        first = y.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            w.matmul_device(x.data_ptr(), 0, 1, 2, y.data_ptr(), 1)
        y.zero_()
        g.replay()
    side.synchronize()
    assert torch.equal(y, first)
    check(y.to(torch.float64).cpu().numpy(), x.cpu(), dense)
    del g
    w.close()
    own.close()


def test_refusals(ctx):
    payload, _ = ref.q4_weight(np.random.default_rng(0), 4, 256, "q4_0")
    make = lambda *a: cs.Q4Weight.from_payload(*a, ctx)
    with pytest.raises(cs.CompressionError, match="format"):
        make(payload, "q8_0", 4, 256)
    with pytest.raises(cs.CompressionError, match="whole blocks"):
        make(payload, "q4_0", 4, 250)
    with pytest.raises(cs.CompressionError, match="size"):
        make(payload, "q4_0", 5, 256)
    with pytest.raises(cs.CompressionError, match="size"):
        make(payload.reshape(-1)[:-1], "q4_0", 4, 256)
    with pytest.raises(ValueError, match="range"):
        make(payload, "q4_0", 0, 256)
    w = make(payload, "q4_0", 4, 256)
    x, y = torch.zeros(256, device="cuda"), torch.zeros(4, device="cuda")
    for args, what in [((0, 0, 1, 1, y.data_ptr(), 1), "null"), ((x.data_ptr(), 5, 1, 1, y.data_ptr(), 1), "dtype"),
                       ((x.data_ptr(), 0, 2, 1, y.data_ptr(), 1), "layout"), ((x.data_ptr(), 0, 1, 1, 0, 1), "null")]:
        with pytest.raises(ValueError, match=what):
            w.matmul_device(*args)
    before = ctx.launch_count
    w.matmul_device(x.data_ptr(), 0, 1, 0, y.data_ptr(), 1)
    assert ctx.launch_count == before


def test_refuses_pointers_inside_an_element(ctx):
    payload, _ = ref.q4_weight(np.random.default_rng(0), 4, 256, "q4_0")
    w = cs.Q4Weight.from_payload(payload, "q4_0", 4, 256, ctx)
    x, y = torch.zeros(300, device="cuda").data_ptr(), torch.zeros(8, device="cuda").data_ptr()
    for args in [(x + 2, 0, 1, 1, y, 1), (x + 1, 1, 1, 1, y, 1), (x + 1, 2, 1, 1, y, 1), (x, 0, 1, 1, y + 2, 1), (x, 0, 1, 1, y, 1, y + 1)]:
        with pytest.raises(ValueError, match="whole element"):
            w.matmul_device(*args)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("warm", [False, True])
def test_a_captured_wide_product(layout, warm):
    """Captured first of all in its context, and behind one that sized the scratch; then replayed after a larger product
    has moved that scratch."""
    rng = np.random.default_rng(11)
    side = torch.cuda.Stream()
    own = cs.Context(0, side.cuda_stream)
    payload, dense = ref.q4_weight(rng, 300, 4096, "q4_k")
    w = cs.Q4Weight.from_payload(payload, "q4_k", 300, 4096, own)
    big, _ = ref.q4_weight(rng, 64, 16384, "q4_0")
    larger = cs.Q4Weight.from_payload(big, "q4_0", 64, 16384, own)
    x = torch.tensor(rng.normal(0, 1, (40, 4096)), dtype=torch.float32).cuda()
    given = x.t().contiguous() if layout == 0 else x
    y = torch.zeros(40, 300, device="cuda")
    x2, y2 = torch.zeros(128, 16384, device="cuda"), torch.empty(128, 64, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        if warm:
            w.matmul_device(given.data_ptr(), 0, layout, 40, y.data_ptr(), 1)
            side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            w.matmul_device(given.data_ptr(), 0, layout, 40, y.data_ptr(), 1)
        for _ in range(2):
            y.zero_()
            g.replay()
            side.synchronize()
            check(y.to(torch.float64).cpu().numpy(), x.cpu(), dense)
            larger.matmul_device(x2.data_ptr(), 0, 1, 128, y2.data_ptr(), 1)
    side.synchronize()
    assert (y2 == 0).all()
    del g
    w.close()
    larger.close()
    own.close()


def test_a_wait_that_runs_out_is_reported():
    own = cs.Context(0)
    rng = np.random.default_rng(12)
    payload, dense = ref.q4_weight(rng, 512, 8192, "q4_0")
    w = cs.Q4Weight.from_payload(payload, "q4_0", 512, 8192, own)
    x = torch.tensor(rng.normal(0, 1, (48, 8192)), dtype=torch.float32)
    want = run(w, x, 1, 512, own)
    own.set_wait_limits(barrier_rounds=1)
    for _ in range(3):
        try:
            got = run(w, x, 1, 512, own)
        except cs.CudaError:
            continue
        np.testing.assert_array_equal(got, want)
    own.set_wait_limits()
    np.testing.assert_array_equal(run(w, x, 1, 512, own), want)
    w.close()
    own.close()


def test_a_captured_product_of_another_kind_keeps_its_scratch():
    """A graph of a product with a compressed weight, whose activations go through scratch of the context; then the largest 4-bit
    product so far, whose fragments take up to 16 MB; then the graph again."""
    rng = np.random.default_rng(13)
    side = torch.cuda.Stream()
    own = cs.Context(0, side.cuda_stream)
    seg = cs.Segment.from_payload(synth.hsdr_payload(384, 1024, n_atoms=128, k=6, seed=4), own)
    big, dense = ref.q4_weight(rng, 64, 16384, "q4_0")
    larger = cs.Q4Weight.from_payload(big, "q4_0", 64, 16384, own)
    x, y = torch.tensor(rng.normal(0, 1, (16, 1024)), dtype=torch.float32).cuda(), torch.zeros(16, 384, device="cuda")
    x2, y2 = torch.tensor(rng.normal(0, 1, (128, 16384)), dtype=torch.float32).cuda(), torch.empty(128, 64, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        seg.matmul_device(x.data_ptr(), 0, 1, 16, y.data_ptr(), 1)
        side.synchronize()
        first = y.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            seg.matmul_device(x.data_ptr(), 0, 1, 16, y.data_ptr(), 1)
        larger.matmul_device(x2.data_ptr(), 0, 1, 128, y2.data_ptr(), 1)
        y.zero_()
        g.replay()
    side.synchronize()
    assert torch.equal(y, first)
    check(y2.to(torch.float64).cpu().numpy(), x2.cpu(), dense)
    del g
    larger.close()
    seg.close()
    own.close()


def check_wide(y, x, dense, units):
    """check() for any width: a product carries 2^-22 + 2^-23, and of q4_0 the 8 of every code as much again; a rank adds up at most
    `units` partial sums, eight ranks and a bias their sums, each rounded to 2^-24, and matrix units cut off 2^-23 in each of
    sixteen steps of a unit."""
    x = x.to(torch.float64).numpy()
    want, room = x @ dense.T, np.abs(x) @ np.abs(dense).T
    assert (np.abs(y - want) <= (2.0 ** -20 + (units + 8 + 32) * 2.0 ** -24) * room + 1e-30).all()
    assert np.linalg.norm(y - want) <= 2e-6 * np.linalg.norm(want) + 1e-30


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt,cols", [("q4_0", 96), ("q4_0", 1152), ("q4_k", 512)])
@pytest.mark.parametrize("batch", [1, 3, 40])
def test_more_row_blocks_than_the_gpu_holds(ctx, fmt, cols, batch, dtype):
    """CTAs take blocks of rows in turn."""
    rows = 128 * 2 * torch.cuda.get_device_properties(0).multi_processor_count + 128 * 17 + 5      # two CTAs an SM, and some more
    rng = np.random.default_rng(cols + batch)
    payload, dense = ref.q4_weight(rng, rows, cols, fmt)
    w = cs.Q4Weight.from_payload(payload, fmt, rows, cols, ctx)
    x = torch.tensor(rng.normal(0, 1, (batch, cols)), dtype=torch.float32).to(DTYPES[dtype][0])
    bias = torch.tensor(rng.normal(0, 1, rows), dtype=torch.float32).cuda()
    for layout in (0, 1):
        got = run(w, x, layout, rows, ctx)
        check(got, x, dense)
        np.testing.assert_allclose(run(w, x, layout, rows, ctx, bias), got + bias.cpu().numpy(), rtol=1e-6, atol=1e-5)
    w.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fmt,cols", [("q4_0", 102432), ("q4_k", 97280)])
@pytest.mark.parametrize("batch", [1, 5, 33])
def test_activations_that_do_not_fit_at_a_time(ctx, fmt, cols, batch, dtype):
    """An eighth of the columns is more than shared memory holds as fragments: they are brought in parts, by the CTAs themselves
    and by copies of what a launch has made."""
    units = -(-cols // (256 if fmt == "q4_k" else 128))
    assert -(-units // 8) * (4384 if fmt == "q4_k" else 2080) > 208 * 1024 - 6144      # the least that fragments and results are
    rows, rng = 300, np.random.default_rng(cols + batch)
    payload, dense = ref.q4_weight(rng, rows, cols, fmt)
    side = torch.cuda.Stream()
    own = cs.Context(0, side.cuda_stream)
    w = cs.Q4Weight.from_payload(payload, fmt, rows, cols, own)
    x = torch.tensor(rng.normal(0, 1, (batch, cols)), dtype=torch.float32).to(DTYPES[dtype][0])
    # captured first of all: without scratch, so by the CTAs themselves
    xd, y = x.cuda(), torch.zeros(batch, rows, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            w.matmul_device(xd.data_ptr(), DTYPES[dtype][1], 1, batch, y.data_ptr(), 1)
        g.replay()
    side.synchronize()
    check_wide(y.to(torch.float64).cpu().numpy(), x, dense, units)
    for layout in (0, 1):
        check_wide(run(w, x, layout, rows, own), x, dense, units)
    del g
    w.close()
    own.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_fragments_than_a_launch_takes(ctx, dtype):
    """Token tiles go over several pairs of launches, the last one ragged, all through the same scratch."""
    rows, cols, batch = 130, 4096, 4099
    rng = np.random.default_rng(17)
    payload, dense = ref.q4_weight(rng, rows, cols, "q4_k")
    w = cs.Q4Weight.from_payload(payload, "q4_k", rows, cols, ctx)
    x = torch.tensor(rng.normal(0, 1, (batch, cols)), dtype=torch.float32).to(DTYPES[dtype][0])
    for x_layout, y_layout in ((0, 0), (1, 1), (1, 0)):
        before = ctx.launch_count
        got = run(w, x, x_layout, rows, ctx, y_layout=y_layout)
        assert ctx.launch_count - before >= 4
        check(got, x, dense)
    w.close()


def test_packed_products_of_prompts_are_not_slower_than_widened_ones(ctx, tmp_path):
    """A decoder's stored-raw linears stay packed at any number of tokens: the dense fp32 product of the widened weight, which they
    were before, must not be the faster one. Device time between events, medians, a fifth to spare."""
    rows, cols, batch = 4864, 896, 1024
    rng = np.random.default_rng(18)
    payload, dense = ref.q4_weight(rng, rows, cols, "q4_0")
    synth.write_sdr(str(tmp_path / "w.sdr"), [synth.raw_segment("w", dense.astype(np.float32), synth.SEG_ATTENTION, 0)])
    loader = cs.SDRModelLoader(str(tmp_path / "w.sdr"), ctx)
    engine = cs.SDRInferenceEngine(loader)
    w = cs.Q4Weight.from_payload(payload, "q4_0", rows, cols, ctx)
    x = rng.normal(0, 1, (cols, batch)).astype(np.float32)
    xd = torch.tensor(x).t().contiguous()

    def median(call):
        call()
        took = []
        for _ in range(7):
            ctx.profile(True)
            call()
            took.append(sum(ms for _, ms in ctx.profile_read().values()))
            ctx.profile(False)
        return sorted(took)[3]

    assert median(lambda: run(w, xd, 1, rows, ctx)) <= 1.2 * median(lambda: engine.matmulForLayer("w", x, batch))
    w.close()
    loader.close()


@pytest.mark.parametrize("fmt,rows,cols,batch,copies", [("q4_0", 512, 8192, 48, True), ("q4_k", 300, 8192, 48, False), ("q4_0", 300, 99200, 33, True),
                                                        ("q4_k", 4096, 4096, 48, True)])
def test_waits_that_are_given_up(fmt, rows, cols, batch, copies):
    """Copies of the activations' fragments are given up on their way, in one part and in several. Where CTAs make the fragments
    themselves nothing waits."""
    own = cs.Context(0)
    rng = np.random.default_rng(19)
    payload, dense = ref.q4_weight(rng, rows, cols, fmt)
    w = cs.Q4Weight.from_payload(payload, fmt, rows, cols, own)
    x = torch.tensor(rng.normal(0, 1, (batch, cols)), dtype=torch.float32)
    before = own.launch_count
    want = run(w, x, 1, rows, own)
    assert own.launch_count - before == (2 if copies else 1)      # the first makes the fragments
    for _ in range(2):
        own.set_wait_limits(barrier_rounds=_lib.WAIT_GIVE_UP)
        if copies:
            with pytest.raises(cs.CudaError, match="wait ran out"):
                run(w, x, 1, rows, own)
        else:
            np.testing.assert_array_equal(run(w, x, 1, rows, own), want)
        own.set_wait_limits()
        np.testing.assert_array_equal(run(w, x, 1, rows, own), want)
    w.close()
    own.close()


def test_results_past_32_bits(ctx):
    """More than 2^32 results, either way round."""
    rows, cols, batch = 40001, 64, 110_003
    rng = np.random.default_rng(20)
    payload, dense = ref.q4_weight(rng, rows, cols, "q4_0")
    w = cs.Q4Weight.from_payload(payload, "q4_0", rows, cols, ctx)
    x = torch.tensor(rng.normal(0, 1, (batch, cols)), dtype=torch.float32)
    toks = np.unique(np.concatenate([rng.integers(0, batch, 200), [0, 1, batch - 2, batch - 1, (1 << 32) // rows, (1 << 32) // rows + 1]]))
    picked = np.unique(np.concatenate([rng.integers(0, rows, 200), [0, rows - 1, (1 << 32) // batch, (1 << 32) // batch + 1]]))
    y = torch.empty(batch * rows, device="cuda")
    for layout in (0, 1):
        xd = (x if layout else x.t()).contiguous().cuda()
        y.fill_(7.0)
        torch.cuda.synchronize()
        w.matmul_device(xd.data_ptr(), 0, layout, batch, y.data_ptr(), layout)
        ctx.synchronize()
        got = y.view(batch, rows) if layout else y.view(rows, batch).t()
        check(got[torch.tensor(toks, device="cuda")].to(torch.float64).cpu().numpy(), x[toks], dense)
        check(got[:, torch.tensor(picked, device="cuda")].to(torch.float64).cpu().numpy(), x, dense[picked])
    w.close()


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("largest", [2.0 ** -123, 2.0 ** -113, 2.0 ** -105, 2.0 ** 126])
def test_activations_at_the_ends_of_their_range(ctx, fmt, dtype, largest):
    """check()'s bound, and for results that are not normal fp32 numbers their last bit, 2^-149, for every partial sum (16 of
    units and ranks) and for every sixteenth of it where a partial sum is kept 2^4 smaller."""
    rng = np.random.default_rng(21)
    payload, dense = ref.q4_weight(rng, 48, 768, fmt)
    w = cs.Q4Weight.from_payload(payload, fmt, 48, 768, ctx)
    x = torch.tensor(rng.normal(0, 1, (3, 768)))
    x = (x / x.abs().max() * largest / (64 if largest > 1 else 1)).to(DTYPES[dtype][0])      # (sums of the largest stay finite)
    y = run(w, x, 1, 48, ctx)
    xx = x.to(torch.float64).numpy()
    want, room = xx @ dense.T, np.abs(xx) @ np.abs(dense).T
    assert np.isfinite(want.astype(np.float32)).all() and (want != 0).all()
    assert (np.abs(y - want) <= 2.0 ** -19 * room + 16 * 16 * 2.0 ** -149).all()
    w.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch", [1, 4, 24])
def test_loud_columns(ctx, dtype, batch):
    """A few activations are far greater than the rest, in columns that half of the rows give no weight: they add nothing there,
    and the others keep their bits. check()'s 2^-19 of sum |x w|, and 2^-25 of what a unit's largest is scaled to, 2^14."""
    rng = np.random.default_rng(22)
    rows, cols = 200, 2048
    payload, dense = ref.q4_weight(rng, rows, cols, "q4_0")
    blocks = payload.reshape(rows, cols // 32, 18)
    x = rng.normal(0, 1, (batch, cols))
    loud = rng.choice(cols // 2, 6, replace=False) * 2      # low halves of their bytes
    for c in loud:
        blocks[::2, c // 32, 2 + c % 32 // 2] = blocks[::2, c // 32, 2 + c % 32 // 2] & 0xF0 | 8
        dense[::2, c] = 0
    x[:, loud] *= 3e4 if dtype != "f16" else 3e3
    x = torch.tensor(x, dtype=torch.float32).to(DTYPES[dtype][0])
    w = cs.Q4Weight.from_payload(blocks.reshape(-1), "q4_0", rows, cols, ctx)
    for layout in (0, 1):
        y = run(w, x, layout, rows, ctx)
        xx = np.abs(x.to(torch.float64).numpy())
        largest = np.repeat(xx.reshape(batch, cols // 128, 128).max(-1), 128, axis=1)
        room = 2.0 ** -19 * xx @ np.abs(dense).T + 2.0 ** -39 * largest @ np.abs(dense).T
        assert (np.abs(y - x.to(torch.float64).numpy() @ dense.T) <= room).all()
    w.close()
