"""What the projection of many requests promises beyond single calls of ordinary numbers: calls from
several host threads, long sums, small numbers, numbers that are not finite, memory."""

import threading

import pytest
import torch

from brosoundml_b200 import _lib
from tests import multilora_ref as ref
from tests.conftest import cuda_available
from tests.test_gpu_multilora import TYPES, _agree, _expect, _lora, _make, _rng, _run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


@pytest.mark.parametrize("dtype,shapes", [
    # one kernel each, whose shared memory differs by the rank, and by the columns and parts of a tile
    ("fp32", [(1, 128, 256, 128, 1, "each"), (1, 128, 256, 1, 1, "each")]),
    ("bf16", [(16, 1024, 256, 8, 2, "each"), (128, 1024, 1024, 8, 2, "each")])])
def test_threads_share_a_kernel(dtype, shapes):
    """Calls of one type and two shapes from several host threads, each on its own stream, are all taken,
    and are what they are one after the other."""
    problems = [_make(dtype, *s, seed=i) for i, s in enumerate(shapes)]
    L, C = _lora(), _lib.lib()
    want = [L.multi_lora_forward(c["x"], c["W"], c["A"], c["B"], c["ids"]) for c in problems]
    streams, outs, calls = [torch.cuda.Stream() for _ in range(4)], [], []
    for i in range(4):
        c, (M, K, N, R, nA, _) = problems[i % 2], shapes[i % 2]
        outs.append(torch.zeros_like(want[i % 2]))
        at = [c[k].data_ptr() for k in ("x", "W", "A", "B", "ids")]
        calls.append((_lib.BsmlMultiLoraShape(L.DTYPE[TYPES[dtype]], M, K, N, R, nA, 0, 0.0), at[0], K, at[1], None,
                      at[2], at[3], None, at[4], None, outs[i].data_ptr(), N, None, streams[i].cuda_stream))
    torch.cuda.synchronize()
    refused, start = [], threading.Barrier(4)

    def work(i):   # nothing but the calls, which let other threads run
        start.wait()
        for _ in range(5000):
            if C.bsml_multilora_forward(*calls[i]):
                refused.append(C.bsml_last_error().decode())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused, f"{len(refused)} calls: {refused[0]}"
    for i in range(4):
        assert torch.equal(outs[i], want[i % 2])


def test_a_refused_call_leaves_nothing_behind():
    """A call that the device refuses (scratch beyond its memory, before any launch) says so; the next one
    does not."""
    c = _make("bf16", 40, 1032, 200, 8, 4, "scattered")
    want = _run(c)
    shape = _lib.BsmlMultiLoraShape(1, (1 << 30) - 1, 1032, 200, 128, 4, 0, 0.0)
    at = [c[k].data_ptr() for k in ("x", "W", "A", "B", "ids")]
    rc = _lib.lib().bsml_multilora_forward(shape, at[0], 1032, at[1], None, at[2], at[3], None, at[4], None,
                                           want["y"].data_ptr(), 200, None, torch.cuda.current_stream().cuda_stream)
    assert rc != 0 and "memory" in _lib.lib().bsml_last_error().decode()
    got = _run(c)
    for k in want:
        assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rank", [1, 4, 12])
@pytest.mark.parametrize("rows", [2, 1500])
def test_the_smallest_adapter_at_its_buffers_end(dtype, rank, rows):
    """One adapter of one output, B alone in the last bytes of its buffer, on a 16-byte boundary."""
    c = _make(dtype, rows, 40, 1, rank, 1, "each")
    end = torch.zeros(8 * 64, dtype=TYPES[dtype], device="cuda")[:8 + rank]   # (the allocation itself is longer)
    end[8:] = c["B"].view(-1)
    c["B"] = end[8:].view(1, 1, rank)
    _agree(_run(c), _expect(c))


def test_the_adapters_gradients_alone_copy_nothing():
    """fp32 rows read where they stand: without dx the backward is the thin product and the outer ones, and
    the gradients are what they are beside dx."""
    L, C = _lora(), _lib.lib()
    c = _make("fp32", 60, 640, 520, 8, 3, "scattered")
    want = _run(c)
    n = C.bsml_launch_count()
    got = L.multi_lora_backward(c["dy"], c["x"], c["W"], c["A"], c["B"], c["ids"], want["h"], scale=c["scale"],
                                want_dx=False)
    assert C.bsml_launch_count() - n == 2
    assert torch.equal(got["dA"], want["dA"]) and torch.equal(got["dB"], want["dB"])


@pytest.mark.parametrize("M", [3, 700])
def test_gradients_need_only_their_own_operands(M):
    """dx without x and h; dA without h, dB without x: what all together give."""
    L = _lora()
    c = _make("bf16", M, 640, 1030, 16, 3, "runs", seed=5)
    want = _run(c)
    args, kw = (c["W"], c["A"], c["B"], c["ids"]), dict(scale=c["scale"])
    got = L.multi_lora_backward(c["dy"], None, *args, None, want_adapters=False, **kw)
    assert torch.equal(got["dx"], want["dx"]) and got["dA"] is None and got["dB"] is None
    got = L.multi_lora_backward(c["dy"], c["x"], *args, None, want_dx=False, want_adapters=False,
                                dA=torch.empty_like(c["A"]), **kw)
    assert torch.equal(got["dA"], want["dA"]) and got["dB"] is None
    got = L.multi_lora_backward(c["dy"], None, *args, want["h"], want_dx=False, want_adapters=False,
                                dB=torch.empty_like(c["B"]), **kw)
    assert torch.equal(got["dB"], want["dB"]) and got["dA"] is None
    with pytest.raises(TypeError, match="x: "):
        L.multi_lora_backward(c["dy"], None, *args, want["h"], **kw)
    with pytest.raises(TypeError, match="h: "):
        L.multi_lora_backward(c["dy"], c["x"], *args, None, **kw)
    with pytest.raises(ValueError, match="x: "):
        L.multi_lora_backward(c["dy"], c["x"][:, :32], *args, None, want_adapters=False, **kw)


def test_scratch_comes_back():
    """The planes of a large fp32 weight are the device's again; the next call takes them anew."""
    L = _lora()
    c = _make("fp32", 2, 4096, 8192, 8, 2, "each")
    want = _run(c)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    L.release_scratch()
    assert torch.cuda.mem_get_info()[0] - before >= 3 * 2 * 4096 * 8192
    got = _run(c)
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_a_wait_that_ran_out_is_told_and_spoils_no_later_call():
    """The code of an expired wait stands until it is read; the calls in between are what they were."""
    C = _lib.lib()
    problems = [_make("bf16", *s) for s in ((3000, 264, 2056, 8, 9, "short"), (16, 2056, 384, 8, 16, "each"))]
    want = [_run(c) for c in problems]
    assert C.bsml_device_error() == 0
    _lib.check(C.bsml_selftest_multilora_wait(torch.cuda.current_stream().cuda_stream))
    got = [_run(c) for c in problems]
    assert C.bsml_device_error() == 1
    for g, w in zip(got, want):
        for k in w:
            assert torch.equal(torch.nan_to_num(g[k]), torch.nan_to_num(w[k])), k
    assert C.bsml_device_error() == 0


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("where", ["W", "x", "A", "B"])
def test_no_numbers_hold_a_call_up(dtype, p, where):
    """A weight, rows or an adapter of NaN among short prompts: the call takes what it takes with ordinary
    numbers, up to the products of the rows beside that adapter on the CUDA cores (a few times as long; the
    shared product again for every element would be hundreds). Rows of the others keep their results."""
    M, W = {"fp32": (2500, 2048), "bf16": (5000, 4096), "fp16": (2500, 4500)}[dtype]   # fp16: a tile of several sums
    c = _make(dtype, M, W, W, 8, 5, "short", seed=2)
    bad = {k: v.clone() for k, v in c.items()}
    if where in "AB":
        bad[where][1] = float("nan")
    elif where == "W":
        bad["W"].fill_(float("nan"))
    else:
        bad["x"][::2] = float("nan")
        bad["dy"][::2] = float("inf")
    L = _lora()
    h = torch.empty(M, 8, device="cuda")

    def run(c):
        y = L.multi_lora_forward(c["x"], c["W"], c["A"], c["B"], c["ids"], h=h, **kw)
        return y, L.multi_lora_backward(c["dy"], None, c["W"], c["A"], c["B"], c["ids"], None, want_adapters=False,
                                        **kw)["dx"]

    kw = dict(dropout=p, rng=_rng() if p else None)

    def time(c):
        run(c)
        best = 1e9
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            run(c)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert time(bad) < 20 * time(c)
    assert _lib.lib().bsml_device_error() == 0
    clean = c["ids"] >= -1
    clean &= {"W": c["ids"] < -5, "A": c["ids"] != 1, "B": c["ids"] != 1,
              "x": (torch.arange(M, device="cuda") % 2 == 1)}[where]
    want, got = run(c), run(bad)
    for w, g in zip(want, got):
        w, g = w[clean].double(), g[clean].double()
        # both are within the output's rounding and the sums' of the same value
        assert bool(torch.isfinite(g).all())
        tol = torch.finfo(c["x"].dtype).eps * w.abs() + 2 * (W + 10) * 2.0**-23 * 4 * W**0.5
        assert bool(((w - g).abs() <= tol).all())


@pytest.mark.parametrize("shape", [(40, 1032, 200, 8, 4, "scattered"), (16, 1024, 320, 100, 3, "runs"), (900, 640, 1030, 16, 3, "runs"),
                                   (3000, 640, 1700, 40, 4, "short"), (600, 600, 320, 24, 2, "runs")],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("rows,adapters", [(1e-5, 300.0), (2.0**-20, 1000.0), (1.0, 1e-4)])
def test_small_numbers_between_the_products_fp16(shape, p, rows, adapters):
    """h and g of any size keep their relative accuracy beside fp16 operands: where they are far below fp16's
    normal numbers and the adapters' entries above 1, the outputs are within the bounds all the same."""
    c = _make("fp16", *shape, seed=7)
    for k in ("x", "dy"):
        c[k] *= rows
    c["A"] = (c["A"].float() * adapters).half()
    c["B"] = (c["B"].float() * adapters / 8).half()
    c["W"] *= 2.0**-6
    c["scale"] *= 2.0**-10 if adapters > 1 else 1.0
    want = _expect(c, p=p, bias=False)
    assert float(want["h"][0].abs().max()) < (0.25 if adapters > 1 else 2.0**-6)
    got = _run(c, p=p, bias=False)
    assert all(bool(torch.isfinite(got[k]).all()) for k in ("y", "dx"))
    _agree(got, {k: want[k] for k in ("y", "h", "dx")})


@pytest.mark.parametrize("M", [24, 1500])
def test_rows_of_very_different_sizes_fp16(M):
    """Rows whose numbers differ by 2^60 among neighbours, and numbers of a row by 2^16."""
    c = _make("fp16", M, 640, 320, 12, 3, "runs", seed=9)
    c["scale"] = torch.tensor([2.0**-40, 1.0, 2.0**20], device="cuda")
    c["A"][:, ::3] *= 2.0**-10
    c["x"] *= 2.0**-12
    c["x"][::2] *= 2.0**-4
    c["B"] *= 2.0**-6
    c["dy"] *= 2.0**-10
    want = _expect(c, bias=False)
    got = _run(c, bias=False)
    # (what is beyond fp16's range in the outputs is infinite there)
    for k in ("y", "h", "dx"):
        fits = want[k][0].abs() < 65000
        assert bool(torch.isfinite(got[k].cpu()[fits]).all())
        assert ref.worst(got[k].cpu()[fits], tuple(v[fits] for v in want[k])) <= 1.0, k


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rank", [2, 8, 20, 40])
@pytest.mark.parametrize("M,length", [(40, 1), (40, 16), (700, 13), (3000, 300), (3000, 9)])
def test_numbers_between_the_products_are_whole(dtype, rank, M, length):
    """Products that cancel: ranks in pairs, h = s (a, b, ..) times B = (b, -a, ..), and g = s (b, -a, ..) times
    A = (a, b, ..), with s of 24 bits. What is left is what the numbers between the products lost: nothing of
    fp32's 24 bits, 2^-22 beside fp16 operands, and 2^-23 for each of the sum's additions (an MMA for every 16
    ranks and part or plane product, 6 at most, the rows' two and the epilogue's two)."""
    L, t = _lora(), TYPES[dtype]
    K, N, nA = 640, 1700 if M > 1000 else 264, 16
    g = torch.Generator().manual_seed(rank + M)
    a = (torch.randn(nA, rank, generator=g)).to(t)
    b = torch.empty_like(a)
    b[:, 0::2], b[:, 1::2] = a[:, 1::2], -a[:, 0::2]
    A, B = a[:, :, None].expand(-1, -1, K).contiguous().cuda(), b[:, None, :].expand(-1, N, -1).contiguous().cuda()
    scale = (torch.rand(nA, generator=g) + 0.5).cuda()
    ids = (torch.arange(M) // length % nA).int().cuda()
    x, dy = torch.zeros(M, K, dtype=t, device="cuda"), torch.zeros(M, N, dtype=t, device="cuda")
    x[torch.arange(M), torch.arange(M) % K] = 1
    dy[torch.arange(M), torch.arange(M) % N] = 1
    W = torch.zeros(N, K, dtype=t, device="cuda")
    h = torch.empty(M, rank, device="cuda")
    y = L.multi_lora_forward(x, W, A, B, ids, scale=scale, h=h)
    dx = L.multi_lora_backward(dy, x, W, A, B, ids, h, scale=scale, want_adapters=False)["dx"]
    sizes = (scale.double() * (a.double() * b.double()).abs().sum(1).cuda())[ids.long()]
    adds = 6 * (-(-rank // 16)) + 4
    bound = ((2.0**-22 if dtype == "fp16" else 0.0) + adds * 2.0**-23) * sizes + (2.0**-25 if dtype == "fp16" else 0.0)
    for k, v in (("y", y), ("dx", dx)):
        worst = float((v.double().abs().amax(1) / bound).max())
        assert worst <= 1.0, f"{k}: {worst:.3g} times its bound"


def _ones_like_sums(dtype, M, K, N, R, seed=0):
    """Positive operands, whose sums a truncation always pulls the same way; adapters of one type and size."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[dtype]
    u = lambda *s, f=1.0: (torch.rand(*s, generator=g, device="cuda") * f).to(t)  # noqa: E731
    return dict(x=u(M, K), W=u(N, K, f=1 / K), A=u(1, R, K, f=1 / K), B=u(1, N, R, f=1 / R), dy=u(M, N, f=1 / N),
                ids=torch.zeros(M, dtype=torch.int32, device="cuda"))


# How far a sum of positive numbers may be off, whatever its length. Products and additions on the tensor cores are
# each off by at most 2^-23 of the sum so far (truncated), so a piece of n columns, whose sum grows evenly, by
# n / 2 * 2^-23 of its value, and the sum of all pieces (rounded to nearest, 2^-24 times the square root of their number)
# by as much: fp32's pieces are 512 columns, fp16's 4096, bf16's 16384. (Without pieces 2^20 columns may be off by 2^-4, and
# were by 2^-10.)
LONG = {"fp32": 512 / 2 * 2.0**-23, "fp16": 4096 / 2 * 2.0**-23, "bf16": 16384 / 2 * 2.0**-23}


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N", [(8, 1 << 20, 128), (130, 1 << 17, 264), (40, 20000, 2056), (700, 60000, 1700), (2000, 9000, 2056)])
def test_long_sums_of_the_shared_product(dtype, M, K, N):
    """Sums over up to 2^20 columns, forward and backward, with no adapter at work: rounded once from a sum
    that is off by no more than the bounds above."""
    L = _lora()
    rows = min(M, 64)
    eps = torch.finfo(TYPES[dtype]).eps / 2
    held = LONG[dtype]
    for back in (False, True):
        c = _ones_like_sums(dtype, M, K if not back else N, N if not back else K, 8)
        c["ids"].fill_(-1)
        if back:
            got = L.multi_lora_backward(c["dy"], None, c["W"], c["A"], c["B"], c["ids"], None, want_adapters=False)["dx"]
            z, W = c["dy"][:rows], c["W"]
        else:
            got = L.multi_lora_forward(c["x"], c["W"], c["A"], c["B"], c["ids"])
            z, W = c["x"][:rows], c["W"].T
        want = torch.zeros(rows, N, dtype=torch.float64, device="cuda")
        for k in range(0, K, 16384):
            want += z[:, k:k + 16384].double() @ W[k:k + 16384].double()
        off = ((got[:rows].double() - want).abs() - eps * want - (2.0**-25 if dtype == "fp16" else 0)) / want
        assert float(off.max()) <= held, f"{'dx' if back else 'y'}: off by {float(off.max()):.3g}, bound {held:.3g}"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,R", [(8, 1 << 20, 8), (64, 1 << 18, 16), (1100, 20000, 16), (1100, 60000, 40), (2000, 4096, 8)])
def test_long_sums_of_the_thin_products(dtype, M, K, R):
    """h over up to 2^20 columns, and g (by dA of one row whose x is one): sums of positive numbers off by no more than
    2^-23 of themselves for each of a piece's additions, half of that as the piece grows: 512 columns a piece
    beside 16-bit operands, 64 of six plane products beside fp32 ones, split over eight warps; the pieces, at most
    2^11, rounded to nearest, 2^-24 each in the root of their number."""
    L = _lora()
    pieces = (384 if dtype == "fp32" else 512) / 2 * 2.0**-23 + 2.0**5.5 * 2.0**-24
    c = _ones_like_sums(dtype, M, K, 64, R)
    c["W"].zero_()
    h = torch.empty(M, R, device="cuda")
    L.multi_lora_forward(c["x"], c["W"], c["A"], c["B"], c["ids"], h=h)
    rows = min(M, 64)
    want = torch.zeros(rows, R, dtype=torch.float64, device="cuda")
    for k in range(0, K, 16384):
        want += c["x"][:rows, k:k + 16384].double() @ c["A"][0, :, k:k + 16384].double().T
    off = float(((h[:rows].double() - want) / want).abs().max())
    assert off <= pieces, f"h: off by {off:.3g}, bound {pieces:.3g}"
    # g of row 3 alone: x is zero in the others, and each column of dA is then g
    c = _ones_like_sums(dtype, M, 64, K, R)
    c["x"].zero_()
    c["x"][3] = 1
    dA = L.multi_lora_backward(c["dy"], c["x"], torch.zeros_like(c["W"]), c["A"], c["B"], c["ids"], None, want_dx=False,
                               want_adapters=False, dA=torch.empty_like(c["A"]))["dA"]
    want = torch.zeros(R, dtype=torch.float64, device="cuda")
    for k in range(0, K, 16384):
        want += c["B"][0, k:k + 16384].double().T @ c["dy"][3, k:k + 16384].double()
    eps = torch.finfo(TYPES[dtype]).eps / 2
    off = ((dA[0].double() - want[:, None]).abs() - (2.0**-25 if dtype == "fp16" else 0)) / want[:, None] - eps
    assert float(off.max()) <= pieces + 2.0**-21, f"g: off by {float(off.max()):.3g}"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,R,nA", [(1 << 20, 8, 1), (1 << 20, 8, 100), (200000, 100, 1), (3000, 40, 2)])
def test_long_sums_of_the_adapters_gradients(dtype, M, R, nA):
    """dA and dB over up to 2^20 rows of one adapter, positive numbers: off by their output's rounding and 2^-23 of
    the sum for each of a piece's additions, half of that as the piece grows (64 rows of four products for
    fp32, 1024 of two for 16-bit types, whose 2^-23 of g and h are within), and 2^-22 for an fp32 product's operands;
    the pieces, at most 2^11 a warp and 2^8 warps' sums, rounded to nearest. g is a power of two, exactly."""
    L, t = _lora(), TYPES[dtype]
    K = N = 64
    held = (64 * 4 if dtype == "fp32" else 1024 * 2) / 2 * 2.0**-23 + 2.0**-22 + 2.0**-19
    g = torch.Generator(device="cuda").manual_seed(R)
    x, dy = torch.rand(M, K, generator=g, device="cuda").to(t), torch.rand(M, N, generator=g, device="cuda").to(t)
    h = torch.rand(M, R, generator=g, device="cuda") / M
    ids = torch.full((M,), nA - 1, dtype=torch.int32, device="cuda")
    W, A = torch.zeros(N, K, dtype=t, device="cuda"), torch.zeros(nA, R, K, dtype=t, device="cuda")
    B = torch.zeros(nA, N, R, dtype=t, device="cuda")
    B[:, 0] = 1
    dy[:, 0] = 0.5
    scale = torch.full((nA,), 1.0 / M, device="cuda")
    got = L.multi_lora_backward(dy, x, W, A, B, ids, h, scale=scale, want_dx=False)
    gr = 0.5 * float(scale[0])
    want_A = sum(x[i:i + 65536].double().sum(0) for i in range(0, M, 65536)) * gr
    want_B = sum(dy[i:i + 65536].double().T @ h[i:i + 65536].double() for i in range(0, M, 65536))
    eps = torch.finfo(t).eps / 2
    for k, v, w in (("dA", got["dA"][nA - 1], want_A[None].expand(R, -1)), ("dB", got["dB"][nA - 1], want_B)):
        off = float(((v.double() - w).abs() / w).max()) - eps
        assert off <= held, f"{k}: off by {off:.3g} more than its rounding, bound {held:.3g}"
    assert not got["dA"][:nA - 1].any() and not got["dB"][:nA - 1].any()


def test_numbers_at_the_end_of_the_range():
    """fp32's largest numbers times small ones are finite in every output."""
    L = _lora()
    M, K, N, R = 40, 640, 264, 8
    big = torch.finfo(torch.float32).max
    c = dict(_ones_like_sums("fp32", M, K, N, R), W=torch.full((N, K), 1e-12, device="cuda"))
    c["A"].fill_(1e-12)
    c["B"].fill_(1e-12)
    c["x"].fill_(big)
    h = torch.empty(M, R, device="cuda")
    y = L.multi_lora_forward(c["x"], c["W"], c["A"], c["B"], c["ids"], h=h)
    assert float((y.double() / (big * K * 1e-12) - 1).abs().max()) < 2.0**-18   # (W's and A's own roundings, fp32 sums)
    dy = torch.full((M, N), 1e-6, device="cuda")
    dA = L.multi_lora_backward(dy, c["x"], c["W"], c["A"], c["B"], c["ids"], h, want_dx=False)["dA"]
    assert float((dA.double() / (M * big * N * 1e-18) - 1).abs().max()) < 2.0**-18
    dy.fill_(big)
    dB = L.multi_lora_backward(dy, c["x"], c["W"], c["A"], c["B"], c["ids"], torch.full_like(h, 1e-12), want_dx=False)["dB"]
    assert float((dB.double() / (M * big * 1e-12) - 1).abs().max()) < 2.0**-18
