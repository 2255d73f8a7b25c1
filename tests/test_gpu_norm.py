"""Residual add, RMS norm and 8-bit rows in one launch, and the 8-bit rows read back.

Tolerance of the normed rows, from the arithmetic: t is one addition (2^-24 of it), the sum of squares adds at most 64 squares a thread and 5 + 32 partial
sums, each off by 2^-24 of the sum: with the division, eps and the square's own rounding at most 104 * 2^-24 of the sum, half of that in its root; rsqrt is
within 2 ulp (2^-22) and two products follow: |x| * (1 + 52 + 4 + 2) * 2^-24 < |x| * 2^-18.  A bf16 row adds its own rounding, 2^-8 |x|.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
EPS = 1e-6


def rows_of(T, seed, rows, n, dtype, lead=0, gap=0):
    """[rows, n] values, `lead` elements behind an aligned start and `gap` between the rows."""
    g = T.Generator(device="cuda").manual_seed(seed)
    x = T.randn((rows, lead + n + gap), generator=g, device="cuda") * (0.1 + 3 * T.rand((rows, 1), generator=g, device="cuda"))
    return x.to(dtype)[:, lead:lead + n]


def check(T, rows, n, h, add, x_dtype, image, eps=EPS):
    from project_maya_b200 import api
    w = 1 + 0.3 * T.randn(n, device="cuda")
    h_out = T.full((rows, n), 7.0, device="cuda").to(h.dtype)
    x = T.full((rows, n), 7.0, device="cuda").to(x_dtype)
    xq = api.rms_q8(h, add, w, eps, image=image, h_out=h_out, x=x)
    t = h.double() + (add.double() if add is not None else 0.0)
    want = t / T.sqrt((t * t).mean(-1, keepdim=True) + eps) * w.double()
    exact = h.float() + add.float() if add is not None else h.float()
    assert T.equal(h_out, exact.to(h.dtype))
    tol = want.abs() * (2.0 ** -18 + (2.0 ** -8 if x_dtype == T.bfloat16 else 0.0)) + 1e-37
    assert bool(((x.double() - want).abs() <= tol).all())
    if image is None:
        assert xq is None
        return
    x32 = T.empty((rows, n), device="cuda")
    api.rms_q8(h, add, w, eps, image=None, x=x32)
    other = api.native_quantize_q8_1(x32) if image == api.XQ_Q8_1 else api.mmq_quantize(x32, None, api.Q8_0)
    assert T.equal(xq.view(-1)[:other.numel()], other.view(-1))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,n", [(1, 32), (1, 6144), (3, 96), (2, 8192), (5, 8224), (1, 32768), (300, 512), (200, 6144), (150, 32768), (149, 16416),
                                    (400, 224)])
@pytest.mark.parametrize("image", [1, 2])
def test_rows_and_their_8_bit_form(cuda, dtype, rows, n, image):
    import torch as T
    dt = getattr(T, dtype)
    check(T, rows, n, rows_of(T, n, rows, n, dt), rows_of(T, n + 1, rows, n, dt), T.float32, image)
    check(T, rows, n, rows_of(T, n + 2, rows, n, dt), None, T.bfloat16, image)


@pytest.mark.parametrize("rows,n", [(1, 1), (2, 7), (3, 33), (200, 40), (4, 8200), (1, 30001)])
def test_rows_of_any_length_without_an_image(cuda, rows, n):
    import torch as T
    for dt, ad, xd in ((T.float32, T.float32, T.float32), (T.bfloat16, T.float32, T.bfloat16), (T.float32, T.bfloat16, T.float32)):
        check(T, rows, n, rows_of(T, n, rows, n, dt), rows_of(T, n + 1, rows, n, ad), xd, None)


@pytest.mark.parametrize("lead,gap", [(8, 8), (1, 2), (3, 0), (4, 12)])
def test_rows_that_lie_apart_and_off_the_alignment(cuda, lead, gap):
    import torch as T
    for dt in (T.float32, T.bfloat16):
        for rows, n in ((1, 64), (5, 608), (170, 2048)):
            for image in (1, 2):
                check(T, rows, n, rows_of(T, 1, rows, n, dt, lead, gap), rows_of(T, 2, rows, n, dt, gap, lead), T.float32, image)


def test_in_place(cuda):
    import torch as T
    from project_maya_b200 import api
    w = T.ones(4096, device="cuda")
    for rows in (1, 9, 200):
        h, add = rows_of(T, 1, rows, 4096, T.float32), rows_of(T, 2, rows, 4096, T.float32)
        x = T.empty_like(h)
        h_out = T.empty_like(h)
        xq = api.rms_q8(h, add, w, EPS, h_out=h_out, x=x)
        a, b, c = h.clone(), add.clone(), h.clone()
        assert T.equal(api.rms_q8(a, add, w, EPS, h_out=a), xq) and T.equal(a, h_out)
        assert T.equal(api.rms_q8(h, b, w, EPS, h_out=b), xq) and T.equal(b, h_out)
        assert T.equal(api.rms_q8(c, add, w, EPS, x=c), xq) and T.equal(c, x)


def test_zeros_infinities_and_nan_stay_in_their_rows(cuda):
    import torch as T
    from project_maya_b200 import api
    w = T.ones(512, device="cuda")
    h = rows_of(T, 3, 5, 512, T.float32).clone()
    h[1] = 0.0
    h[2, 7] = float("nan")
    h[3, 500] = float("inf")
    for image in (1, 2):
        x = T.empty_like(h)
        xq = api.rms_q8(h, None, w, EPS, image=image, x=x)
        other = api.native_quantize_q8_1(x) if image == 1 else api.mmq_quantize(x, None, api.Q8_0)
        assert T.equal(xq.view(-1), other.view(-1))
        assert bool((x[1] == 0).all()) and bool(x[2].isnan().all()) and bool(x[3].isnan().any()) and bool(x[[0, 4]].isfinite().all())
        alone = T.empty_like(h[:1])
        api.rms_q8(h[4:5], None, w, EPS, image=None, x=alone)
        assert T.equal(alone[0], x[4])


def test_a_row_is_the_same_beside_others(cuda):
    """A row alone (a thread a run) and among many (four runs a thread) adds its squares in another order: equal to the tolerance, not to the bit; the
    same call gives the same bits."""
    import torch as T
    from project_maya_b200 import api
    w = T.ones(6144, device="cuda")
    h = rows_of(T, 4, 400, 6144, T.float32)
    x, y, one = T.empty_like(h), T.empty_like(h), T.empty_like(h[:1])
    a, b = api.rms_q8(h, None, w, EPS, x=x), api.rms_q8(h, None, w, EPS, x=y)
    api.rms_q8(h[5:6], None, w, EPS, image=None, x=one)
    assert T.equal(a, b) and T.equal(x, y)
    assert bool(((one[0] - x[5]).abs() <= 2.0 ** -17 * x[5].abs()).all())


@pytest.mark.parametrize("image", [1, 2])
def test_read_back(cuda, image):
    import torch as T
    from project_maya_b200 import api
    for rows, n in ((1, 32), (3, 96), (7, 2080), (129, 512)):
        x = rows_of(T, n, rows, n, T.float32).contiguous()
        xq = api.native_quantize_q8_1(x) if image == 1 else api.mmq_quantize(x, None, api.Q8_0)
        raw = xq.cpu().numpy().view(np.uint8)
        if image == 1:
            b = raw.reshape(rows, n // 32, 36)
            d, s = (b[..., i:i + 2].copy().view(np.float16).astype(np.float32) for i in (0, 2))
            want, sums = (b[..., 4:].view(np.int8) * d).reshape(rows, n), s[..., 0]
        else:
            b = raw.view(np.float16).reshape(rows, -1).astype(np.float32)
            want = b[:, :n]
            sums = b[:, n:n + n // 32] + want.reshape(rows, -1, 32).sum(-1, dtype=np.float32)
        for dt in (T.float32, T.bfloat16):
            values, got = api.q8_read(xq, rows, n, image, dtype=dt)
            assert T.equal(values.cpu(), T.from_numpy(want).to(dt))
            assert T.equal(got.cpu(), T.from_numpy(sums).half())
        # the sums are those of the values before rounding: 32 additions in f32, one rounding to f16 (and for the image the stored difference's and the result's)
        assert bool(((got.double() - x.double().view(rows, -1, 32).sum(-1)).abs() <= 2.0 ** -9 * x.view(rows, -1, 32).abs().sum(-1)).all())


def test_captured_and_on_another_stream(cuda):
    import torch as T
    from project_maya_b200 import api
    w = T.ones(2048, device="cuda")
    h, add = rows_of(T, 5, 3, 2048, T.float32), rows_of(T, 6, 3, 2048, T.float32)
    h_out, xq = T.empty_like(h), T.empty(api.xq_bytes(api.XQ_MMQ, 3, 2048), dtype=T.uint8, device="cuda")
    s = T.cuda.Stream()
    s.wait_stream(T.cuda.current_stream())
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g, stream=s):
        api.rms_q8(h, add, w, EPS, image=api.XQ_MMQ, xq=xq, h_out=h_out)
    for seed in (7, 8):
        h.copy_(rows_of(T, seed, 3, 2048, T.float32))
        g.replay()
        want_h = T.empty_like(h)
        want = api.rms_q8(h, add, w, EPS, image=api.XQ_MMQ, h_out=want_h)
        assert T.equal(xq, want) and T.equal(h_out, want_h)


def test_feeds_the_products(cuda):
    """rms_q8 in front of the GEMV and of the prompt path's GEMM: the same outputs as norm and quantizer by themselves."""
    import torch as T
    from project_maya_b200 import api
    n, out = 512, 256
    w = T.ones(n, device="cuda")
    weights = api.synth_weights(api.Q8_0, 3, 0.02, out, n)
    for rows in (1, 8, 70):
        h, add = rows_of(T, 9, rows, n, T.float32), rows_of(T, 10, rows, n, T.float32)
        x = T.empty_like(h)
        if rows <= api.MAX_COLS:
            y = api.native_mmvq(api.Q8_0, weights, api.rms_q8(h, add, w, EPS, x=x), n, out, rows)
            assert T.equal(y, api.native_mmvq(api.Q8_0, weights, api.native_quantize_q8_1(x), n, out, rows))
        else:
            bounds, ys = T.tensor([0, rows], dtype=T.int32, device="cuda"), []
            for q in (api.rms_q8(h, add, w, EPS, image=api.XQ_MMQ, x=x), api.mmq_quantize(x, None, api.Q8_0)):
                ys.append(T.empty((rows, out), device="cuda"))
                api.mmq_run(api.mmq_product(weights, api.Q8_0, out, n, weights.numel(), 1, q, bounds, None, rows, ys[-1], out))
            assert T.equal(*ys)
