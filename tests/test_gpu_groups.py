"""gemv_i4_groups against its formula in 64 bits.

Tolerance. u = 2^-24 is half a step of f32, A = sum |s c x| over a row, B the same with each |x| replaced by the largest of
its 128 neighbours. A vector's elements are rounded to 2^-24 of that largest (B u), or
to 2^-127 where that is more (the factor that makes them integers is 2^126 at most): 2^-127 C, C the sum of |s c|; a group's sum is exact, or (more than
eight vectors) of f16 pairs, which are 4 u off, by a unit that adds 16 products at a time and cuts off: 2 u for each of 8
steps and as much again inside a step; its conversion, the joining of partial sums, the unit, the scale and each addition of
a group's result to the row's are roundings of at most A; the bias one more: u (B + (groups + 32) A + 2 |y|) + 2^-127 C."""
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch


@pytest.fixture
def rt(pkg):
    return pkg.runtime


def make(torch, m, n, T, group, dtype, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = (n + 31) // 32 * 16
    W = torch.randint(0, 256, (m, ld), device="cuda", generator=g, dtype=torch.uint8)      # also past n
    scale = (0.01 * torch.randn(m, -(-n // group), device="cuda", generator=g)).to(dtype)  # negative ones too
    x = torch.randn(T, n + pad, device="cuda", generator=g)[:, :n]
    return W, scale, x


def product64(torch, W, scale, x, group, bias=None):
    n = x.shape[1]
    codes = torch.stack((W & 15, W >> 4), -1).flatten(1)[:, :n].to(torch.int32)
    w = (torch.where(codes > 7, codes - 16, codes).double() * scale.double().repeat_interleave(group, 1)[:, :n])
    xd = x.double()
    top = torch.nn.functional.pad(xd.abs(), (0, -n % 128)).unflatten(1, (-1, 128)).amax(-1).repeat_interleave(128, 1)[:, :n]
    y = xd @ w.T + (0 if bias is None else bias.double())
    a, b = xd.abs() @ w.abs().T, top @ w.abs().T
    return y, U * (b + (scale.shape[1] + 32) * a + 2 * y.abs()) + 2.0 ** -127 * w.abs().sum(1)


def close(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / tol.clamp(min=1e-300)).nan_to_num(1e9).max()))


SHAPES = [(1, 1, 1), (1, 32, 1), (7, 31, 2), (16, 128, 1), (17, 130, 3), (64, 257, 1), (130, 4096, 1), (100, 1000, 5),
          (333, 1111, 8), (257, 2048, 13), (128, 4098, 16), (129, 640, 17), (300, 5632, 33), (148, 11008, 64), (65, 384, 65),
          (40, 96, 200), (5000, 64, 1), (4099, 160, 7), (20, 16384, 2), (3, 16001, 9), (18, 30000, 1),
          (5, 40002, 7)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,T", SHAPES)
def test_products(torch, rt, m, n, T, group):
    dtype = torch.bfloat16 if (m + n + T) % 2 else torch.float32
    W, scale, x = make(torch, m, n, T, group, dtype, seed=m + n)
    want, tol = product64(torch, W, scale, x, group)
    close(rt.gemv_i4_groups(W, scale, x, group), want, tol)


@pytest.mark.parametrize("T", [1, 2, 5, 16, 40])
def test_bias_strides_and_rows_of_a_wider_buffer(torch, rt, T):
    """x and y as slices with odd strides; what lies beside y stays."""
    m, n = 77, 515
    W, scale, x = make(torch, m, n, T, 64, torch.float32, pad=6)
    bias = torch.randn(m, device="cuda")
    big = torch.full((T + 2, m + 5), 7.0, device="cuda")
    y = rt.gemv_i4_groups(W, scale, x, 64, bias=bias, y=big[1:T + 1, 3:m + 3])
    want, tol = product64(torch, W, scale, x, 64, bias)
    close(y, want, tol)
    big[1:T + 1, 3:m + 3] = 7.0
    assert bool((big == 7.0).all())


@pytest.mark.parametrize("n", [33, 160, 1000, 1120])
@pytest.mark.parametrize("T", [1, 5, 9, 20, 64])
def test_columns_at_the_end_of_a_wider_matrix(torch, rt, T, n):
    """W as the last columns of a wider matrix that ends with its memory: 16-byte aligned rows that are `wide` bytes apart
    (through the C call: the wrapper takes whole rows)."""
    m, group, wide = 300, 32, 4096
    big = torch.randint(0, 256, (8192, wide), device="cuda", dtype=torch.uint8)            # 32 MB: memory of its own
    own = (n + 31) // 32 * 16
    W, scale, x = make(torch, m, n, T, group, torch.float32, seed=n + T)
    at = (8192 - m) * wide + wide - own
    view = big.view(-1)[at:]
    big[8192 - m:, wide - own:] = W[:, :own]
    y, ws = torch.empty(T, m, device="cuda"), rt.gemv_i4_groups_workspace(T, n)
    rt.check(rt.lib().b2_gemv_i4_groups(view.data_ptr(), wide, scale.data_ptr(), scale.shape[1], 0, group, x.data_ptr(), n, None,
                                        y.data_ptr(), m, m, n, T, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    want, tol = product64(torch, W, scale, x, group)
    close(y, want, tol)


def test_one_vector_without_a_row(torch, rt):
    W, scale, x = make(torch, 50, 300, 1, 128, torch.bfloat16)
    want, tol = product64(torch, W, scale, x, 128)
    y = rt.gemv_i4_groups(W, scale, x[0], 128)
    assert y.shape == (50,)
    close(y[None], want, tol)


@pytest.mark.parametrize("T", [1, 3, 16, 64])
def test_large_channels_cost_their_neighbours_alone(torch, rt, T):
    """A channel 10^4 times the others: elements outside its 128 neighbours keep their precision."""
    W, scale, x = make(torch, 40, 1024, T, 128, torch.float32)
    x[:, 700] = 1e4
    scale[:, 5] = 0                                                # its group counts nothing: what is left are the others
    want, tol = product64(torch, W, scale, x, 128)
    close(rt.gemv_i4_groups(W, scale, x, 128), want, tol)


@pytest.mark.parametrize("factor", [1e-30, 1e-38, 1e30])
def test_ranges(torch, rt, factor):
    """Tiny and huge vectors, and one of zeros."""
    W, scale, x = make(torch, 40, 500, 4, 32, torch.float32)
    x *= factor
    x[2] = 0
    y = rt.gemv_i4_groups(W, scale, x, 32)
    want, tol = product64(torch, W, scale, x, 32)
    close(y, want, tol + 600 * 8 * 2.0 ** -149)                    # below f32's normal numbers a step is 2^-149
    assert not y[2].any()


@pytest.mark.parametrize("T", [1, 2, 5, 8, 9, 40])
@pytest.mark.parametrize("x_factor,s_factor", [(1e-12, 1e-20), (1.0, 1e-30), (1e-30, 1.0), (1e-24, 1e-10), (1e25, 1e-30), (1e-30, 1e30), (1e30, 1e5)])
def test_small_and_large_scales(torch, rt, T, x_factor, s_factor):
    """Outputs down to 1e-33 from factors that are small each: as precise as any (what f32 cannot hold on the way, its last
    digits below 2^-149, is left to it: a step for each group of each of three sums)."""
    W, scale, x = make(torch, 40, 500, T, 32, torch.float32, seed=T)
    x *= x_factor
    scale *= s_factor
    want, tol = product64(torch, W, scale, x, 32)
    close(rt.gemv_i4_groups(W, scale, x, 32), want, tol + 3 * 16 * 2.0 ** -149)


@pytest.mark.parametrize("T", [1, 2, 5, 8, 9, 40])
@pytest.mark.parametrize("group", [32, 128])
def test_vectors_up_to_the_largest_number(torch, rt, T, group):
    """All elements of the size of f32's largest, scales that bring their sums back."""
    W, scale, x = make(torch, 40, 500, T, group, torch.float32, seed=T)
    x = x.sign() * (3.0e38 + 0.4e38 * x.abs().clamp(max=1))
    scale *= 1e-4
    want, tol = product64(torch, W, scale, x, group)
    close(rt.gemv_i4_groups(W, scale, x, group), want, tol)
    W.fill_(0x77)                                                  # sums as large as they come
    x.abs_()
    want, tol = product64(torch, W, scale, x, group)
    close(rt.gemv_i4_groups(W, scale, x, group), want, tol)


@pytest.mark.parametrize("T", [1, 2, 9, 30])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_stays_in_its_vector(torch, rt, T, bad):
    W, scale, x = make(torch, 33, 400, T, 64, torch.float32)
    x[0, 130] = bad
    y = rt.gemv_i4_groups(W, scale, x, 64)
    assert bool(y[0].isnan().all())
    if T > 1:
        want, tol = product64(torch, W, scale, x[1:], 64)
        close(y[1:], want, tol)


def test_non_finite_scale_stays_in_its_row(torch, rt):
    W, scale, x = make(torch, 33, 400, 3, 64, torch.float32)
    scale[4, 2] = float("nan")
    y = rt.gemv_i4_groups(W, scale, x, 64)
    assert bool(y[:, 4].isnan().all()) and int(y.isnan().sum()) == 3


def test_quantised_weights(torch, rt, pkg):
    import numpy as np
    w = np.random.default_rng(0).standard_normal((60, 515)).astype(np.float32)
    W, scale = (torch.from_numpy(a).cuda() for a in pkg.pack.quantize_groups_i4(w, 64))
    x = torch.randn(6, 515, device="cuda")
    y = rt.gemv_i4_groups(W, scale, x, 64)
    want, tol = product64(torch, W, scale, x, 64)
    close(y, want, tol)
    # a code is at most half a step of its group off
    w64, step = torch.from_numpy(w).cuda().double(), scale.double().repeat_interleave(64, 1)[:, :515]
    assert bool(((y.double() - x.double() @ w64.T).abs() <= 0.5001 * x.double().abs() @ step.T + tol).all())


@pytest.mark.parametrize("T", [1, 4, 20])
def test_capture_and_replay(torch, rt, T):
    """Two graphs with a workspace each, replayed at once on two streams with new inputs."""
    cases = []
    for i in range(2):
        W, scale, x = make(torch, 500, 1024, T, 64, torch.float32, seed=i)
        x = x.contiguous()
        y, ws = torch.zeros(T, 500, device="cuda"), rt.gemv_i4_groups_workspace(T, 1024)
        rt.gemv_i4_groups(W, scale, x, 64, y=y, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            rt.gemv_i4_groups(W, scale, x, 64, y=y, workspace=ws)
        cases.append((g, W, scale, x, y, torch.cuda.Stream()))
    for rnd in range(3):
        for g, W, scale, x, y, s in cases:
            x.copy_(torch.randn_like(x) * (rnd + 1))
        torch.cuda.synchronize()
        for g, *_, s in cases:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, W, scale, x, y, s in cases:
            want, tol = product64(torch, W, scale, x, 64)
            close(y, want, tol)


def test_another_stream_and_order_behind_it(torch, rt):
    W, scale, x = make(torch, 2000, 2048, 3, 128, torch.float32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x2 = x * 2
        y = rt.gemv_i4_groups(W, scale, x2, 128)
        z = y * 1
    y3 = rt.gemv_i4_groups(W, scale, x, 128, stream=s.cuda_stream)
    s.synchronize()
    want, tol = product64(torch, W, scale, x, 128)
    close(z, 2 * want, 2 * tol)
    close(y3, want, tol)


def test_threads_with_calls_of_different_sizes(torch, rt):
    """Threads on streams of their own, whose calls need different amounts of shared memory; the first calls are theirs."""
    import threading
    cases = [make(torch, 48, n, T, 64, torch.bfloat16, seed=n) for n, T in ((9000, 1), (128, 1), (20000, 2), (640, 2), (4000, 4), (256, 5))]
    want = [product64(torch, *c, 64) for c in cases]
    torch.cuda.synchronize()
    got, failed = [[] for _ in cases], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i].append(rt.gemv_i4_groups(*cases[i], 64))
            s.synchronize()
        except Exception as e:                                     # noqa: BLE001 (told by the assertion)
            failed.append(repr(e))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for ys, (y, tol) in zip(got, want):
        assert len(ys) == 20
        for z in ys:
            close(z, y, tol)


def test_same_bits_every_time(torch, rt):
    for T in (1, 6, 24):
        W, scale, x = make(torch, 700, 3000, T, 32, torch.bfloat16)
        y = rt.gemv_i4_groups(W, scale, x, 32)
        for _ in range(5):
            assert torch.equal(y, rt.gemv_i4_groups(W, scale, x, 32))


def test_bad_tensors_are_refused(torch, rt):
    W, scale, x = make(torch, 16, 64, 2, 32, torch.float32)
    for bad in (dict(x=x.double()), dict(x=x.cpu()), dict(x=x.t().contiguous().t()), dict(W=W.to(torch.int8)), dict(W=W[:, ::2]),
                dict(scale=scale.half()), dict(scale=scale[:, :1]), dict(group=48), dict(bias=torch.zeros(15, device="cuda")),
                dict(y=torch.zeros(2, 15, device="cuda")), dict(y=torch.zeros(16, 2, device="cuda").t()), dict(x=x[:, :63], W=W[:, :16]),
                dict(y=x[:, :16]), dict(workspace=torch.zeros(8, device="cuda"))):
        a = dict(W=W, scale=scale, x=x, group=32, bias=None, y=None, workspace=None)
        a.update(bad)
        with pytest.raises(rt.B2Error):
            rt.gemv_i4_groups(**a)
