"""Norms of q, k and v for each head with the rotation by positions of one or
several axes, against the formulas in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def rows(seed, shape, scale=1.0):
    import torch

    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale
    return x.bfloat16().cuda()


def reference(x, w, eps, pos=None, rope_dims=0, theta=1.0, sections=()):
    """f64 of bf16 rows [n, heads, D]; w None: no weight."""
    import torch

    x = x.double().cpu()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double().cpu()
    half = rope_dims // 2
    if pos is None or half == 0:
        return y
    axis = np.repeat(np.arange(len(sections)), sections)
    f = theta ** (-np.arange(half, dtype=np.float64) / half)
    ang = torch.from_numpy(pos.cpu().numpy().astype(np.float64).reshape(len(sections), -1).T[:, axis] * f)[:, None]
    a, b = y[..., :half], y[..., half:rope_dims]
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), y[..., rope_dims:]], -1)


def check(out, ref, what, far=0, theta=1e4):
    """bf16 outputs of values y, |y| <= 2^6: half a step of their own, 2^-8 |y|;
    the f32 sums, root and products before it 2^-20 |row|; sines and cosines in
    turns, to 2^-20, and an angle of 2^-24 of a turn: 2^-19 of the pair's size.
    (What far positions lose in the reference's own 64 bits: 2^-53 of the
    angle, twice.)"""
    got = out.double().cpu()
    size = ref.abs().amax(-1, keepdim=True)
    allow = 2.0 ** -8 * ref.abs() + (2.0 ** -18 + far * 2.0 ** -51) * size
    bad = ~((got - ref).abs() <= allow)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} off, largest {float((got - ref).abs().max()):.3e}"


def prologue(gpu, D, rope_dims, theta=1e6, **kw):
    return gpu.make_qkv_prologue(1 + rows(91, (D,), 0.3), 1 + rows(92, (D,), 0.3), 1e-6, rope_dims, theta, **kw)


def run_and_check(gpu, n, Hq, Hkv, D, rope_dims, sections, pos, theta=1e6, fused=False, seed=1, **kw):
    import torch

    pro = prologue(gpu, D, rope_dims, theta, sections=sections, **kw)
    if fused:
        x = rows(seed, (n, Hq + 2 * Hkv + 1, D))  # (and a row that belongs to none)
        q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:Hq + 2 * Hkv]
    else:
        q, k, v = rows(seed, (n, Hq, D)), rows(seed + 1, (n, Hkv, D)), rows(seed + 2, (n, Hkv, D), 3.0)
    p = torch.from_numpy(np.asarray(pos, np.int32)).cuda()
    far = int(np.abs(np.asarray(pos, np.int64)).max()) if n else 0
    oq, ok, ov = gpu.qkv_norm_rope(q, k, v, p, pro)
    torch.cuda.synchronize()
    cut = sections or (rope_dims // 2,)
    check(oq, reference(q, pro.weights[0], 1e-6, p, rope_dims, theta, cut), "q", far)
    check(ok, reference(k, pro.weights[1], 1e-6, p, rope_dims, theta, cut), "k", far)
    check(ov, reference(v, None, 1e-6) if pro.v_norm else v.double().cpu(), "v")


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("n", [1, 2, 33, 1000])
@pytest.mark.parametrize("Hq,Hkv", [(16, 8), (16, 2), (7, 1), (1, 1)])
def test_norm_rope(gpu, D, n, Hq, Hkv):
    rng = np.random.default_rng(n)
    run_and_check(gpu, n, Hq, Hkv, D, D, None, rng.integers(0, 40000, n), fused=n % 2 == 1)


@pytest.mark.parametrize("D,rope_dims,sections", [
    (128, 0, None), (128, 8, None), (128, 24, None), (128, 96, None), (256, 64, (8, 12, 12)), (256, 256, (64, 64)),
    (512, 128, (16, 24, 24)), (512, 512, (1, 2, 3, 250)), (128, 128, (0, 64, 0)), (256, 200, (33, 33, 34))])
def test_parts_of_a_head_and_axes(gpu, D, rope_dims, sections):
    n, axes = 77, len(sections or (1,))
    rng = np.random.default_rng(D + rope_dims)
    pos = rng.integers(0, 5000, (axes, n))
    if rope_dims == 0:
        pos[:] = 0
    run_and_check(gpu, n, 5, 3, D, rope_dims, sections, pos, theta=1e4)


@pytest.mark.parametrize("theta", [1.0, 1e4, 1e6])
def test_far_and_negative_positions(gpu, theta):
    """Angles keep their precision at every 32-bit position."""
    pos = [0, 1, -1, 99999, 1 << 20, -(1 << 20), (1 << 24) + 1, (1 << 31) - 1, -(1 << 31)]
    run_and_check(gpu, len(pos), 3, 2, 256, 256, None, pos, theta=theta)


def test_values_that_are_not_ordinary(gpu):
    """Zero rows stay zero, tiny rows lean on eps, an infinity or NaN stays in its
    row."""
    import torch

    D = 256
    pro = prologue(gpu, D, D)
    q, k = rows(1, (6, 4, D)), rows(2, (6, 2, D))
    q[0], q[1], k[0, 1] = 0, q[1] * 1e-6, 0
    clean = gpu.qkv_norm_rope(q, k, k, torch.arange(6, dtype=torch.int32, device="cuda"), pro)
    torch.cuda.synchronize()
    pos = torch.arange(6, dtype=torch.int32)
    check(clean[0], reference(q, pro.weights[0], 1e-6, pos, D, 1e6, (D // 2,)), "q")
    assert bool((clean[0][0] == 0).all()) and bool((clean[1][0, 1] == 0).all()) and bool((clean[2][0, 1] == 0).all())
    q2, k2 = q.clone(), k.clone()
    q2[3, 2, 5], k2[4, 0, 9] = float("inf"), float("nan")
    out = gpu.qkv_norm_rope(q2, k2, k2, pos.cuda(), pro)
    torch.cuda.synchronize()
    for o, c, row in ((out[0], clean[0], (3, 2)), (out[1], clean[1], (4, 0)), (out[2], clean[2], (4, 0))):
        assert not bool(torch.isfinite(o[row]).all())
        o[row] = c[row]
        assert torch.equal(o, c)


def test_parts_in_place_and_v_from_k(gpu):
    """q alone, k and v alone, V taken from K, V left as it is, outputs over their
    own inputs, rows at any 2-byte alignment."""
    import torch

    n, Hq, Hkv, D = 19, 6, 3, 128
    pos = torch.arange(100, 100 + n, dtype=torch.int32, device="cuda")
    pro = prologue(gpu, D, 64)
    q, k, v = rows(1, (n, Hq, D)), rows(2, (n, Hkv, D)), rows(3, (n, Hkv, D))
    oq, ok, ov = gpu.qkv_norm_rope(q, k, v, pos, pro)
    assert torch.equal(gpu.qkv_norm_rope(q, None, None, pos, pro)[0], oq)
    a = gpu.qkv_norm_rope(None, k, v, pos, pro)
    assert a[0] is None and torch.equal(a[1], ok) and torch.equal(a[2], ov)
    a = gpu.qkv_norm_rope(q, k, None, pos, pro)
    assert a[2] is None and torch.equal(a[0], oq) and torch.equal(a[1], ok)
    same = prologue(gpu, D, 64, v_from_k=True)
    a = gpu.qkv_norm_rope(q, k, None, pos, same)
    assert torch.equal(a[0], oq) and torch.equal(a[1], ok)
    check(a[2], reference(k, None, 1e-6), "v from k")
    raw = prologue(gpu, D, 64, v_norm=False)
    assert torch.equal(gpu.qkv_norm_rope(q, k, v, pos, raw)[2], v)
    b = [x.clone() for x in (q, k, v)]
    gpu.qkv_norm_rope(*b, pos, pro, out=b)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(b, (oq, ok, ov)))
    c, vo = k.clone(), torch.empty_like(k)
    gpu.qkv_norm_rope(None, c, None, pos, same, out=(None, c, vo))
    torch.cuda.synchronize()
    assert torch.equal(c, ok) and torch.equal(vo, a[2])
    for shift in (1, 2, 3, 5):
        flat = torch.zeros(q.numel() + 8, dtype=torch.bfloat16, device="cuda")
        d = flat[shift:shift + q.numel()].view(q.shape).copy_(q)
        o = torch.zeros_like(flat)
        r = o[shift:shift + q.numel()].view(q.shape)
        gpu.qkv_norm_rope(d, None, None, pos, pro, out=(r, None, None))
        torch.cuda.synchronize()
        assert torch.equal(r, oq) and bool((o[:shift] == 0).all()) and bool((o[shift + q.numel():] == 0).all())


def test_graph_and_stream(gpu):
    import torch

    n, D = 5, 512
    pro = prologue(gpu, D, 128, sections=(16, 24, 24))
    q, k, v = (rows(s, (n, h, D)) for s, h in ((1, 16), (2, 2), (3, 2)))
    pos = torch.zeros((3, n), dtype=torch.int32, device="cuda")
    out = [torch.empty_like(x) for x in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu.qkv_norm_rope(q, k, v, pos, pro, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.qkv_norm_rope(q, k, v, pos, pro, out=out)
    for i in range(3):
        pos.copy_(torch.arange(3 * n, dtype=torch.int32).view(3, n) * (i + 1))
        q.copy_(rows(50 + i, (n, 16, D)))
        graph.replay()
        want = gpu.qkv_norm_rope(q, k, v, pos, pro)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_rows_feed_the_cache(gpu, ora):
    """One fused projection to the cache and the window: the call's rows appended
    and attended are those of the formulas, in bf16, appended and attended."""
    import torch

    from window_util import check_window, window_reference

    n, Hq, Hkv, D, scale = 70, 16, 8, 256, 256 ** -0.5
    x = rows(5, (n, Hq + 2 * Hkv, D))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    pro = prologue(gpu, D, D)
    q, k, v = gpu.qkv_norm_rope(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], pos, pro)
    pool = gpu.PagedPool(gpu.make_desc(Hkv, D, 4), 6)
    table, zero = torch.arange(5, dtype=torch.int32, device="cuda")[None], torch.zeros(1, dtype=torch.int32, device="cuda")
    out = pool.window_prefill_step(k[None], v[None], table, zero, q[None], 20, 3, scale, dtype=torch.float32)
    torch.cuda.synchronize()
    oc = ora.OracleCache(Hkv, D, 4, 0, n)
    bits = [t.cpu().view(torch.int16).numpy().view(np.uint16) for t in (q, k, v)]
    oc.append(bits[1], bits[2])
    for i in (0, 2, 30, n - 1):
        check_window(out[0, i], window_reference(ora, oc, bits[0][i], i, 20, 3, scale), 6.0, f"row {i}")


@pytest.mark.parametrize("change", [
    dict(eps=0.0), dict(eps=float("inf")), dict(theta=0.5), dict(theta=float("nan")), dict(rope_dims=12),
    dict(rope_dims=136), dict(rope_dims=-8), dict(sections=(10, 10)), dict(sections=(40, -8)),
    dict(v_from_k=True)])
def test_bad_prologues_are_refused(gpu, change):
    import torch

    a = dict(eps=1e-6, rope_dims=64, theta=1e4, sections=None, v_from_k=False)
    a.update(change)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    pro = gpu.make_qkv_prologue(w, w, a["eps"], a["rope_dims"], a["theta"], sections=a["sections"],
                                v_from_k=a["v_from_k"])
    q, k = rows(1, (4, 4, 128)), rows(2, (4, 2, 128))
    pos = torch.zeros((pro.n_axes, 4), dtype=torch.int32, device="cuda")
    out = tuple(torch.full_like(x, 7.0) for x in (q, k, k))
    with pytest.raises(gpu.Exception_):
        gpu.qkv_norm_rope(q, k, k, pos, pro, out=out)
    torch.cuda.synchronize()
    assert all(bool((o == 7.0).all()) for o in out)


def test_bad_arguments_are_refused(gpu):
    import ctypes

    import torch

    lib, bad = gpu.load_library(), gpu.FMKV_ERR_INVALID_ARG
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    pro = gpu.make_qkv_prologue(w, w, 1e-6, 64, 1e4)
    q, k = rows(1, (4, 4, 128)), rows(2, (4, 2, 128))
    qo, ko, vo = torch.empty_like(q), torch.empty_like(k), torch.empty_like(k)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    base = dict(pro=ctypes.byref(pro), D=128, hq=4, hk=2, n=4, q=q.data_ptr(), qs=512, k=k.data_ptr(), ks=256,
                v=None, vs=0, pos=pos.data_ptr(), qo=qo.data_ptr(), ko=ko.data_ptr(), vo=None)

    def call(**change):
        a = {**base, **change}
        return lib.fmkv_qkv_norm_rope(a["pro"], a["D"], a["hq"], a["hk"], a["n"], a["q"], a["qs"], a["k"], a["ks"],
                                      a["v"], a["vs"], a["pos"], a["qo"], a["ko"], a["vo"], None)

    for change in (dict(pro=None), dict(hq=0, hk=0, q=None, k=None), dict(hq=-1), dict(n=-1), dict(n=1 << 31),
                   dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(hq=0), dict(hk=0), dict(qs=511),
                   dict(ks=0), dict(pos=None), dict(qs=(1 << 31) + 1), dict(v=k.data_ptr(), vs=256),
                   dict(qo=q.data_ptr() + 2), dict(qo=q.data_ptr(), qs=520), dict(ko=q.data_ptr()),
                   dict(ko=qo.data_ptr() + 1024), dict(v=vo.data_ptr(), vs=256, vo=ko.data_ptr())):
        assert call(**change) == bad, change
    assert call(D=64) == call(D=96) == gpu.FMKV_ERR_UNSUPPORTED
    assert call(n=0) == gpu.FMKV_OK
    nw = gpu.make_qkv_prologue(None, w, 1e-6, 64, 1e4)
    assert call(pro=ctypes.byref(nw)) == bad
    for f in (lambda: gpu.qkv_norm_rope(q.float(), k, None, pos, pro), lambda: gpu.qkv_norm_rope(q, k[:2], None, pos, pro),
              lambda: gpu.qkv_norm_rope(q.transpose(0, 1), k, None, pos, pro),
              lambda: gpu.qkv_norm_rope(q, k, None, pos.long(), pro), lambda: gpu.qkv_norm_rope(q, k, None, pos[:3], pro),
              lambda: gpu.qkv_norm_rope(None, None, None, pos, pro), lambda: gpu.qkv_norm_rope(q, None, k, pos, pro),
              lambda: gpu.qkv_norm_rope(q, k, None, pos, pro, out=(qo, None, None)),
              lambda: gpu.qkv_norm_rope(q[..., :64].contiguous(), None, None, pos, pro)):
        with pytest.raises(ValueError):
            f()


def test_outputs_over_weights_or_positions_are_refused(gpu):
    """Every row reads them, in no order: refused, and nothing is written."""
    import torch

    D, n = 128, 4
    for which in ("q_norm_weight", "k_norm_weight", "positions", "last weight", "one axis off"):
        flat = torch.ones(4 * n * 4 * D, dtype=torch.bfloat16, device="cuda")
        q, k, v = rows(1, (n, 4, D)), rows(2, (n, 2, D)), rows(3, (n, 2, D))
        w = torch.ones(D, dtype=torch.bfloat16, device="cuda")
        pos = torch.zeros((2, n), dtype=torch.int32, device="cuda")
        out = [torch.zeros_like(x) for x in (q, k, v)]
        qw, kw = w, w
        if which == "q_norm_weight":
            out[0], qw = flat[:n * 4 * D].view(n, 4, D), flat[n * 4 * D - 1:n * 4 * D - 1 + D]
        elif which == "k_norm_weight":
            out[2], kw = flat[:n * 2 * D].view(n, 2, D), flat[:D]
        elif which == "last weight":
            out[0], kw = flat[D - 1:D - 1 + n * 4 * D].view(n, 4, D), flat[:D]
        elif which == "positions":
            out[1], pos = flat[:n * 2 * D].view(n, 2, D), flat[2:2 + 4 * n].view(torch.int32).view(2, n)
        else:  # the second axis's last position
            out[1] = flat[4 * n - 2:4 * n - 2 + n * 2 * D].view(n, 2, D)
            pos = flat[:4 * n].view(torch.int32).view(2, n)
        before = flat.clone()
        pro = gpu.make_qkv_prologue(qw, kw, 1e-6, 64, 1e4, sections=(16, 16))
        with pytest.raises(gpu.Exception_, match="overlaps") as e:
            gpu.qkv_norm_rope(q, k, v, pos, pro, out=tuple(out))
        torch.cuda.synchronize()
        assert e.value.code == gpu.FMKV_ERR_INVALID_ARG and torch.equal(flat, before), which
    # what is not read does not count, and neighbours are not overlaps
    flat = torch.ones(n * 4 * D + 2 * D, dtype=torch.bfloat16, device="cuda")
    pro = gpu.make_qkv_prologue(flat[:D], flat[-D:], 1e-6, 64, 1e4)
    got = flat[D:-D].view(n, 4, D)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    gpu.qkv_norm_rope(q, None, None, pos, pro, out=(got, None, None))
    torch.cuda.synchronize()
    check(got, reference(q, flat[:D], 1e-6, pos, 64, 1e4, (32,)), "q")
    assert bool((flat[:D] == 1).all()) and bool((flat[-D:] == 1).all())
