"""The 8-bit floating point operators on the GPU against their definitions in 64 bits (include/inzg.h).

Tolerances, with u = 2^-24 (half an fp32 step) and e = finfo(type).eps / 2 (one rounding to the type):
* norm: h is one rounding of x + res; the sum of squares adds at most 32 squares per thread and ten shuffles, each
  rounding once, all terms positive: relative 43u, half of that in r; the mean's division, eps, the square root, the
  reciprocal and two products add 6u, h itself 2u (once in the product, once in r): 30u, then e.
* silu: exp(-g) within 6u (2^t good to 2 ulp, the factor that carries the product's error 2u), 1 + exp 1u, the reciprocal 2u,
  two products 1u each; where exp(-g) leaves the normal range (g < -87) or the quotient's divisor passes 2^126 the value may be 0 while
  the true one is below 2^-120 |u|.
* scales: one rounding more than the values' largest; q: half a step of e4m3 at v / s (2^-4 relative, 2^-10 below the
  smallest normal) plus the value's own error, 4u for the scale and its reciprocal.
* products: small integers with power-of-two scales sum exactly in fp32 and have to match bit for bit after the one
  rounding to out_type. Real values: a block of 128 k (or all k for bf16 / f16) adds k numbers in fp32, each addition
  off by at most one step (2u, whether it rounds or truncates) of a running sum no larger than sum |a w|, and the fold
  rounds as * ws, the product-sum and the row scale: (2 k_block + 2 blocks + 4) u sum |a w| as ws, then e.
"""
import numpy as np
import pytest
import torch

from inferenz_b200 import InzgError, MoePool, T_BF16, T_E4M3, T_F16, T_F32, lib
from inferenz_b200.ep import stream_handle

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {T_F32: torch.float32, T_F16: torch.float16, T_BF16: torch.bfloat16, T_E4M3: torch.float8_e4m3fn}
TYPES = [T_F32, T_F16, T_BF16]
F8 = torch.float8_e4m3fn
CANARY = 80.0  # a value that every type here holds


def half_step(dt):
    return torch.finfo(dt).eps / 2


@pytest.fixture(scope="module")
def pool():
    with MoePool(2048, 640, 512, 10, max_tokens=64, n_layers=1, device=0) as p:
        yield p


def _st():
    return stream_handle(torch.cuda.current_stream())


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(n, cols, ld, dt, fill=CANARY, offset=0):
    """A [n][cols] view with pitch ld (and the buffer behind it), `offset` elements into an allocation"""
    buf = torch.full((n * ld + offset + 8,), fill, device="cuda").to(dt)
    return buf[offset:offset + n * ld].view(n, ld)[:, :cols], buf


def _behind_is_untouched(buf, view, offset=0):
    n, cols = view.shape
    b = buf.float().clone()
    if n:
        b[offset:offset + n * view.stride(0)].view(n, view.stride(0))[:, :cols] = CANARY
    assert bool((b == torch.tensor(CANARY).to(buf.dtype).float().item()).all()), "wrote outside its rows"


def _check_quantized(q, s, v, err):
    """q, s against v (64 bits) whose computed form is off by at most err (absolute, per element)"""
    n, cols = v.shape
    nb = (cols + 127) // 128
    pad = lambda t: torch.nn.functional.pad(t, (0, nb * 128 - cols)).view(n, nb, 128)  # noqa: E731
    want = pad(v.abs()).amax(2).clamp(min=2.0 ** -100) / 448
    assert bool(((s.double() - want).abs() <= pad(err).amax(2) / 448 + 2 * U * want).all()), "scales"
    S = s.double().repeat_interleave(128, 1)[:, :cols]
    x = v / S
    slack = err / S + 4 * U * x.abs()
    step = torch.maximum((x.abs() + slack) * 2.0 ** -4, torch.full_like(x, 2.0 ** -10))
    assert bool(((q.double() - x).abs() <= step + slack).all()), "quantized values"


def _norm_want(x, res, w, eps):
    h = x.double() + (res.double() if res is not None else 0)
    return h, h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w.double()


NORM_SHAPES = [(1, 1), (1, 2560), (3, 127), (5, 129), (2, 4096), (7, 10240), (1, 8191), (2, 16385), (1, 32768),
               (333, 640), (600, 2048), (200, 77)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,cols", NORM_SHAPES)
@pytest.mark.parametrize("res,pad,offset", [(True, 0, 0), (False, 3, 1), (True, 8, 8)])
def test_rmsnorm(pool, t, n, cols, res, pad, offset):
    dt, g, ld = DT[t], _gen(n * 7 + cols), cols + pad
    x, _ = _rows(n, cols, ld, dt, offset=offset)
    x.copy_(torch.randn(n, cols, generator=g, device="cuda"))
    r = None
    if res:
        r, _ = _rows(n, cols, ld, dt)
        r.copy_(3 * torch.randn(n, cols, generator=g, device="cuda"))
    w = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
    total, tb = _rows(n, cols, ld, dt)
    y, yb = _rows(n, cols, ld, dt, offset=offset)
    q, qb = _rows(n, cols, ld, F8)
    s, sb = _rows(n, (cols + 127) // 128, (cols + 127) // 128 + 1, torch.float32)
    pool.rmsnorm_q8_device(n, cols, t, x.data_ptr(), w.data_ptr(), 1e-6, ldx=ld, res_ptr=r.data_ptr() if res else None,
                           ldres=ld, sum_ptr=total.data_ptr(), ldsum=ld, y_ptr=y.data_ptr(), ldy=ld, q_ptr=q.data_ptr(),
                           ldq=ld, s_ptr=s.data_ptr(), lds=s.stride(0), stream=_st())
    h, v = _norm_want(x, r, w, 1e-6)
    e = half_step(dt)
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    assert bool(((total.double() - h).abs() <= (e + 2 * U) * h.abs() + tiny).all())
    assert bool(((y.double() - v).abs() <= (e + 30 * U) * v.abs() * (1 + e) + tiny).all())
    _check_quantized(q, s, v, 30 * U * v.abs())
    for buf, view, off in ((tb, total, 0), (yb, y, offset), (qb, q, 0), (sb, s, 0)):
        _behind_is_untouched(buf, view, off)


@pytest.mark.parametrize("cols", [640, 2560])
def test_rmsnorm_in_place_and_optional_outputs(pool, cols):
    """sum over the residual, then over x; each output alone gives what all together give"""
    n, g, t = 5, _gen(1), T_BF16
    x = torch.randn(n, cols, generator=g, device="cuda").bfloat16()
    r = torch.randn(n, cols, generator=g, device="cuda").bfloat16()
    w = torch.ones(cols, device="cuda")
    outs = []
    for place in ("apart", "res", "x"):
        a, b = x.clone(), r.clone()
        total = {"apart": torch.empty_like(a), "res": b, "x": a}[place]
        q, s = torch.empty(n, cols, dtype=F8, device="cuda"), torch.empty(n, cols // 128, device="cuda")
        pool.rmsnorm_q8_device(n, cols, t, a.data_ptr(), w.data_ptr(), 1e-5, res_ptr=b.data_ptr(),
                               sum_ptr=total.data_ptr(), q_ptr=q.data_ptr(), s_ptr=s.data_ptr(), stream=_st())
        outs.append((total, q.view(torch.uint8), s))
    for o in outs[1:]:
        assert all(torch.equal(i, j) for i, j in zip(o, outs[0]))
    y = torch.empty_like(x)
    pool.rmsnorm_q8_device(n, cols, t, x.data_ptr(), w.data_ptr(), 1e-5, res_ptr=r.data_ptr(), y_ptr=y.data_ptr(),
                           stream=_st())
    _, v = _norm_want(x, r, w, 1e-5)
    assert bool(((y.double() - v).abs() <= (half_step(y.dtype) + 30 * U) * v.abs() * 1.01).all())


def test_quantizer_edges(pool):
    """all-zero rows and blocks, values at both ends of the range, infinities and NaN (inzg_rmsnorm_q8 with w only)"""
    n, cols = 6, 300
    x = torch.zeros(n, cols, device="cuda")
    x[1, 5] = 1.0
    x[2] = 1e-20 * torch.arange(1, cols + 1, device="cuda")
    x[3, 0], x[3, 200] = float("inf"), 1.0
    x[4, 7], x[4, 1] = float("nan"), 2.0
    x[5] = 1e18
    w = torch.ones(cols, device="cuda")
    y, q = torch.empty_like(x), torch.empty(n, cols, dtype=F8, device="cuda")
    s = torch.empty(n, 3, device="cuda")
    pool.rmsnorm_q8_device(n, cols, T_F32, x.data_ptr(), w.data_ptr(), 1e-6, y_ptr=y.data_ptr(), q_ptr=q.data_ptr(),
                           s_ptr=s.data_ptr(), stream=_st())
    floor = float(np.float32(2.0 ** -100) / np.float32(448))
    back = q.float() * s.repeat_interleave(128, 1)[:, :cols]
    assert bool((q[0].float() == 0).all()) and bool((s[0] == floor).all())
    assert s[1, 1] == floor and q[1, 5].float() == 448 and bool((q[1, 128:].float() == 0).all())
    _, v = _norm_want(x[[1, 2, 5]], None, w, 1e-6)
    assert bool(((y[[1, 2, 5]].double() - v).abs() <= 31 * U * v.abs()).all())
    _check_quantized(q[[1, 2, 5]], s[[1, 2, 5]], v, 30 * U * v.abs())
    assert bool(torch.isnan(back[3, 0])) and bool((back[3, 1:] == 0).all())  # inf * 0 in its place, 1 / inf elsewhere
    assert bool(torch.isnan(back[4]).any())  # a NaN takes its row's norm with it


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,cols", [(1, 1), (1, 640), (320, 640), (3, 127), (5, 129), (2, 4096), (1000, 33), (4097, 640)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1), (8, 8)])
def test_silu_mul(pool, t, n, cols, pad, offset):
    dt, g = DT[t], _gen(n + cols)
    ldx, ld = 2 * cols + pad, cols + pad
    x, _ = _rows(n, 2 * cols, ldx, dt, offset=offset)
    x.copy_(4 * torch.randn(n, 2 * cols, generator=g, device="cuda"))
    y, yb = _rows(n, cols, ld, dt)
    q, qb = _rows(n, cols, ld, F8)
    s, sb = _rows(n, (cols + 127) // 128, (cols + 127) // 128 + 2, torch.float32)
    pool.silu_mul_q8_device(n, cols, t, x.data_ptr(), ldx=ldx, y_ptr=y.data_ptr(), ldy=ld, q_ptr=q.data_ptr(), ldq=ld,
                            s_ptr=s.data_ptr(), lds=s.stride(0), stream=_st())
    gate, up = x[:, :cols].double(), x[:, cols:].double()
    v = gate * torch.sigmoid(gate) * up
    e, tiny = half_step(dt), torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    assert bool(((y.double() - v).abs() <= (e + 12 * U) * v.abs() * 1.01 + tiny).all())
    _check_quantized(q, s, v, 12 * U * v.abs())
    for buf, view in ((yb, y), (qb, q), (sb, s)):
        _behind_is_untouched(buf, view)


def test_silu_more_rows_than_one_launch_counts(pool):
    """narrow rows: 2^26 and a few, counted in two launches"""
    n = (1 << 26) + 5
    x = torch.randn(n, 2, generator=_gen(8), device="cuda", dtype=torch.bfloat16)
    y = torch.full((n, 1), CANARY, device="cuda", dtype=torch.bfloat16)
    pool.silu_mul_q8_device(n, 1, T_BF16, x.data_ptr(), y_ptr=y.data_ptr(), stream=_st())
    for at in (slice(0, 1000), slice(n // 2, n // 2 + 1000), slice(n - 1000, n)):
        g, u = x[at, 0].double(), x[at, 1].double()
        v = g * torch.sigmoid(g) * u
        assert bool(((y[at, 0].double() - v).abs() <= (half_step(y.dtype) + 12 * U) * v.abs() * 1.01 + 1e-38).all())


def test_silu_extremes(pool):
    """gates far out on both sides, infinities and NaN"""
    inf, nan = float("inf"), float("nan")
    gate = torch.tensor([0.0, -0.0, 20.0, -20.0, 80.0, -80.0, -86.0, -100.0, 100.0, -1e30, 1e30, inf, -inf, nan, 1.0, 1.0],
                        device="cuda")
    up = torch.tensor([1.0] * 14 + [inf, nan], device="cuda")
    x = torch.cat([gate, up])[None].contiguous()
    y = torch.empty(1, 16, device="cuda")
    pool.silu_mul_q8_device(1, 16, T_F32, x.data_ptr(), y_ptr=y.data_ptr(), stream=_st())
    want = gate.double() * torch.sigmoid(gate.double()) * up.double()
    y = y[0].double()
    fine = torch.isfinite(want)
    assert bool(((y - want).abs()[fine] <= (12 * U * want.abs() + 2.0 ** -120)[fine]).all())
    assert y[11] == inf and bool(torch.isnan(y[12])) and bool(torch.isnan(y[13])) and y[14] == inf and bool(torch.isnan(y[15]))


# ---------------------------------------------------------------------------------------------------------------------


def _lists_want(sel, E):
    flat = sel.reshape(-1).cpu().numpy().astype(np.int64)
    key = np.where((flat < 0) | (flat >= E), E, flat)
    order = np.argsort(key, kind="stable")
    order = order[key[order] < E]
    return np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])]), order


def _lists(pool, sel, E, w=None, offset=0):
    n, K = sel.shape
    buf = torch.empty(n * K + 4, dtype=torch.int32, device="cuda")
    buf[offset:offset + n * K] = sel.reshape(-1)
    off = torch.full((E + 1,), -5, dtype=torch.int32, device="cuda")
    rows, slots = (torch.full((n * K,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    wo = torch.full((n * K,), -7.0, device="cuda") if w is not None else None
    pool.expert_lists_device(n, K, E, buf.data_ptr() + 4 * offset, off.data_ptr(), rows.data_ptr(), slots.data_ptr(),
                             w_ptr=w.data_ptr() if w is not None else None,
                             w_out_ptr=wo.data_ptr() if w is not None else None, stream=_st())
    return off, rows, slots, wo


@pytest.mark.parametrize("n,K,E", [(1, 1, 1), (1, 10, 512), (2, 10, 512), (32, 10, 512), (13, 7, 33), (333, 10, 64),
                                   (4096, 10, 512), (1000, 16, 2048), (257, 1, 3), (5, 16, 16)])
@pytest.mark.parametrize("absent,offset", [(False, 0), (True, 1)])
def test_expert_lists(pool, n, K, E, absent, offset):
    g = _gen(n + E)
    sel = torch.rand(n, E, generator=g, device="cuda").argsort(1)[:, :K].to(torch.int32)
    if absent:
        sel = torch.where(torch.rand(n, K, generator=g, device="cuda") < 0.4, -1 - sel, sel)
    w = torch.rand(n, K, generator=g, device="cuda")
    off, rows, slots, wo = _lists(pool, sel, E, w, offset)
    want_off, order = _lists_want(sel, E)
    m = len(order)
    assert np.array_equal(off.cpu().numpy(), want_off)
    assert np.array_equal(slots.cpu().numpy()[:m], order) and np.array_equal(rows.cpu().numpy()[:m], order // K)
    assert torch.equal(wo[:m], w.reshape(-1)[slots[:m].long()])
    assert bool((rows[m:] == -7).all()) and bool((slots[m:] == -7).all()) and bool((wo[m:] == -7).all())
    pool.device_status(_st())


def test_expert_lists_of_one_expert_and_no_tokens(pool):
    sel = torch.full((500, 3), 5, dtype=torch.int32, device="cuda")  # one expert named three times by each token
    off, rows, slots, _ = _lists(pool, sel, 8)
    assert off.tolist() == [0] * 6 + [1500] * 3 and torch.equal(slots, torch.arange(1500, dtype=torch.int32, device="cuda"))
    off.fill_(9)
    pool.expert_lists_device(0, 3, 8, None, off.data_ptr(), None, None, stream=_st())
    assert off.tolist() == [0] * 9


@pytest.mark.parametrize("n,K,E,kind", [(20_000, 10, 512, "random"), (3001, 3, 512, "one"), (2049, 1, 7, "two"), (700, 3, 9, "none"),
                                        (4096, 8, 2048, "runs")])
def test_expert_lists_long_and_skewed(pool, n, K, E, kind):
    """past one block's entries: many of them, all of one expert, of two in turn, none on this rank, long runs"""
    i = torch.arange(n * K, device="cuda")
    sel = {"random": torch.randint(0, E, (n * K,), generator=_gen(4), device="cuda"), "one": torch.full_like(i, E - 1),
           "two": (i % 2) * (E - 1), "none": torch.full_like(i, -1), "runs": i * E // (n * K)}[kind].to(torch.int32).view(n, K)
    w = torch.rand(n, K, generator=_gen(5), device="cuda")
    off, rows, slots, wo = _lists(pool, sel, E, w)
    want_off, order = _lists_want(sel, E)
    m = len(order)
    assert np.array_equal(off.cpu().numpy(), want_off) and np.array_equal(slots.cpu().numpy()[:m], order)
    assert np.array_equal(rows.cpu().numpy()[:m], order // K) and torch.equal(wo[:m], w.reshape(-1)[slots[:m].long()])
    assert bool((slots[m:] == -7).all())
    pool.device_status(_st())


def test_expert_lists_report_a_bad_expert_once(pool):
    sel = torch.tensor([[0, 4], [2, 1]], dtype=torch.int32, device="cuda")
    off, rows, slots, _ = _lists(pool, sel, 4)
    assert off.tolist() == [0, 1, 2, 3, 3] and slots.tolist() == [0, 3, 2, -7]
    with pytest.raises(InzgError) as e:
        pool.device_status(_st())
    assert e.value.status == 7 and "expert id" in str(e.value)
    pool.device_status(_st())


# ---------------------------------------------------------------------------------------------------------------------


def _ints(n, k, ld, dt, g, lo=-2, hi=2):
    """rows of small integers; NaN behind each row, which no product may see"""
    buf = torch.full((n, ld), float("nan"), device="cuda")
    buf[:, :k] = torch.randint(lo, hi + 1, (n, k), generator=g, device="cuda").float()
    return buf.to(dt)[:, :k]


def _up(v, to):
    return -(-v // to) * to


def _pow2(shape, g):
    return torch.exp2(torch.randint(-2, 3, shape, generator=g, device="cuda").float())


def _deq(a, s):
    return a.double() * s.double().repeat_interleave(128, 1)[:, :a.shape[1]]


def _deq_w(w, ws, n):
    """w [E * n][k], ws [E][nb][kb] -> [E][n][k] in 64 bits"""
    E = ws.shape[0]
    s = ws.repeat_interleave(128, 1)[:, :n].reshape(E * n, -1)
    return _deq(w, s).view(E, n, -1)


def _product_bound(absprod, k, f8, exact, dt):
    kb = min(k, 128) if f8 else k
    blocks = (k + 127) // 128 if f8 else 1
    acc = (2 * kb + 2 * blocks + 4) * U * absprod
    return acc + half_step(dt) * (exact.abs() + acc) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


MATMUL = [(1, 1, 1), (1, 640, 2560), (2, 127, 16), (3, 128, 64), (15, 129, 127), (16, 130, 128), (17, 257, 129),
          (33, 16, 640), (63, 64, 1040), (64, 128, 2048), (65, 300, 256), (96, 129, 1000), (127, 128, 1153), (128, 384, 512),
          (129, 1, 300), (300, 260, 2064), (1000, 70, 96), (5, 2000, 48), (257, 1300, 700),
          (9700, 70, 96), (1000, 1300, 700), (257, 5000, 300), (129, 8000, 1153), (2500, 512, 2064)]  # more tiles than two per SM


@pytest.mark.parametrize("m,n,k", MATMUL)
@pytest.mark.parametrize("out", TYPES)
def test_matmul_exact(pool, m, n, k, out):
    g = _gen(m * 3 + n * 5 + k)
    kb, pad = (k + 127) // 128, 16 * (m % 3)
    a, w = _ints(m, k, _up(k, 16) + pad, F8, g), _ints(n, k, _up(k, 16), F8, g)
    sa, sw = _rows(m, kb, kb + m % 2, torch.float32)[0], _pow2(((n + 127) // 128, kb), g)
    sa.copy_(_pow2((m, kb), g))
    o, ob = _rows(m, n, n + m % 4, DT[out])
    pool.matmul_q8_device(m, n, k, a.data_ptr(), sa.data_ptr(), w.data_ptr(), sw.data_ptr(), o.data_ptr(), out,
                          lda=a.stride(0), lda_scale=sa.stride(0), ldw=w.stride(0), ldo=o.stride(0), stream=_st())
    want = _deq(a, sa) @ _deq_w(w, sw[None], n)[0].t()  # multiples of 2^-4 below 2^24 * 2^-4: exact in fp32 in any order
    assert float(want.abs().max()) < 2.0 ** 20
    assert torch.equal(o.double(), want.to(DT[out]).double())
    _behind_is_untouched(ob, o)
    pool.device_status(_st())


@pytest.mark.parametrize("m,n,k,out", [(1, 1280, 2560, T_BF16), (77, 300, 1111, T_F32), (400, 640, 2048, T_F16),
                                       (130, 2560, 640, T_F32), (1000, 1300, 2048, T_BF16)])
def test_matmul_real(pool, m, n, k, out):
    g, kb = _gen(m), (k + 127) // 128
    fp8 = lambda r: (torch.randn(r, _up(k, 16), generator=g, device="cuda") * 120).clamp(-448, 448).to(F8)[:, :k]  # noqa: E731
    a, w = fp8(m), fp8(n)
    sa = 0.01 * torch.exp(torch.randn(m, kb, generator=g, device="cuda"))
    sw = 0.01 * torch.rand((n + 127) // 128, kb, generator=g, device="cuda")
    o = torch.empty(m, n, dtype=DT[out], device="cuda")
    pool.matmul_q8_device(m, n, k, a.data_ptr(), sa.data_ptr(), w.data_ptr(), sw.data_ptr(), o.data_ptr(), out,
                          lda=a.stride(0), ldw=w.stride(0), stream=_st())
    A, W = _deq(a, sa), _deq_w(w, sw[None], n)[0]
    want, mag = A @ W.t(), A.abs() @ W.abs().t()
    assert bool(((o.double() - want).abs() <= _product_bound(mag, k, True, want, DT[out])).all())


def test_matmul_nan_and_zero_rows(pool):
    """a NaN row gives NaN and touches no other row; zero scales give zeros; no rows are no work"""
    g = _gen(9)
    a, w = _ints(40, 256, 256, F8, g), _ints(130, 256, 256, F8, g)
    a = a.float()
    a[3, 200] = float("nan")
    a = a.to(F8)
    sa, sw = torch.ones(40, 2, device="cuda"), torch.ones(2, 2, device="cuda")
    sa[5] = 0
    o = torch.full((40, 130), CANARY, device="cuda")
    pool.matmul_q8_device(40, 130, 256, a.data_ptr(), sa.data_ptr(), w.data_ptr(), sw.data_ptr(), o.data_ptr(), T_F32, stream=_st())
    want = a.double() @ w.double().t()
    rest = [i for i in range(40) if i not in (3, 5)]
    assert bool(torch.isnan(o[3]).all()) and bool((o[5] == 0).all()) and torch.equal(o[rest].double(), want[rest])
    pool.matmul_q8_device(0, 130, 256, None, None, None, None, None, T_F32, stream=_st())


# ---------------------------------------------------------------------------------------------------------------------


def _group_sizes(E, total, g, empty):
    """sizes of E groups that sum to total, some of them empty"""
    p = torch.rand(E, generator=g, device="cuda").pow(3)
    if empty and E > 1:
        p[torch.rand(E, generator=g, device="cuda") < 0.4] = 0
        p[int(torch.randint(0, E, (1,), generator=g, device="cuda"))] = 1
    sizes = torch.bincount(torch.multinomial(p, total, replacement=True, generator=g), minlength=E)
    return torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), sizes.cumsum(0)]).to(torch.int32)


def _grouped_case(t, E, entries, n, k, gather, scatter, seed, ints=True, first=0):
    g, dt, f8 = _gen(seed), DT[t], t == T_E4M3
    kb, a_rows, out_rows_n = (k + 127) // 128, max(1, entries // 3) if gather else entries, entries + 5 if scatter else entries
    ld = _up(k, 16)
    mk = _ints if ints else (lambda r, k, ld, dt, g: (torch.randn(r, ld, generator=g, device="cuda")).to(dt)[:, :k])
    c = {"a": mk(a_rows, k, ld, dt, g), "w": mk(E * n, k, ld, dt, g), "out_rows_n": out_rows_n,
         "off": _group_sizes(E, entries - first, g, True) + first}
    scale = (lambda *s: _pow2(s, g)) if ints else (lambda *s: torch.rand(*s, generator=g, device="cuda") + 0.1)
    c["as"], c["ws"] = (scale(a_rows, kb), scale(E, (n + 127) // 128, kb)) if f8 else (None, None)
    c["in"] = torch.randint(0, a_rows, (entries,), generator=g, device="cuda").to(torch.int32) if gather else None
    c["to"] = torch.randperm(out_rows_n, generator=g, device="cuda")[:entries].to(torch.int32) if scatter else None
    c["sc"] = scale(entries) if scatter else None
    return c


def _run_grouped(pool, t, c, E, entries, n, k, out, stream=None):
    ld = n + 3
    o, ob = _rows(c["out_rows_n"], n, ld, DT[out])
    p = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
    pool.grouped_matmul_device(t, E, n, k, c["a"].shape[0], entries, p(c["a"]), p(c["w"]), p(c["off"]), p(o), out,
                               lda=c["a"].stride(0), ldw=c["w"].stride(0), ldo=ld, a_scale_ptr=p(c["as"]), w_scale_ptr=p(c["ws"]),
                               in_rows_ptr=p(c["in"]), out_rows_ptr=p(c["to"]), out_scale_ptr=p(c["sc"]),
                               out_rows_n=c["out_rows_n"], stream=stream or _st())
    return o, ob


def _grouped_want(c, E, entries, n):
    """(exact, magnitude, written) in 64 bits"""
    A = _deq(c["a"], c["as"]) if c["as"] is not None else c["a"].double()
    W = _deq_w(c["w"], c["ws"], n) if c["ws"] is not None else c["w"].double().view(E, n, -1)
    off = c["off"].tolist()
    want, mag = (torch.full((c["out_rows_n"], n), CANARY, dtype=torch.float64, device="cuda") for _ in range(2))
    wrote = torch.zeros(c["out_rows_n"], dtype=torch.bool, device="cuda")
    for e in range(E):
        i = torch.arange(off[e], off[e + 1], device="cuda")
        if len(i) == 0:
            continue
        x = A[c["in"][i].long() if c["in"] is not None else i]
        to = c["to"][i].long() if c["to"] is not None else i
        sc = c["sc"][i].double()[:, None] if c["sc"] is not None else 1.0
        want[to], mag[to], wrote[to] = x @ W[e].t() * sc, x.abs() @ W[e].abs().t() * sc, True
    return want, mag, wrote


GROUPED = [(1, 1, 128, 128), (1, 200, 130, 160), (4, 3, 64, 1), (8, 40, 256, 640), (16, 10, 1280, 2048), (5, 333, 127, 129),
           (64, 500, 129, 320), (512, 320, 128, 256), (2, 700, 260, 96), (2048, 100, 16, 32), (3, 129, 1, 2048),
           (1, 10_300, 127, 129), (16, 9000, 130, 2064), (100, 7000, 260, 300), (3, 1700, 1300, 520), (2, 640, 2000, 20_011)]


@pytest.mark.parametrize("E,entries,n,k", GROUPED)
@pytest.mark.parametrize("t,out,gather,scatter", [(T_E4M3, T_F32, True, True), (T_E4M3, T_BF16, False, False),
                                                  (T_BF16, T_F16, True, False), (T_F16, T_F32, False, True)])
def test_grouped_exact(pool, E, entries, n, k, t, out, gather, scatter):
    c = _grouped_case(t, E, entries, n, k, gather, scatter, E * 11 + entries)
    o, ob = _run_grouped(pool, t, c, E, entries, n, k, out)
    want, _, wrote = _grouped_want(c, E, entries, n)
    assert float(want.abs().max()) < 2.0 ** 20
    assert torch.equal(o.double(), torch.where(wrote[:, None], want, torch.tensor(CANARY, dtype=torch.float64, device="cuda"))
                       .to(DT[out]).double())
    _behind_is_untouched(ob, o)
    pool.device_status(_st())


@pytest.mark.parametrize("t", [T_E4M3, T_BF16, T_F16])
@pytest.mark.parametrize("E,entries,n,k,out", [(16, 10, 1280, 2048, T_F32), (6, 450, 640, 1100, T_BF16), (3, 700, 200, 520, T_F32),
                                             (100, 7000, 260, 1100, T_BF16)])
def test_grouped_real(pool, t, E, entries, n, k, out):
    c = _grouped_case(t, E, entries, n, k, True, True, 5 + E, ints=False)
    o, _ = _run_grouped(pool, t, c, E, entries, n, k, out)
    want, mag, wrote = _grouped_want(c, E, entries, n)
    bound = _product_bound(mag, k, t == T_E4M3, want, DT[out])
    assert bool(((o.double() - want).abs() <= bound)[wrote].all())


@pytest.mark.parametrize("t,entries,n,k", [(T_E4M3, 2048 * 52, 9600, 16), (T_E4M3, 2048, 12_000, 16), (T_F16, 2048, 12_000, 8)])
def test_grouped_many_items(pool, t, entries, n, k):
    """more items per SM than the list that each CTA keeps of them (2048 groups x n / 256 or n / 128 row blocks over 148 SMs)"""
    E, g = 2048, _gen(3)
    off = torch.arange(E + 1, device="cuda", dtype=torch.int64) * entries // E
    a, w = _ints(entries, k, 16, DT[t], g), _ints(E * n, k, 16, DT[t], g)
    f8 = t == T_E4M3
    sa, sw = (_pow2((entries, 1), g), _pow2((E, (n + 127) // 128, 1), g)) if f8 else (None, None)
    o = torch.full((entries, n), CANARY, device="cuda", dtype=torch.bfloat16)
    p = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
    off32 = off.to(torch.int32)
    pool.grouped_matmul_device(t, E, n, k, entries, entries, p(a), p(w), p(off32), p(o), T_BF16, lda=16, ldw=16, a_scale_ptr=p(sa),
                               w_scale_ptr=p(sw), stream=_st())
    pool.device_status(_st())
    cols = torch.randint(0, n, (40,), generator=g, device="cuda")
    group = torch.searchsorted(off[1:], torch.arange(entries, device="cuda"), right=True)
    for c in torch.cat([cols, torch.tensor([0, n - 1], device="cuda")]).tolist():
        want = (a.float() * w.view(torch.uint8).view(E, n, -1)[:, c].contiguous().view(w.dtype).float()[group]).sum(1) if f8 else \
            (a.float() * w.unflatten(0, (E, n))[:, c].float()[group]).sum(1)
        if f8:
            want = want * sa[:, 0] * sw[group, c // 128, 0]
        assert torch.equal(o[:, c], want.to(torch.bfloat16))


@pytest.mark.parametrize("t,m,k", [(T_E4M3, 5, 20_011), (T_E4M3, 300, 20_011), (T_BF16, 5, 10_003), (T_BF16, 300, 10_003)])
def test_grouped_long_rows(pool, t, m, k):
    """157 blocks of k: the rings and the staged scales go round many times"""
    c = _grouped_case(t, 2, m, 200, k, True, True, m)
    o, _ = _run_grouped(pool, t, c, 2, m, 200, k, T_F32)
    want, _, wrote = _grouped_want(c, 2, m, 200)
    assert float(want.abs().max()) < 2.0 ** 20 and torch.equal(o.double()[wrote], want[wrote])


@pytest.mark.parametrize("t", [T_E4M3, T_BF16])
def test_grouped_lists_inside_the_entries(pool, t):
    """offsets that begin after 0 and end before `entries`: what they leave out stays as it was"""
    E, entries, n, k = 6, 150, 140, 256
    c = _grouped_case(t, E, entries, n, k, False, False, 3, first=40)
    c["off"] = torch.where(c["off"] > 120, 120, c["off"]).to(torch.int32)
    o, _ = _run_grouped(pool, t, c, E, entries, n, k, T_F32)
    want, _, wrote = _grouped_want(c, E, entries, n)
    assert not bool(wrote[:40].any()) and not bool(wrote[120:].any()) and torch.equal(o.double(), want)


@pytest.mark.parametrize("break_it,word", [("descending", "offsets"), ("past", "offsets"), ("negative", "offsets"),
                                           ("in", "row index"), ("in_negative", "row index"), ("to", "row index")])
def test_grouped_checks_on_the_device(pool, break_it, word):
    """bad offsets: nothing is written; a bad row index: that entry alone is skipped. Reported once."""
    E, entries, n, k = 4, 90, 130, 256
    c = _grouped_case(T_E4M3, E, entries, n, k, True, True, 17)
    c["off"] = torch.tensor([0, 30, 30, 70, 90], dtype=torch.int32, device="cuda")
    good = {k_: v.clone() if torch.is_tensor(v) else v for k_, v in c.items()}
    bad_entry = None
    if break_it == "descending":
        c["off"][2] = 20
    elif break_it == "past":
        c["off"][4] = 91
    elif break_it == "negative":
        c["off"][0] = -1
    elif break_it == "to":
        bad_entry, c["to"][33] = 33, c["out_rows_n"]
    else:
        bad_entry, c["in"][33] = 33, c["a"].shape[0] if break_it == "in" else -1
    o, _ = _run_grouped(pool, T_E4M3, c, E, entries, n, k, T_F32)
    with pytest.raises(InzgError) as e:
        pool.device_status(_st())
    assert e.value.status == 7 and word in str(e.value)
    want, _, _ = _grouped_want(good, E, entries, n)
    if bad_entry is None:
        assert bool((o == CANARY).all())
    else:
        want[good["to"][bad_entry].long()] = CANARY
        assert torch.equal(o.double(), want)
    pool.device_status(_st())


@pytest.mark.parametrize("t", [T_E4M3, T_BF16])
def test_many_entries_checked_partial_and_replayed(pool, t):
    """the tiles of many entries: bad offsets and indexes, lists that leave entries out, no listed entries, NaN in one row, a
    replay on new contents"""
    E, entries, n, k = 100, 7000, 400, 256
    base = _grouped_case(t, E, entries, n, k, True, True, 41)
    base["off"] = (torch.arange(E + 1, device="cuda") * entries // E).to(torch.int32)

    def case():
        return {k_: v.clone() if torch.is_tensor(v) else v for k_, v in base.items()}

    def same(o, want):
        assert torch.equal(o.double(), want)

    def reported(word):
        with pytest.raises(InzgError) as e:
            pool.device_status(_st())
        assert e.value.status == 7 and word in str(e.value)

    good = _grouped_want(base, E, entries, n)[0]
    c = case()
    c["off"][57] = 3
    o, _ = _run_grouped(pool, t, c, E, entries, n, k, T_F32)
    reported("offsets")
    assert bool((o == CANARY).all())
    for bad in ("in", "to"):
        c = case()
        c[bad][333] = c["a"].shape[0] if bad == "in" else -1
        o, _ = _run_grouped(pool, t, c, E, entries, n, k, T_F32)
        reported("row index")
        want = good.clone()
        want[base["to"][333].long()] = CANARY
        same(o, want)
    c = case()
    c["off"] = c["off"].clamp(205, 6800).to(torch.int32)
    o, _ = _run_grouped(pool, t, c, E, entries, n, k, T_F32)
    same(o, _grouped_want(c, E, entries, n)[0])
    c["off"].fill_(entries)
    o, _ = _run_grouped(pool, t, c, E, entries, n, k, T_F32)
    assert bool((o == CANARY).all())
    c = case()
    a = c["a"].float()
    a[7, 100] = float("nan")
    c["a"].copy_(a.to(DT[t]))
    o, _ = _run_grouped(pool, t, c, E, entries, n, k, T_F32)
    hit = base["to"][base["in"] == 7].long()
    rest = torch.ones(len(good), dtype=torch.bool, device="cuda")
    rest[hit] = False
    assert bool(torch.isnan(o[hit]).all()) and torch.equal(o[rest].double(), good[rest])
    pool.device_status(_st())

    c, o = case(), torch.full_like(good, CANARY, dtype=torch.float32)
    p = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.grouped_matmul_device(t, E, n, k, c["a"].shape[0], entries, p(c["a"]), p(c["w"]), p(c["off"]), p(o), T_F32,
                                   lda=c["a"].stride(0), ldw=c["w"].stride(0), a_scale_ptr=p(c["as"]), w_scale_ptr=p(c["ws"]),
                                   in_rows_ptr=p(c["in"]), out_rows_ptr=p(c["to"]), out_scale_ptr=p(c["sc"]),
                                   out_rows_n=c["out_rows_n"], stream=torch.cuda.current_stream().cuda_stream)
    c["off"].copy_(_group_sizes(E, entries, _gen(8), True))
    c["in"].copy_(c["in"].flip(0))
    graph.replay()
    torch.cuda.synchronize()
    same(o, _grouped_want(c, E, entries, n)[0])
    pool.device_status(_st())


# ---------------------------------------------------------------------------------------------------------------------


def test_refusals_reach_the_caller_and_leave_the_device(pool):
    x = torch.zeros(4, 100, dtype=F8, device="cuda")
    s = torch.ones(4, 1, device="cuda")
    o = torch.full((4, 4), CANARY, device="cuda")
    with pytest.raises(InzgError) as e:
        pool.matmul_q8_device(4, 4, 100, x.data_ptr(), s.data_ptr(), x.data_ptr(), s.data_ptr(), o.data_ptr(), T_F32, stream=_st())
    assert e.value.status == 1 and "multiples of 16 bytes" in str(e.value)
    assert bool((o == CANARY).all()) and torch.cuda.current_device() == 0


def test_streams_and_graph(pool):
    """two calls at once on two streams, then both captured into a graph and replayed on new inputs"""
    E, entries, n, k = 8, 200, 260, 384
    cs = [_grouped_case(T_E4M3, E, entries, n, k, True, True, 100 + i) for i in range(2)]
    outs = [torch.empty(c["out_rows_n"], n, device="cuda") for c in cs]
    p = lambda x: x.data_ptr()  # noqa: E731

    def call(c, o, st):
        pool.grouped_matmul_device(T_E4M3, E, n, k, c["a"].shape[0], entries, p(c["a"]), p(c["w"]), p(c["off"]), p(o), T_F32,
                                   lda=c["a"].stride(0), ldw=c["w"].stride(0), a_scale_ptr=p(c["as"]), w_scale_ptr=p(c["ws"]),
                                   in_rows_ptr=p(c["in"]), out_rows_ptr=p(c["to"]), out_scale_ptr=p(c["sc"]),
                                   out_rows_n=c["out_rows_n"], stream=st)

    def check():
        for c, o in zip(cs, outs):
            want, _, wrote = _grouped_want(c, E, entries, n)
            assert torch.equal(o.double()[wrote], want[wrote])

    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, o, s in zip(cs, outs, streams):
            call(c, o, s.cuda_stream)
    torch.cuda.synchronize()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        for c, o in zip(cs, outs):
            call(c, o, st)
    for c, o in zip(cs, outs):  # other inputs in the same buffers: the replay reads them
        g = _gen(7)
        c["w"].copy_(torch.randint(-2, 3, c["w"].shape, generator=g, device="cuda").float().to(F8))
        c["off"].copy_(_group_sizes(E, entries, g, True))
        o.fill_(0)
    graph.replay()
    torch.cuda.synchronize()
    check()
    pool.device_status(_st())


@pytest.mark.parametrize("t", [T_E4M3, T_BF16])
@pytest.mark.parametrize("entries", [7, 600])
def test_grouped_with_no_listed_entries(pool, t, entries):
    c = _grouped_case(t, 9, entries, 140, 256, True, True, 2)
    c["off"].fill_(3)
    o, _ = _run_grouped(pool, t, c, 9, entries, 140, 256, T_F32)
    pool.device_status(_st())
    assert bool((o == CANARY).all())


def test_grouped_scale_pitch_and_repeated_rows(pool):
    """scales with a pitch of their own; every entry of one group reads the same row of a"""
    for entries in (20, 400):
        E, n, k, g = 2, 200, 600, _gen(entries)
        c = _grouped_case(T_E4M3, E, entries, n, k, True, False, 31)
        c["in"].fill_(c["a"].shape[0] - 1)
        wide = torch.full((c["a"].shape[0], 9), float("nan"), device="cuda")
        wide[:, :5] = c["as"]
        o = torch.empty(entries, n, device="cuda")
        p = lambda x: x.data_ptr()  # noqa: E731
        pool.grouped_matmul_device(T_E4M3, E, n, k, c["a"].shape[0], entries, p(c["a"]), p(c["w"]), p(c["off"]), p(o), T_F32,
                                   lda=c["a"].stride(0), ldw=c["w"].stride(0), a_scale_ptr=p(wide), lda_scale=9,
                                   w_scale_ptr=p(c["ws"]), in_rows_ptr=p(c["in"]), stream=_st())
        want, _, wrote = _grouped_want(c, E, entries, n)
        assert bool(wrote.all()) and torch.equal(o.double(), want)


def test_every_operator_captured_and_replayed(pool):
    """norm -> lists -> gate|up -> SiLU * up -> down in one graph; the replay on new contents of the same buffers gives what calls on
    them give"""
    n, H, FF, E, K, g = 300, 512, 256, 16, 4, _gen(12)
    dt = torch.bfloat16
    p = lambda x: x.data_ptr()  # noqa: E731
    f8 = lambda r, k: (torch.randn(r, k, generator=g, device="cuda") * 120).clamp(-448, 448).to(F8)  # noqa: E731
    x, res, w = torch.empty(n, H, dtype=dt, device="cuda"), torch.empty(n, H, dtype=dt, device="cuda"), torch.ones(H, device="cuda")
    wg, wd = f8(E * 2 * FF, H), f8(E * H, FF)
    sg, sd = torch.rand(E, 4, 4, generator=g, device="cuda") / 3000, torch.rand(E, 4, 2, generator=g, device="cuda") / 3000
    sel, rw = torch.empty(n, K, dtype=torch.int32, device="cuda"), torch.rand(n, K, generator=g, device="cuda")
    total, q, s = torch.empty_like(x), torch.empty(n, H, dtype=F8, device="cuda"), torch.empty(n, 4, device="cuda")
    off, rows, slots = (torch.empty(m, dtype=torch.int32, device="cuda") for m in (E + 1, n * K, n * K))
    lw, gu = torch.empty(n * K, device="cuda"), torch.empty(n * K, 2 * FF, dtype=dt, device="cuda")
    hq, hs, out = torch.empty(n * K, FF, dtype=F8, device="cuda"), torch.empty(n * K, 2, device="cuda"), torch.empty(n * K, H, device="cuda")

    def layer(st):
        pool.rmsnorm_q8_device(n, H, T_BF16, p(x), p(w), 1e-6, res_ptr=p(res), sum_ptr=p(total), q_ptr=p(q), s_ptr=p(s), stream=st)
        pool.expert_lists_device(n, K, E, p(sel), p(off), p(rows), p(slots), w_ptr=p(rw), w_out_ptr=p(lw), stream=st)
        pool.grouped_matmul_device(T_E4M3, E, 2 * FF, H, n, n * K, p(q), p(wg), p(off), p(gu), T_BF16, a_scale_ptr=p(s),
                                   w_scale_ptr=p(sg), in_rows_ptr=p(rows), stream=st)
        pool.silu_mul_q8_device(n * K, FF, T_BF16, p(gu), q_ptr=p(hq), s_ptr=p(hs), stream=st)
        pool.grouped_matmul_device(T_E4M3, E, H, FF, n * K, n * K, p(hq), p(wd), p(off), p(out), T_F32, a_scale_ptr=p(hs),
                                   w_scale_ptr=p(sd), out_rows_ptr=p(slots), out_scale_ptr=p(lw), stream=st)

    def fill(seed):
        f = _gen(seed)
        x.copy_(torch.randn(n, H, generator=f, device="cuda"))
        res.copy_(torch.randn(n, H, generator=f, device="cuda"))
        sel.copy_(torch.rand(n, E, generator=f, device="cuda").argsort(1)[:, :K])

    fill(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(torch.cuda.current_stream().cuda_stream)
    for seed in (2, 3):
        fill(seed)
        out.fill_(CANARY)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (total, s, off, slots, gu, hs, out)]
        layer(_st())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, (total, s, off, slots, gu, hs, out)))
    pool.device_status(_st())


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_pool_of_another_device_than_the_current():
    with MoePool(2048, 640, 512, 10, max_tokens=16, n_layers=1, device=1) as pool:
        torch.cuda.set_device(0)
        x, w = torch.ones(2, 256, device="cuda:1"), torch.ones(256, device="cuda:1")
        y = torch.empty_like(x)
        torch.cuda.synchronize(1)
        pool.rmsnorm_q8_device(2, 256, T_F32, x.data_ptr(), w.data_ptr(), 0.0, y_ptr=y.data_ptr())
        assert torch.cuda.current_device() == 0
        pool.device_status()
        assert bool((y == 1).all())


@pytest.mark.parametrize("n,kind", [(1, T_E4M3), (37, T_E4M3), (37, T_BF16)])
def test_layer_of_8bit_experts(n, kind):
    """The operators as a layer: norm of the residual, the pool's router, lists, gate|up on gathered rows, SiLU * up,
    down into the slots, the pool's combine; each step against its definition on the step's own inputs, and the layer's
    output against the 64-bit layer of the same quantized weights and selections."""
    H, FF, E, K, dt = 2048, 640, 512, 10, torch.bfloat16
    from inferenz_b200 import synth
    g = _gen(n)
    f8 = kind == T_E4M3
    scale = lambda *s: (torch.rand(*s, generator=g, device="cuda") + 0.5) / (120 * 45)  # noqa: E731
    if f8:
        quant = lambda r, k: (torch.randn(r, k, generator=g, device="cuda") * 120).clamp(-448, 448).to(F8)  # noqa: E731
        wg, wd = quant(E * 2 * FF, H), quant(E * H, FF)
        sg, sd = scale(E, 2 * FF // 128, H // 128), scale(E, H // 128, FF // 128)
    else:
        wg = (torch.randn(E * 2 * FF, H, generator=g, device="cuda") / 45).to(dt)
        wd = (torch.randn(E * H, FF, generator=g, device="cuda") / 25).to(dt)
        sg = sd = None
    p = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
    x, res = torch.randn(n, H, generator=g, device="cuda").to(dt), torch.randn(n, H, generator=g, device="cuda").to(dt)
    w = 1 + 0.1 * torch.randn(H, generator=g, device="cuda")
    with MoePool(H, FF, E, K, max_tokens=64, n_layers=1, device=0) as pool:
        pool.set_router(0, synth.router(0, E, H))
        st = _st()
        y = torch.empty_like(x)
        q, s = torch.empty(n, H, dtype=F8, device="cuda"), torch.empty(n, H // 128, device="cuda")
        pool.rmsnorm_q8_device(n, H, T_BF16, p(x), p(w), 1e-6, res_ptr=p(res), sum_ptr=p(res), y_ptr=p(y), q_ptr=p(q), s_ptr=p(s), stream=st)
        xin = y.float()
        sel, rw = torch.empty(n, K, dtype=torch.int32, device="cuda"), torch.empty(n, K, device="cuda")
        pool.route_device(0, n, p(xin), p(sel), p(rw), stream=st)
        off, rows, slots = (torch.empty(m, dtype=torch.int32, device="cuda") for m in (E + 1, n * K, n * K))
        lw = torch.empty(n * K, device="cuda")
        pool.expert_lists_device(n, K, E, p(sel), p(off), p(rows), p(slots), w_ptr=p(rw), w_out_ptr=p(lw), stream=st)
        gu = torch.empty(n * K, 2 * FF, dtype=dt, device="cuda")
        a, sa = (q, s) if f8 else (y, None)
        pool.grouped_matmul_device(kind, E, 2 * FF, H, n, n * K, p(a), p(wg), p(off), p(gu), T_BF16, a_scale_ptr=p(sa),
                                   w_scale_ptr=p(sg), in_rows_ptr=p(rows), stream=st)
        hy = torch.empty(n * K, FF, dtype=dt, device="cuda")
        hq, hs = torch.empty(n * K, FF, dtype=F8, device="cuda"), torch.empty(n * K, FF // 128, device="cuda")
        pool.silu_mul_q8_device(n * K, FF, T_BF16, p(gu), y_ptr=p(hy), q_ptr=p(hq), s_ptr=p(hs), stream=st)
        out = torch.empty(n * K, H, device="cuda")
        a2, sa2 = (hq, hs) if f8 else (hy, None)
        pool.grouped_matmul_device(kind, E, H, FF, n * K, n * K, p(a2), p(wd), p(off), p(out), T_F32, a_scale_ptr=p(sa2),
                                   w_scale_ptr=p(sd), out_rows_ptr=p(slots), out_scale_ptr=p(lw), stream=st)
        z = torch.empty(n, H, device="cuda")
        pool.combine_device(n, p(out), p(z), stream=st)
        pool.device_status(st)
    # each step on its own inputs
    A = _deq(q, s) if f8 else y.double()
    hA = _deq(hq, hs) if f8 else hy.double()
    off_ = off.tolist()
    want_z = torch.zeros(n, H, dtype=torch.float64, device="cuda")
    for e in range(E):
        i = torch.arange(off_[e], off_[e + 1], device="cuda")
        if not len(i):
            continue
        we, wde = wg[e * 2 * FF:(e + 1) * 2 * FF], wd[e * H:(e + 1) * H]
        W = _deq_w(we, sg[e:e + 1], 2 * FF)[0] if f8 else we.double()
        D = _deq_w(wde, sd[e:e + 1], H)[0] if f8 else wde.double()
        xe = A[rows[i].long()]
        want = xe @ W.t()
        assert bool(((gu[i].double() - want).abs() <= _product_bound(xe.abs() @ W.abs().t(), H, f8, want, dt)).all())
        sc = lw[i].double()[:, None]
        want = hA[i] @ D.t() * sc
        got = out[slots[i].long()].double()
        assert bool(((got - want).abs() <= _product_bound(hA[i].abs() @ D.abs().t() * sc, FF, f8, want, torch.float32)).all())
        gate = xe @ W.t()
        v = gate[:, :FF] * torch.sigmoid(gate[:, :FF]) * gate[:, FF:]
        want_z.index_add_(0, rows[i].long(), v @ D.t() * sc)
    v = gu[:, :FF].double() * torch.sigmoid(gu[:, :FF].double()) * gu[:, FF:].double()
    assert bool(((hy.double() - v).abs() <= (half_step(dt) + 12 * U) * v.abs() * 1.01 + 1e-38).all())
    assert torch.equal(z.double(), torch.stack([out.view(n, K, H)[:, j] for j in range(K)]).cumsum(0)[-1].double()) or \
        bool(((z.double() - out.view(n, K, H).double().sum(1)).abs() <= 10 * U * out.view(n, K, H).double().abs().sum(1)).all())
    # the whole layer: bf16 gate|up (2^-8 of each of g and u; silu's slope is at most 1.1 |g| + ..., so at most 3 * 2^-8 of
    # v relative to the row) and e4m3 hidden values (2^-4 each, independent): in the 2-norm of a token below 2^-4
    rel = (z.double() - want_z).norm(dim=1) / want_z.norm(dim=1)
    assert float(rel.max()) <= 2.0 ** -4


# ---------------------------------------------------------------------------------------------------------------------
# Sums of bf16 / f16 products over a long k. What stands in TMEM is a chunk of 256 k: 16 MMAs, each adding 16 products to the sum and
# truncating it (towards zero, by less than one step, 2u of the sum); the chunks' sums are added in fp32 to the nearest.


@pytest.mark.parametrize("t", [T_BF16, T_F16])
@pytest.mark.parametrize("m,gather", [(5, True), (300, False)])
def test_grouped_long_sums_do_not_drift(pool, t, m, gather):
    """Positive values, 200,008 k: every truncation of the running sum goes the same way. A chunk is off by at most one step per
    product, 2 * 256 u of it, the chunks' sums by u per addition: (512 + k / 256 + 4) u = 1298 u. Truncated over the whole k the
    sum would lose some 0.2 u per 16 k, 2400 u."""
    E, n, k, g = 2, 130, 200_008, _gen(m)
    a, w = (torch.rand(r, k, generator=g, device="cuda").add_(0.5).to(DT[t]) for r in (m, E * n))
    off = torch.tensor([0, m // 2, m], dtype=torch.int32, device="cuda")
    rows = torch.randperm(m, generator=g, device="cuda").to(torch.int32) if gather else None
    o = torch.full((m, n), CANARY, device="cuda")
    pool.grouped_matmul_device(t, E, n, k, m, m, a.data_ptr(), w.data_ptr(), off.data_ptr(), o.data_ptr(), T_F32,
                               in_rows_ptr=rows.data_ptr() if gather else None, stream=_st())
    for e in range(E):
        i = slice(m // 2 * e, m // 2 if e == 0 else m)
        x = a[rows[i].long()] if gather else a[i]
        want = x.double() @ w[e * n:(e + 1) * n].double().t()
        assert bool(((o[i].double() - want).abs() <= (512 + k // 256 + 4) * U * want).all())
    pool.device_status(_st())


@pytest.mark.parametrize("t", [T_BF16, T_F16])
@pytest.mark.parametrize("m,k", [(5, 10_240), (300, 10_240), (40, 2568), (300, 2568), (300, 264)])
def test_grouped_sums_have_no_bias(pool, t, m, k):
    """Random signs: the mean error in the direction of the result, relative to the mean result. The running sum of a chunk grows
    like the root of its MMAs: truncating each by at most 2u takes at most 2u * 16 * 2/3 = 21.3u of the chunk's size; rounding to the
    nearest adds nothing on the mean, but a mean over m n results of an error of sqrt(k / 256 + 1) u each strays by
    sqrt((k / 256 + 1) / (m n)) u, six of them allowed: under 1u here. Truncated over the whole k = 10240 it would be 160u."""
    n, g = 640, _gen(k + m)
    a, w = (torch.randn(r, k, generator=g, device="cuda").to(DT[t]) for r in (m, n))
    off = torch.tensor([0, m], dtype=torch.int32, device="cuda")
    o = torch.empty(m, n, device="cuda")
    pool.grouped_matmul_device(t, 1, n, k, m, m, a.data_ptr(), w.data_ptr(), off.data_ptr(), o.data_ptr(), T_F32, stream=_st())
    want = a.double() @ w.double().t()
    bias = ((o.double() - want) * want.sign()).mean() / want.abs().mean()
    assert abs(float(bias)) <= 22.3 * U


def test_layer_with_absent_experts():
    """The layer on one of two ranks: half of the experts are on the other one, a padded token has none at all. The slots held NaN and
    are cleared before the down product; combine gives the sum of this rank's experts, 0 for the padded token."""
    n, H, FF, E, K = 37, 2048, 640, 512, 10
    from inferenz_b200 import synth
    g = _gen(77)
    quant = lambda r, k: (torch.randn(r, k, generator=g, device="cuda") * 120).clamp(-448, 448).to(F8)  # noqa: E731
    scale = lambda *s: (torch.rand(*s, generator=g, device="cuda") + 0.5) / (120 * 45)  # noqa: E731
    own = E // 2  # experts 256 to 511
    wg, wd, sg, sd = quant(own * 2 * FF, H), quant(own * H, FF), scale(own, 2 * FF // 128, H // 128), scale(own, H // 128, FF // 128)
    p = lambda t: t.data_ptr()  # noqa: E731
    x, res = torch.randn(n, H, generator=g, device="cuda"), torch.randn(n, H, generator=g, device="cuda")
    w = 1 + 0.1 * torch.randn(H, generator=g, device="cuda")
    with MoePool(H, FF, E, K, max_tokens=64, n_layers=1, device=0) as pool:
        pool.set_router(0, synth.router(0, E, H))
        st = _st()
        y, q, s = torch.empty_like(x), torch.empty(n, H, dtype=F8, device="cuda"), torch.empty(n, H // 128, device="cuda")
        pool.rmsnorm_q8_device(n, H, T_F32, p(x), p(w), 1e-6, res_ptr=p(res), sum_ptr=p(res), y_ptr=p(y), q_ptr=p(q), s_ptr=p(s), stream=st)
        sel, rw = torch.empty(n, K, dtype=torch.int32, device="cuda"), torch.empty(n, K, device="cuda")
        pool.route_device(0, n, p(y), p(sel), p(rw), stream=st)
        local = torch.where(sel >= own, sel - own, -1 - sel)
        local[5] = -1
        off, rows, slots = (torch.empty(m, dtype=torch.int32, device="cuda") for m in (own + 1, n * K, n * K))
        lw = torch.empty(n * K, device="cuda")
        pool.expert_lists_device(n, K, own, p(local), p(off), p(rows), p(slots), w_ptr=p(rw), w_out_ptr=p(lw), stream=st)
        h = torch.full((n * K, 2 * FF), float("nan"), dtype=torch.bfloat16, device="cuda")
        pool.grouped_matmul_device(T_E4M3, own, 2 * FF, H, n, n * K, p(q), p(wg), p(off), p(h), T_BF16, a_scale_ptr=p(s),
                                   w_scale_ptr=p(sg), in_rows_ptr=p(rows), stream=st)
        hq, hs = torch.empty(n * K, FF, dtype=F8, device="cuda"), torch.empty(n * K, FF // 128, device="cuda")
        pool.silu_mul_q8_device(n * K, FF, T_BF16, p(h), q_ptr=p(hq), s_ptr=p(hs), stream=st)
        out = torch.full((n * K, H), float("nan"), device="cuda")
        out.zero_()
        pool.grouped_matmul_device(T_E4M3, own, H, FF, n * K, n * K, p(hq), p(wd), p(off), p(out), T_F32, a_scale_ptr=p(hs),
                                   w_scale_ptr=p(sd), out_rows_ptr=p(slots), out_scale_ptr=p(lw), stream=st)
        z = torch.full((n, H), float("nan"), device="cuda")
        pool.combine_device(n, p(out), p(z), stream=st)
        pool.device_status(st)
    listed = int(off[own])
    assert 0 < listed == int((local >= 0).sum()) < n * K
    want, mag = (torch.zeros(n, H, dtype=torch.float64, device="cuda") for _ in range(2))
    hA, off_ = _deq(hq, hs), off.tolist()
    for e in range(own):
        i = torch.arange(off_[e], off_[e + 1], device="cuda")
        if len(i):
            D, sc = _deq_w(wd[e * H:(e + 1) * H], sd[e:e + 1], H)[0], lw[i].double()[:, None]
            want.index_add_(0, rows[i].long(), hA[i] @ D.t() * sc)
            mag.index_add_(0, rows[i].long(), hA[i].abs() @ D.abs().t() * sc)
    # per entry (2 * 128 + 2 blocks + 4) u, the combine at most one u more per slot
    assert bool(((z.double() - want).abs() <= (256 + 2 * (FF // 128) + 4 + K) * U * mag).all())
    assert bool((z[5] == 0).all())


# ---------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("n,cols,scale", [(20_000, 640, 1.0), (6000, 644, 1e-3), (3000, 300, 1e15), (3000, 640, 1e-14), (2000, 384, 1e-16),
                                          (2000, 131, 1e-18)])
def test_silu_quantizes_the_fp32_quotient(pool, n, cols, scale):
    """q = e4m3(v / s) and s = max |v| / 448 bit for bit, with v the fp32 result and divisions in fp32; blocks of all magnitudes"""
    g = _gen(cols)
    x = torch.randn(n, 2 * cols, generator=g, device="cuda")
    x[:, cols:] *= scale
    y, q = torch.empty(n, cols, device="cuda"), torch.empty(n, cols, dtype=F8, device="cuda")
    nb = (cols + 127) // 128
    s = torch.empty(n, nb, device="cuda")
    # gates below 1 in small cases take v down to the floor of the scale
    x[:, :cols] *= min(1.0, scale)
    pool.silu_mul_q8_device(n, cols, T_F32, x.data_ptr(), y_ptr=y.data_ptr(), q_ptr=q.data_ptr(), s_ptr=s.data_ptr(), stream=_st())
    blocks = torch.nn.functional.pad(y, (0, nb * 128 - cols)).view(n, nb, 128)
    floor = torch.tensor(2.0 ** -100, device="cuda")
    most = torch.maximum(blocks.abs().amax(2), floor)
    by = torch.full_like(most, 448.0)  # a tensor: by a number torch multiplies by the reciprocal
    assert torch.equal(s, most / by)
    want = (blocks / s[:, :, None]).to(F8).view(n, -1)[:, :cols]
    assert torch.equal(q.view(torch.uint8), want.contiguous().view(torch.uint8))


@pytest.mark.parametrize("t", [T_F32, T_BF16])
def test_silu_of_far_negative_gates_beside_large_values(pool, t):
    """gates from -80 to -190 with up values to 2^127: the result is a normal number although exp(-g) is none. Three exponentials of 2u
    and four products: 10u; a result below the normal range is off by half a step of it (2^-150), and so may be a product before it, times
    a factor below 1."""
    dt, g = DT[t], _gen(3)
    n, cols = 300, 256
    x = torch.empty(n, 2 * cols, device="cuda")
    x[:, :cols] = -80 - 110 * torch.rand(n, cols, generator=g, device="cuda")
    x[:, :cols:7] = torch.randn(n, (cols + 6) // 7, generator=g, device="cuda")  # ordinary gates among them
    x[:, cols:] = torch.exp2(127 * torch.rand(n, cols, generator=g, device="cuda")) * torch.where(
        torch.rand(n, cols, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    x[0, :9] = torch.tensor([-87.0, -87.001, -86.999, -90.0, -100.0, -103.9, -176.0, -87.4, -88.7], device="cuda")
    x[0, cols:cols + 9] = 1.5e38
    x = x.to(dt)
    y = torch.empty(n, cols, device="cuda", dtype=dt)
    q, s = torch.empty(n, cols, dtype=F8, device="cuda"), torch.empty(n, cols // 128, device="cuda")
    pool.silu_mul_q8_device(n, cols, t, x.data_ptr(), y_ptr=y.data_ptr(), q_ptr=q.data_ptr(), s_ptr=s.data_ptr(), stream=_st())
    gate, up = x[:, :cols].double(), x[:, cols:].double()
    want = gate * torch.exp(torch.minimum(gate, torch.zeros_like(gate))) / (1 + torch.exp(-gate.abs())) * up
    assert float(want[0, 3].abs()) > 1  # what was 0
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    # an ordinary gate beside 2^127 leaves the type's range: infinite, and so is its block's scale
    fits = want.abs() <= torch.finfo(dt).max
    assert bool(((y.double() - want).abs() <= (half_step(dt) + 12 * U) * want.abs() * 1.01 + tiny)[fits].all())
    assert torch.equal(y.double()[~fits], torch.sign(want[~fits]) * float("inf"))
    whole = (want.abs() <= torch.finfo(torch.float32).max).view(n, -1, 128).all(2)
    assert torch.equal(torch.isinf(s), ~whole) and int(whole.sum()) > n // 2
    keep = whole[:, :, None].expand(n, cols // 128, 128).reshape(n, cols)
    S = torch.where(whole, s, 1.0)
    _check_quantized(torch.where(keep, q.float(), 0.0), torch.where(whole, S, float(2.0 ** -100) / 448), torch.where(keep, want, 0.0),
                     torch.where(keep, 12 * U * want.abs() + 2.0 ** -149, 0.0))


def test_silu_quantizes_around_infinities_and_nan(pool):
    """a NaN stays in its place and leaves its block's scale; an infinite value makes its block's scale infinite and its values NaN"""
    n, cols = 1, 384
    x = torch.ones(n, 2 * cols, device="cuda")
    x[0, 5], x[0, cols + 200] = float("nan"), float("inf")
    x[0, 300] = -float("inf")  # (-inf) exp(-inf): NaN
    y = torch.empty(n, cols, device="cuda")
    q, s = torch.empty(n, cols, dtype=F8, device="cuda"), torch.empty(n, 3, device="cuda")
    pool.silu_mul_q8_device(n, cols, T_F32, x.data_ptr(), y_ptr=y.data_ptr(), q_ptr=q.data_ptr(), s_ptr=s.data_ptr(), stream=_st())
    nan = torch.isnan(q.float())[0].nonzero().flatten().tolist()
    assert nan == [5] + list(range(128, 256)) + [300] and s[0, 1] == float("inf")
    one = torch.tensor(float(y[0, 0]), device="cuda") / torch.tensor(448.0, device="cuda")
    assert s[0, 0] == one and s[0, 2] == one and q[0, 0].float() == 448 and q[0, 383].float() == 448


@pytest.mark.parametrize("t", [T_F32, T_BF16])
@pytest.mark.parametrize("cols", [200, 2560, 8192, 16_388])
@pytest.mark.parametrize("eps,place", [(0.0, "apart"), (1e-6, "res"), (1e-33, "x"), (1e-6, "apart")])
def test_rmsnorm_of_rows_whose_squares_leave_the_range(pool, t, cols, eps, place):
    """rows from 2^-140 to 2^124, ordinary ones among them and next to each other in a block's walk; the tolerances of any row (30u, the
    factor being a power of two), and half a step of the smallest numbers for results down there"""
    dt, g = DT[t], _gen(cols)
    exps = [-140, 0, 124, -126, 64, 63, 62, 0, 60, 40, -40, -45, -46, -50, -64, -100, 80, 100, 120, 0] * 40  # several rows a block
    n = len(exps)
    x = (torch.randn(n, cols, generator=g, device="cuda").double() * torch.exp2(torch.tensor(exps, device="cuda").double())[:, None]).to(dt)
    w = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
    res = (x.float() * torch.randn(n, cols, generator=g, device="cuda")).to(dt)  # of the row's size
    res[2::20] = x[2::20] * 0.5  # but no sum past the range
    eps32 = float(np.float32(eps))
    h, v = _norm_want(x, res, w, eps32)
    assert float(h.abs().max()) < 3.3e38
    total = {"apart": torch.empty_like(x), "res": res, "x": x}[place]
    y, q = torch.empty_like(x), torch.empty(n, cols, dtype=F8, device="cuda")
    s = torch.empty(n, (cols + 127) // 128, device="cuda")
    pool.rmsnorm_q8_device(n, cols, t, x.data_ptr(), w.data_ptr(), eps, res_ptr=res.data_ptr(), sum_ptr=total.data_ptr(),
                           y_ptr=y.data_ptr(), q_ptr=q.data_ptr(), s_ptr=s.data_ptr(), stream=_st())
    e, tiny = half_step(dt), torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    assert bool(((total.double() - h).abs() <= (e + 2 * U) * h.abs() + tiny).all())  # the sum is that of the row as it is
    zero = (h == 0).all(1) & (eps32 == 0)  # bf16 ends at 2^-133: such rows are zeros, 0 / 0
    assert int(zero.sum()) == (40 if t == T_BF16 and eps32 == 0 else 0) and bool(torch.isnan(y[zero]).all())
    y, q, s, v = y[~zero], q.view(torch.uint8)[~zero].view(F8), s[~zero], v[~zero]
    assert bool(((y.double() - v).abs() <= (e + 30 * U) * v.abs() * (1 + e) + tiny).all())
    _check_quantized(q, s, v, 30 * U * v.abs() + 2.0 ** -149)


def test_rmsnorm_of_zero_infinite_and_nan_rows(pool):
    """zeros with eps give zeros, without it 0 / 0; an infinity leaves zeros beside its own NaN; a NaN takes its row. Other rows are as
    they are alone."""
    cols, inf, nan = 2560, float("inf"), float("nan")
    x = torch.randn(6, cols, generator=_gen(1), device="cuda")
    x[1], x[2, 7], x[3, 9], x[4] = 0, inf, nan, x[4] * 1e30
    w = torch.ones(cols, device="cuda")
    for eps in (1e-6, 0.0):
        y = torch.empty_like(x)
        pool.rmsnorm_q8_device(6, cols, T_F32, x.data_ptr(), w.data_ptr(), eps, y_ptr=y.data_ptr(), stream=_st())
        assert bool((y[1] == 0).all()) if eps else bool(torch.isnan(y[1]).all())
        assert bool(torch.isnan(y[2, 7])) and int((y[2] == 0).sum()) == cols - 1 and bool(torch.isnan(y[3]).all())
        rest = [0, 4, 5]
        _, v = _norm_want(x[rest], None, w, float(np.float32(eps)))
        assert bool(((y[rest].double() - v).abs() <= 31 * U * v.abs()).all())


def test_a_new_context_is_clear_before_its_first_call(pool):
    """A context made while the legacy stream is busy: its status words are cleared by then, not when that stream comes to it, so an
    error that a first call records on another stream stands."""
    stream = torch.cuda.Stream()
    sel = torch.tensor([[0, 4], [2, 1]], dtype=torch.int32, device="cuda")
    off, rows, slots = (torch.empty(5, dtype=torch.int32, device="cuda") for _ in range(3))
    _lists(pool, torch.zeros_like(sel), 4)  # the library's kernels are loaded: that waits for the device
    MoePool(2048, 640, 512, 10, max_tokens=16, n_layers=1, device=0).close()
    torch.cuda.synchronize()
    torch.cuda._sleep(1_500_000_000)  # some 0.8 s on the legacy stream
    with MoePool(2048, 640, 512, 10, max_tokens=16, n_layers=1, device=0) as pool:
        busy = not torch.cuda.default_stream().query()
        pool.expert_lists_device(2, 2, 4, sel.data_ptr(), off.data_ptr(), rows.data_ptr(), slots.data_ptr(), stream=stream.cuda_stream)
        torch.cuda.synchronize()
        with pytest.raises(InzgError) as e:
            pool.device_status(stream.cuda_stream)
        assert e.value.status == 7 and "expert id" in str(e.value)
        pool.device_status(stream.cuda_stream)
    if not busy:
        pytest.skip("the legacy stream was idle again before the context was made")


def test_device_status_waits_once(pool):
    """inzg_device_status, which callers of the older operators use after each step, is one copy and one wait: no slower than 1.5 times a
    copy of 64 bytes by the runtime (two copies and two waits were twice that). The least of many batches, in turn."""
    import ctypes
    import time
    src, dst = torch.zeros(64, dtype=torch.uint8, device="cuda"), torch.zeros(64, dtype=torch.uint8)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()

    def batch(call):
        t = time.perf_counter()
        for _ in range(100):
            call()
        return time.perf_counter() - t

    handle = ctypes.c_void_p(st.cuda_stream)

    def status():
        assert lib.inzg_device_status(pool._ctx, handle) == 0

    with torch.cuda.stream(st):
        copies, statuses = [], []
        for _ in range(30):
            copies.append(batch(lambda: dst.copy_(src)))
            statuses.append(batch(status))
    assert min(statuses) <= 1.5 * min(copies), (min(statuses), min(copies))


# ---------------------------------------------------------------------------------------------------------------------
# The tiles of 128 entries. The sizes are those of inzg__grouped_matmul_tile; test_q8_checks.py holds that they take these tiles.

LONG_LISTS = [(T_E4M3, 2048, 2048 * 72, 9600), (T_BF16, 2048, 2048 * 42, 9600)]  # type, groups, entries, n
RAGGED = [(T_E4M3, 3, 1700, 1301), (T_E4M3, 1, 1000, 1301), (T_BF16, 3, 1700, 1301), (T_F16, 1, 800, 1301)]


@pytest.mark.parametrize("t,E,entries,n", LONG_LISTS)
@pytest.mark.parametrize("gather", [False, True])
def test_wide_tiles_past_the_list_of_items(pool, t, E, entries, n, gather):
    """More items per SM than the 512 that a CTA lists: the roles search for the later ones. One or two entries of each group are listed, far
    fewer than `entries`: 2048 tiles x 38 (or 75) row blocks over the SMs."""
    g, k = _gen(n + gather), 16
    f8 = t == T_E4M3
    sizes = torch.randint(1, 3, (E,), generator=g, device="cuda")
    off = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), sizes.cumsum(0)])
    listed = int(off[-1])
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert E * ((n + 255) // 256 if f8 else (n + 127) // 128) // sms > 512 and listed < entries
    a_rows = listed if gather else entries
    a, w = _ints(a_rows, k, 16, DT[t], g), _ints(E * n, k, 16, DT[t], g)
    sa, sw = (_pow2((a_rows, 1), g), _pow2((E, (n + 127) // 128, 1), g)) if f8 else (None, None)
    rows = torch.full((entries,), -1, dtype=torch.int32, device="cuda")  # what is not listed is not read
    rows[:listed] = torch.randint(0, a_rows, (listed,), generator=g, device="cuda")
    to = torch.full((entries,), -1, dtype=torch.int32, device="cuda")
    to[:listed] = torch.randperm(listed, generator=g, device="cuda")
    o, off32 = torch.full((listed, n), CANARY, device="cuda"), off.to(torch.int32)
    p = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
    pool.grouped_matmul_device(t, E, n, k, a_rows, entries, p(a), p(w), p(off32), p(o), T_F32, lda=16, ldw=16, a_scale_ptr=p(sa),
                               w_scale_ptr=p(sw), in_rows_ptr=p(rows) if gather else None, out_rows_ptr=p(to), out_rows_n=listed, stream=_st())
    pool.device_status(_st())
    at = torch.arange(listed, device="cuda")
    group = torch.searchsorted(off[1:], at, right=True)
    src = rows[:listed].long() if gather else at
    x = a.float()[src]
    for c0 in range(0, n, 1200):  # small integers with powers of two: exact in fp32
        c1 = min(n, c0 + 1200)
        wc = (w.view(torch.uint8).view(E, n, -1)[:, c0:c1].contiguous().view(w.dtype) if f8 else w.unflatten(0, (E, n))[:, c0:c1]).float()
        want = torch.bmm(wc[group], x[:, :, None])[:, :, 0]
        if f8:
            want = want * sa[src] * sw[group, :, 0].repeat_interleave(128, 1)[:, c0:c1]
        assert torch.equal(o[to[:listed].long(), c0:c1], want)


@pytest.mark.parametrize("t,E,entries,n", RAGGED)
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("gather,scatter,ld", [(True, True, 1304), (False, False, 1304), (True, False, 1312), (False, True, 1301)])
def test_wide_tiles_of_ragged_columns(pool, t, E, entries, n, out, gather, scatter, ld):
    """rows of out whose pitch is a whole number of 16-byte pieces while their width is none: the last piece is written in part, what is
    behind it stays"""
    k = 520
    c = _grouped_case(t, E, entries, n, k, gather, scatter, 61)
    o, ob = _rows(c["out_rows_n"], n, ld, DT[out])
    assert o.data_ptr() % 16 == 0
    p = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
    pool.grouped_matmul_device(t, E, n, k, c["a"].shape[0], entries, p(c["a"]), p(c["w"]), p(c["off"]), p(o), out,
                               lda=c["a"].stride(0), ldw=c["w"].stride(0), ldo=ld, a_scale_ptr=p(c["as"]), w_scale_ptr=p(c["ws"]),
                               in_rows_ptr=p(c["in"]), out_rows_ptr=p(c["to"]), out_scale_ptr=p(c["sc"]),
                               out_rows_n=c["out_rows_n"], stream=_st())
    want, _, wrote = _grouped_want(c, E, entries, n)
    assert float(want.abs().max()) < 2.0 ** 20
    assert torch.equal(o.double(), torch.where(wrote[:, None], want, torch.tensor(CANARY, dtype=torch.float64, device="cuda"))
                       .to(DT[out]).double())
    _behind_is_untouched(ob, o)
    pool.device_status(_st())


@pytest.mark.parametrize("t", [T_F32, T_BF16])
@pytest.mark.parametrize("cols", [200, 2560, 8192, 16_392])
@pytest.mark.parametrize("place", ["res", "x", "apart"])
def test_rmsnorm_in_place_beside_rows_taken_once_more(pool, t, cols, place):
    """Rows that are taken once more among rows whose sum, written over x or res, would look like such a row if it were read again: just
    below the range, or cancelling to 0 without eps. Each row's outputs are those of the row alone."""
    dt, g, n = DT[t], _gen(cols + 1), 6000
    kind = torch.randint(0, 4, (n,), generator=g, device="cuda")[:, None]
    sign = torch.where(torch.rand(n, cols, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    near = 0.8 * (3.4e38 / cols) ** 0.5  # its squares' sum is 0.64 of the largest number, those of twice it are past it
    one = torch.randn(n, cols, generator=g, device="cuda")
    x = torch.where(kind == 0, one * 2.0 ** 100, torch.where(kind == 1, sign * near, one)).to(dt)
    part = {"res": -2.0, "x": -0.5, "apart": -2.0}[place]  # x + (x + res), or (x + res) + res, is 0
    res = torch.where(kind == 0, one * 2.0 ** 99, torch.where(kind == 1, 0.0, torch.where(kind == 2, x.float() * part, one))).to(dt)
    w = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
    h, v = _norm_want(x, res, w, 0.0)
    total = {"apart": torch.empty_like(x), "res": res, "x": x}[place]
    y, q = torch.empty_like(x), torch.empty(n, cols, dtype=F8, device="cuda")
    s = torch.empty(n, (cols + 127) // 128, device="cuda")
    pool.rmsnorm_q8_device(n, cols, t, x.data_ptr(), w.data_ptr(), 0.0, res_ptr=res.data_ptr(), sum_ptr=total.data_ptr(),
                           y_ptr=y.data_ptr(), q_ptr=q.data_ptr(), s_ptr=s.data_ptr(), stream=_st())
    e, tiny = half_step(dt), torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    assert bool(((total.double() - h).abs() <= (e + 2 * U) * h.abs() + tiny).all())
    assert bool(((y.double() - v).abs() <= (e + 30 * U) * v.abs() * (1 + e) + tiny).all())
    _check_quantized(q, s, v, 30 * U * v.abs() + 2.0 ** -149)


def test_rmsnorm_of_more_rows_than_one_launch(pool):
    """a block marks up to 8192 of its rows: more rows take more launches; the last ones far out"""
    n, cols = 148 * 32 * 8192 + 77, 8
    x = torch.ones(n, cols, device="cuda", dtype=torch.bfloat16)
    x[-50:] = 2.0 ** 90
    x[1000] = 2.0 ** 90
    w, y = torch.ones(cols, device="cuda"), torch.zeros(n, cols, device="cuda", dtype=torch.bfloat16)
    pool.rmsnorm_q8_device(n, cols, T_BF16, x.data_ptr(), w.data_ptr(), 0.0, y_ptr=y.data_ptr(), stream=_st())
    assert bool((y == 1).all())
