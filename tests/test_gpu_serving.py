"""The 8-bit decoder layer's operators against their definitions in 64 bits (tests/serving_ref.py)."""
import ctypes

import numpy as np
import pytest
import torch

from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture()
def serving(mlel):
    from mlel_b200 import serving
    assert serving.paged_error() == 0
    yield serving
    assert serving.paged_error() == 0


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def sentinel(*shape, dtype=torch.int8):
    return torch.full(shape, 77, dtype=dtype, device="cuda")


# ---------------------------------------------------------------- rows in 8 bits

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k", [(1, 1), (1, 7), (3, 8), (5, 257), (9, 1024), (2, 1025), (33, 2560), (4, 4096), (3, 4100), (2, 8192),
                                  (2, 8200), (1, 33000), (1000, 64)])
def test_quantize_rows(serving, dtype, m, k):
    x = (randn(gen(m * 10007 + k), m, k) * 3).to(DTYPES[dtype])
    x[m // 2, k // 2] = 300
    q, s = serving.quantize_rows(x)
    want_q, want_s = ref.quantize_rows(x)
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_ties_and_extremes(serving, dtype):
    t = DTYPES[dtype]
    x = torch.zeros(9, 64, dtype=t, device="cuda")
    x[0] = torch.arange(64, device="cuda").to(t) - 31.5
    x[0, 0] = 127  # scale 1: every other element lies in the middle between two integers
    x[1] = (torch.arange(64, device="cuda") * 3 - 94.5).to(t)
    x[1, 0] = -381  # scale 3, whose inverse is rounded
    x[3] = torch.finfo(t).smallest_normal * torch.finfo(t).eps  # the smallest magnitude there is
    x[4] = torch.finfo(t).max
    x[4, ::2] = -torch.finfo(t).max
    x[5, 5] = float("nan")
    x[6, 6] = float("-inf")
    x[6, 7] = 3
    x[7, 3] = -0.0
    x[8] = 1e-4
    q, s = serving.quantize_rows(x)
    want_q, want_s = ref.quantize_rows(x)
    assert np.array_equal(s.cpu().numpy(), want_s, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert torch.isnan((q.float() * s[:, None])[5]).all() and torch.isnan((q.float() * s[:, None])[6]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset, stride", [(0, 200), (1, 173), (8, 184), (3, 170)])
def test_quantize_rows_strided(serving, dtype, offset, stride):
    """Rows at any address on both sides; what lies between the output's rows stays."""
    m, k = 7, 170
    base = (randn(gen(offset + stride), m * stride + offset) * 2).to(DTYPES[dtype])
    x = base[offset:].as_strided((m, k), (stride, 1))
    store, scales = sentinel(m * stride + offset), torch.full((2 * m,), -1.0, device="cuda")
    q = store[offset:].as_strided((m, k), (stride, 1))
    serving.quantize_rows(x, q, scales[:m])
    want_q, want_s = ref.quantize_rows(x)
    assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(scales[:m].cpu().numpy(), want_s)
    untouched = torch.ones_like(store, dtype=torch.bool)
    untouched[offset:].as_strided((m, k), (stride, 1))[:] = False
    assert (store[untouched] == 77).all() and (scales[m:] == -1).all()


# ---------------------------------------------------------------- scaled products

def product_operands(seed, m, n, k, bias, extreme=False):
    g = gen(seed)
    def ints(r):
        if extreme:
            return torch.where(torch.rand(r, k, generator=g, device="cuda") < 0.5, -128, -127).to(torch.int8)
        return torch.randint(-128, 128, (r, k), generator=g, device="cuda", dtype=torch.int8)
    return (ints(m), torch.rand(m, generator=g, device="cuda") * 0.01, ints(n), torch.rand(n, generator=g, device="cuda") * 0.01,
            randn(g, n) if bias else None)


def check_product(serving, operands, dtype, out=None, tag=""):
    y = serving.matmul_scaled(*operands, out=out, dtype=dtype)
    want, off = ref.matmul_scaled(*operands)
    bound = off + ref.half_step(dtype) * (np.abs(want) + off) + ref.smallest_half_step(dtype)
    wrong = np.abs(ref.f64(y) - want) > bound
    assert not wrong.any(), (tag, int(wrong.sum()), np.argwhere(wrong)[:4].tolist(), np.argwhere(wrong)[-1].tolist())


@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 16, 16), (2, 130, 48), (3, 128, 128), (8, 257, 144), (16, 384, 2048), (17, 96, 300),
                                     (33, 1000, 512), (64, 256, 4096), (65, 129, 127), (100, 515, 1040), (128, 256, 256), (129, 257, 129),
                                     (256, 512, 128), (300, 77, 640), (511, 384, 96), (700, 1100, 272), (2000, 264, 160), (40, 8192, 1040)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul_scaled(serving, dtype, m, n, k):
    check_product(serving, product_operands(m + n + k, m, n, k, (m + n) % 2 == 0), DTYPES[dtype])


@pytest.mark.parametrize("m, n, k", [(300, 5000, 272), (1500, 4080, 400), (700, 9500, 128), (2049, 2568, 96)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul_scaled_many_tiles(serving, dtype, m, n, k):
    """Enough tiles of 256 tokens for every pair of SMs, over channels that end inside one; an output of wider rows."""
    t = DTYPES[dtype]
    store = torch.full((m, n + 24), 77.0, device="cuda", dtype=t)
    check_product(serving, product_operands(m + n + k, m, n, k, True), t, out=store[:, :n])
    assert (store[:, n:] == 77).all()


@pytest.mark.parametrize("m", [1, 5, 32, 63, 200, 300])
def test_matmul_scaled_longest_sums(serving, m):
    """Sums that fill 32-bit integers (131071 * 128 * 128 is 2^31 - 16384)."""
    check_product(serving, product_operands(m, m, 130, 131071 // 16 * 16, True, extreme=True), torch.float32)


@pytest.mark.parametrize("m, n, k", [(1, 50, 33), (5, 300, 257), (70, 130, 1001), (300, 520, 77), (20, 64, 20000)])
@pytest.mark.parametrize("a_off, b_off, out_off", [(0, 0, 0), (1, 0, 0), (0, 3, 0), (16, 32, 1), (5, 7, 3)])
def test_matmul_scaled_strided(serving, m, n, k, a_off, b_off, out_off):
    """Rows at any address; what lies between the output's rows stays."""
    a, sa, b, sb, bias = product_operands(m * 31 + n, m, n, k, True)
    def place(t, offset):
        stride = (t.shape[1] + 15) // 16 * 16 + (offset % 16)
        store = sentinel(t.shape[0] * stride + offset)
        view = store[offset:].as_strided(t.shape, (stride, 1))
        view.copy_(t)
        return view
    store = torch.full((m * (n + 8) + out_off,), 77.0, device="cuda", dtype=torch.bfloat16)
    out = store[out_off:].as_strided((m, n), (n + 5 if out_off else (n + 7) // 8 * 8, 1))
    check_product(serving, (place(a, a_off), sa, place(b, b_off), sb, bias), torch.bfloat16, out)
    mask = torch.ones_like(store, dtype=torch.bool)
    mask[out_off:].as_strided(out.shape, out.stride())[:] = False
    assert (store[mask] == 77).all()


@pytest.mark.parametrize("m, n", [(5, 200), (700, 900)])
def test_matmul_scaled_rows_that_overlap(serving, m, n):
    """Windows over one row of tokens, or of weights, 16 apart."""
    g = gen(m)
    line = torch.randint(-128, 128, (16 * 1000 + 96,), generator=g, device="cuda", dtype=torch.int8)
    a, sa, b, sb, bias = product_operands(m, m, n, 96, True)
    check_product(serving, (line.as_strided((m, 96), (16, 1)), sa, b, sb, bias), torch.float32)
    check_product(serving, (a, sa, line.as_strided((n, 96), (16, 1)), sb, bias), torch.float32)


def test_matmul_scaled_scales_that_are_not_finite(serving):
    a, sa, b, sb, _ = product_operands(5, 40, 150, 64, False)
    sa[3], sa[7], sb[100] = float("nan"), float("inf"), float("inf")
    y = serving.matmul_scaled(a, sa, b, sb, dtype=torch.float32).double()
    p = a.double() @ b.double().t()
    want = p * sa.double()[:, None] * sb.double()[None, :]
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))


@pytest.mark.parametrize("shape", [(1, 100), (3, 100), (2, 3, 128), (130, 333), (4, 2064)])
def test_quantized_linear(serving, shape):
    g = gen(sum(shape))
    x, n, k = randn(g, *shape).to(torch.float16), 75, shape[-1]
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    ws, bias = torch.rand(n, generator=g, device="cuda") * 0.01, randn(g, n)
    y = serving.QuantizedLinear(w, ws, bias)(x)
    assert y.shape == (*shape[:-1], n) and y.dtype == x.dtype
    q, s = ref.quantize_rows(x.reshape(-1, k))
    want, off = ref.matmul_scaled(torch.from_numpy(q), torch.from_numpy(s), w, ws, bias)
    bound = off + ref.half_step(x.dtype) * (np.abs(want) + off) + ref.smallest_half_step(x.dtype)
    assert (np.abs(ref.f64(y).reshape(-1, n) - want) <= bound).all()


# ---------------------------------------------------------------- the paged cache

class Paged:
    """A cache with random contents and a batch over it, the sequences given as (new tokens, length)."""

    def __init__(self, serving, seed, sequences, heads, page, d, skip=0, behind=0, wild=True):
        g = gen(seed)
        fresh = [n for n, _ in sequences]
        self.starts = [skip + sum(fresh[:i]) for i in range(len(fresh) + 1)]
        self.lengths = [l for _, l in sequences]
        self.tokens = self.starts[-1] + behind
        needed = [-(-l // page) for l in self.lengths]
        pages = sum(needed) + 2
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table, at = [], 0
        for n in needed:
            # entries that no token needs are not read
            self.table.append(order[at:at + n] + [-5, 1 << 30, 0][:max(needed) + 1 - n] + [-1] * max(0, max(needed) - 2 - n))
            at += n
        width = max(len(r) for r in self.table) if self.table else 1
        self.table = [r + [-7] * (width - len(r)) for r in self.table]
        self.data = torch.randint(-127, 128, (2, pages, heads, page, d), generator=g, device="cuda", dtype=torch.int8)
        self.scales = (0.3 + torch.rand(2, pages, heads, generator=g, device="cuda")) / 60
        if wild:  # scales of pages may differ by orders of magnitude
            self.scales *= 10.0 ** torch.randint(-2, 2, self.scales.shape, generator=g, device="cuda")
        self.spare = order[at:]
        self.scales[:, self.spare] = float("nan")  # pages of nobody
        self.cache = serving.PagedCache(self.data, self.scales)
        i32 = dict(dtype=torch.int32, device="cuda")
        table = torch.tensor(self.table, **i32).reshape(len(sequences), width)
        self.batch = serving.PagedBatch(torch.tensor(self.starts, **i32), torch.tensor(self.lengths, **i32), table, max(fresh, default=0),
                                        max(self.lengths, default=0))
        self.g, self.heads, self.page, self.d = g, heads, page, d

    def arrays(self):
        return self.data.cpu().numpy(), self.scales.cpu().numpy(), self.starts, self.lengths, self.table


MIXED = [(1, 1), (0, 0), (3, 3), (1, 16), (1, 17), (0, 40), (20, 49), (1, 100), (16, 16), (70, 150)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page, d, rot, interleaved", [(16, 64, 64, False), (16, 128, 64, True), (48, 80, 80, False), (64, 256, 128, False),
                                                       (256, 16, 16, True), (32, 96, 0, False)])
def test_append(serving, dtype, page, d, rot, interleaved):
    t, heads, hq = DTYPES[dtype], 3, 6
    p = Paged(serving, page + d, MIXED, heads, page, d, skip=2, behind=3, wild=False)
    wide = randn(p.g, p.tokens, (hq + 2 * heads) * d + 8).to(t)  # one projection's output holds all three
    q, k, v = (wide[:, 8 + a * d:8 + b * d].unflatten(1, (-1, d)) for a, b in [(0, hq), (hq, hq + heads), (hq + heads, hq + 2 * heads)])
    k[2:][::7] *= 30  # some tokens make their page's scale grow
    v[2:][::5] *= 0.01
    angle = torch.arange(200, device="cuda")[:, None] * torch.rand(rot // 2, generator=p.g, device="cuda")
    cos, sin = (angle.cos(), angle.sin()) if rot else (None, None)
    before = p.arrays()
    kept = q.clone()
    out = torch.full((p.tokens, hq, d), 77.0, dtype=t, device="cuda")
    got = p.cache.append(k, v, cos, sin, p.batch, q=q, q_out=out, interleaved=interleaved)
    assert got is out
    c, s = (None, None) if not rot else (ref.f64(cos), ref.f64(sin))
    want, want_scales = ref.append(*before, ref.f64(k), ref.f64(v), c, s, interleaved)
    assert np.array_equal(p.scales.cpu().numpy(), want_scales, equal_nan=True)
    assert np.array_equal(p.data.cpu().numpy(), want)
    x, inside = ref.f64(kept), slice(p.starts[0], p.starts[-1])
    y, off = x.copy(), np.zeros_like(x)
    for b, length in enumerate(p.lengths):
        for i in range(p.starts[b], p.starts[b + 1]):
            if rot:
                position = length - p.starts[b + 1] + i
                y[i] = ref.rotate(x[i], c[position], s[position], interleaved)
                off[i] = 2.0 ** -23 * np.abs(x[i]).max()  # a product and a fused sum of two terms
    bound = off + ref.half_step(t) * (np.abs(y) + off) + ref.smallest_half_step(t)
    assert (np.abs(ref.f64(out) - y) <= bound)[inside].all()
    assert (out[:p.starts[0]] == 77).all() and (out[p.starts[-1]:] == 77).all()
    # in place, and again: the same integers, since nothing grows any more
    p.cache.append(k, v, cos, sin, p.batch, q=q, q_out=q, interleaved=interleaved)
    assert torch.equal(q[inside], out[inside]) and torch.equal(q[:2], kept[:2])
    assert np.array_equal(p.data.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d, rot, interleaved, shift", [(64, 24, False, 0), (64, 48, True, 0), (32, 32, False, 1), (48, 20, True, 3), (128, 8, False, 0)])
def test_append_odd_rotations_and_addresses(serving, dtype, d, rot, interleaved, shift):
    """Rotated parts that no vector width divides, and rows at any element's address."""
    t = DTYPES[dtype]
    p = Paged(serving, d + rot, MIXED, 2, 16, d, wild=False)
    wide = randn(p.g, p.tokens, 6 * d + shift).to(t)
    q, k, v = (wide[:, shift + a * d:shift + b * d].unflatten(1, (-1, d)) for a, b in [(0, 2), (2, 4), (4, 6)])
    angle = torch.arange(200, device="cuda")[:, None] * torch.rand(rot // 2, generator=p.g, device="cuda")
    before = p.arrays()
    out = p.cache.append(k, v, angle.cos(), angle.sin(), p.batch, q=q, interleaved=interleaved)
    c, s = ref.f64(angle.cos()), ref.f64(angle.sin())
    want, want_scales = ref.append(*before, ref.f64(k), ref.f64(v), c, s, interleaved)
    assert np.array_equal(p.scales.cpu().numpy(), want_scales, equal_nan=True) and np.array_equal(p.data.cpu().numpy(), want)
    x = ref.f64(q)
    for b, length in enumerate(p.lengths):
        for i in range(p.starts[b], p.starts[b + 1]):
            position = length - p.starts[b + 1] + i
            y = ref.rotate(x[i], c[position], s[position], interleaved)
            off = 2.0 ** -23 * np.abs(x[i]).max()
            assert (np.abs(ref.f64(out[i]) - y) <= off + ref.half_step(t) * (np.abs(y) + off) + ref.smallest_half_step(t)).all()


def test_append_many_tokens(serving):
    """Blocks of several queries that straddle sequences, some of them empty."""
    sequences = [(500, 500), (0, 7), (1, 90), (0, 0), (3, 3), (700, 733), (1, 1)]
    p = Paged(serving, 4, sequences, 1, 32, 16, skip=3, behind=9, wild=False)
    q, k, v = (randn(p.g, p.tokens, 1, 16).bfloat16() for _ in range(3))
    angle = torch.arange(800, device="cuda")[:, None] * torch.rand(8, generator=p.g, device="cuda")
    before = p.arrays()
    out = torch.full_like(q, 77.0)
    p.cache.append(k, v, angle.cos(), angle.sin(), p.batch, q=q, q_out=out)
    want, want_scales = ref.append(*before, ref.f64(k), ref.f64(v), ref.f64(angle.cos()), ref.f64(angle.sin()), False)
    assert np.array_equal(p.scales.cpu().numpy(), want_scales, equal_nan=True) and np.array_equal(p.data.cpu().numpy(), want)
    position = torch.cat([torch.arange(l - n, l) for n, l in sequences]).cuda()
    x, c, s = q[3:-9, 0].double(), angle.cos()[position].double(), angle.sin()[position].double()
    y = torch.cat((x[:, :8] * c - x[:, 8:] * s, x[:, 8:] * c + x[:, :8] * s), 1)
    assert ((out[3:-9, 0].double() - y).abs() <= 2.0 ** -8 * (y.abs() + 2.0 ** -20 * x.abs().amax()) + 2.0 ** -22 * x.abs().amax()).all()
    assert (out[:3] == 77).all() and (out[-9:] == 77).all()


@pytest.mark.parametrize("tiny", [1e-40, 3e-39, 1e-37])
def test_append_the_smallest_magnitudes(serving, tiny):
    """Scales among the subnormal numbers: quotients are rounded and bounded as elsewhere."""
    p = Paged(serving, 8, [(5, 9), (1, 40)], 2, 16, 16, wild=False)
    p.scales[:, [s for t in p.table for s in t if 0 <= s < p.data.shape[1]]] = 0
    k, v = (randn(p.g, p.tokens, 2, 16) * tiny).bfloat16(), (randn(p.g, p.tokens, 2, 16) * tiny).bfloat16()
    before = p.arrays()
    p.cache.append(k, v, None, None, p.batch)
    want, want_scales = ref.append(*before, ref.f64(k), ref.f64(v), None, None, False)
    assert np.array_equal(p.scales.cpu().numpy(), want_scales, equal_nan=True) and np.array_equal(p.data.cpu().numpy(), want)


def test_append_what_is_not_finite(serving):
    """An infinity or a NaN makes the scale of its page and head that; other heads and pages do not notice."""
    p = Paged(serving, 5, [(20, 24), (4, 9)], 2, 16, 32, wild=False)
    k, v = randn(p.g, p.tokens, 2, 32).half(), randn(p.g, p.tokens, 2, 32).half()
    k[3, 0, 5], v[15, 1, 0] = float("nan"), float("-inf")
    before = p.arrays()
    p.cache.append(k, v, None, None, p.batch)
    want, want_scales = ref.append(*before, ref.f64(k), ref.f64(v), None, None, False)
    got = p.scales.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want_scales)) and np.array_equal(np.isinf(got), np.isinf(want_scales))
    fine = np.isfinite(want_scales)
    assert np.array_equal(got[fine], want_scales[fine])
    assert np.array_equal(p.data.cpu().numpy()[fine], want[fine])


def test_append_zeros_and_growth_by_a_little(serving):
    """Zeros alone give a scale of 0; a scale that grows by one unit in its last place leaves the integers."""
    p = Paged(serving, 6, [(1, 5)], 1, 16, 16, wild=False)
    slot = p.table[0][0]
    p.scales[:, slot] = 0
    zero = torch.zeros(1, 1, 16, dtype=torch.float16, device="cuda")
    p.cache.append(zero, zero, None, None, p.batch)
    assert (p.scales[:, slot] == 0).all() and (p.data[:, slot, 0, 4] == 0).all()
    one = torch.ones(1, 1, 16, dtype=torch.float16, device="cuda")
    now = np.float32(1 / 127)
    p.scales[:, slot] = float(np.nextafter(now, np.float32(0)))
    before = p.data.clone()
    p.cache.append(one, one, None, None, p.batch)
    assert (p.scales[:, slot] == float(now)).all()
    assert torch.equal(p.data[:, slot, 0, :4], before[:, slot, 0, :4]) and (p.data[:, slot, 0, 4] == 127).all()


def check_attention(serving, p, q, out, dtype, **how):
    got = p.cache.attend(q, p.batch, out=out, **how)
    assert got is out
    want, bound = ref.attend(*p.arrays(), ref.f64(q), how.get("scale") or p.d ** -0.5, how.get("causal", True), how.get("window", 0),
                             how.get("softcap", 0.0), dtype)
    got = ref.f64(out)
    left = np.isnan(want)
    assert (got[left] == 77).all()
    wrong = ~(np.abs(got - want) <= bound) & ~left
    assert not wrong.any(), (int(wrong.sum()), np.argwhere(wrong)[:4].tolist(), np.argwhere(wrong)[-1].tolist(),
                             float(np.nanmax(np.where(wrong, np.abs(got - want) / np.maximum(bound, 1e-30), 0))))


def query(p, heads, t, loud=1.0):
    """Queries as part of a projection's output, and where the answer goes: rows apart, heads apart."""
    q = (randn(p.g, p.tokens, heads, p.d + 8) * loud).to(t)[..., :p.d]
    store = torch.full((p.tokens, heads + 1, p.d + 16), 77.0, dtype=t, device="cuda")
    return q, store[:, 1:, 8:8 + p.d]


DECODE = [(1, 1), (1, 2), (0, 30), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 200), (0, 0), (1, 1000)]
FEW = [(2, 2), (3, 70), (0, 9), (5, 5), (1, 300), (4, 129)]
CHUNKS = [(40, 40), (1, 70), (130, 200), (17, 400), (0, 3), (64, 64), (129, 129)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads, group", [(2, 1), (2, 4), (1, 5), (1, 9), (1, 16), (1, 20), (2, 32), (2, 40)])
@pytest.mark.parametrize("page, d", [(16, 64), (64, 128), (48, 80), (32, 256), (256, 16), (16, 96)])
def test_attention_single_tokens(serving, dtype, heads, group, page, d):
    t = DTYPES[dtype]
    p = Paged(serving, heads * group + page + d, DECODE, heads, page, d, skip=1, behind=2)
    check_attention(serving, p, *query(p, heads * group, t, 2.0), t)


@pytest.mark.parametrize("sequences", [FEW, CHUNKS], ids=["few", "chunks"])
@pytest.mark.parametrize("how", [{}, {"causal": False}, {"window": 1}, {"window": 37}, {"softcap": 3.0}, {"scale": -0.3},
                                 {"window": 100, "causal": False, "softcap": 20.0}], ids=str)
@pytest.mark.parametrize("group, page, d", [(4, 16, 128), (3, 32, 64), (1, 64, 256), (8, 48, 80)])
def test_attention_masks(serving, sequences, how, group, page, d):
    t = torch.float16 if group % 2 else torch.bfloat16
    p = Paged(serving, group + page + d, sequences, 2, page, d, skip=1, behind=1)
    check_attention(serving, p, *query(p, 2 * group, t, 2.0), t, **how)


@pytest.mark.parametrize("fresh, length, heads, group, d, page", [(300, 300, 1, 4, 128, 64), (257, 1000, 2, 1, 64, 16), (150, 150, 1, 8, 256, 128),
                                                                  (1, 9000, 1, 8, 128, 16), (2, 5000, 2, 3, 64, 64)])
def test_attention_long(serving, fresh, length, heads, group, d, page):
    p = Paged(serving, fresh + length, [(fresh, length)], heads, page, d)
    check_attention(serving, p, *query(p, heads * group, torch.bfloat16), torch.bfloat16)


@pytest.mark.parametrize("how", [{}, {"window": 700}, {"softcap": 5.0}, {"causal": False}], ids=str)
@pytest.mark.parametrize("sequences, heads, group, d, page", [([(70, 5000)], 1, 1, 128, 64), ([(40, 3000), (33, 40), (0, 9), (1, 2500)], 1, 2, 64, 16),
                                                              ([(300, 2600)], 2, 1, 96, 48), ([(20, 4100)], 1, 4, 256, 32)])
def test_attention_chunks_of_long_sequences(serving, sequences, heads, group, d, page, how):
    """Few tiles of rows over many keys, which blocks share, some sequences with fewer keys than there are shares."""
    p = Paged(serving, d + page, sequences, heads, page, d, behind=1)
    check_attention(serving, p, *query(p, heads * group, torch.float16), torch.float16, **how)


@pytest.mark.parametrize("fresh, d, how", [(3, 64, {}), (7, 128, {"window": 900}), (3, 256, {"softcap": 5.0}), (4, 256, {})], ids=str)
def test_attention_several_tiles_share_the_line(serving, fresh, d, how):
    """Drafts of several tiles of eight rows, cut into pieces over the whole device and joined: many sequences, some long."""
    lengths = [2000, 9, 1500, 40, 300, 17] + [(37 * i) % 120 + fresh for i in range(54)]
    p = Paged(serving, fresh + d, [(min(fresh, 1 + i % fresh) if i % 5 else 0 if i % 2 else fresh, n) for i, n in enumerate(lengths)], 4, 16, d)
    check_attention(serving, p, *query(p, 16, torch.float16), torch.float16, **how)
    assert any(v > 0 for v in p.batch._space.values()), "the case is meant to want a workspace"


@pytest.mark.parametrize("sequences", [[(1, 300)], [(100, 300)]], ids=["one", "chunk"])
def test_attention_one_key_has_all(serving, sequences):
    """A score that drowns all others: the answer is that token's value; and thousands of others share what is left."""
    p = Paged(serving, 77, sequences, 1, 16, 64, wild=False)
    q, out = query(p, 2, torch.float16)
    q[:] = 0
    q[..., 0] = 100
    p.data[0] = 0
    p.data[0, p.table[0][3], 0, 5, 0] = 127
    p.scales[0] = 1 / 127
    check_attention(serving, p, q, out, torch.float16, causal=False, scale=1.0)


def test_attention_what_is_not_finite_stays_with_its_rows(serving):
    """A page without finite scales, and NaN queries: rows that the mask keeps from them are as they were."""
    sequences = [(100, 160), (1, 200), (4, 64)]
    p = Paged(serving, 3, sequences, 1, 16, 64, wild=False)
    q, out = query(p, 4, torch.bfloat16)
    other = torch.full_like(out, 77.0)
    p.cache.attend(q, p.batch, out=out)
    bad_at = 112  # the first row of a page of sequence 0
    p.scales[:, p.table[0][bad_at // 16]] = float("nan")
    q[70, 2] = float("nan")
    p.cache.attend(q, p.batch, out=other)
    for row in range(p.tokens):
        position = 60 + row
        touched = row < 100 and position >= bad_at
        for h in range(4):
            if touched or (row == 70 and h == 2):
                assert torch.isnan(other[row, h]).all(), (row, h)
            else:
                assert torch.equal(other[row, h], out[row, h]), (row, h)
    # a window of 20: row r attends to tokens 60 + r - 19 .. 60 + r, behind the page (112 .. 127) from r = 87 on
    clean = torch.full_like(out, 77.0)
    p.cache.attend(q, p.batch, out=clean, window=20)
    assert torch.isfinite(clean[87:100]).all() and torch.isnan(clean[60:68]).all()


@pytest.mark.parametrize("fresh", [1, 3, 150])
def test_bad_numbers_are_left_out_and_told_of(serving, fresh):
    """Sequences and pages that contradict the shapes: nothing is read or written there, the others are served."""
    p = Paged(serving, 9, [(fresh, 170), (fresh, 180), (fresh, 190)], 2, 16, 64, wild=False)
    q, out = query(p, 4, torch.float16)
    check_attention(serving, p, q, out, torch.float16)
    good = out.clone()
    rows = [slice(p.starts[b], p.starts[b + 1]) for b in range(3)]
    for field, index, value in [("lengths", 1, 200), ("lengths", 1, fresh - 1), ("lengths", 1, -4), ("starts", 3, p.tokens + 1)]:
        keep = getattr(p.batch, field)[index].clone()
        getattr(p.batch, field)[index] = value
        out.fill_(77.0)
        p.cache.attend(q, p.batch, out=out)
        assert serving.paged_error() == 1
        bad = 1 if field == "lengths" else 2
        for b in range(3):
            assert torch.equal(out[rows[b]], good[rows[b]] if b != bad else torch.full_like(out[rows[b]], 77.0)), (field, value, b)
        data, scales = p.data.clone(), p.scales.clone()
        k = randn(p.g, p.tokens, 2, 64).half()
        p.cache.append(k, k, None, None, p.batch, q=q)
        assert serving.paged_error() == 1
        mine = [s for s in p.table[bad] if 0 <= s < p.data.shape[1]]
        assert torch.equal(p.data[:, mine], data[:, mine])
        p.data.copy_(data)
        p.scales.copy_(scales)
        getattr(p.batch, field)[index] = keep
    # a page outside the cache: its tokens are not attended to
    for value in (-1, p.data.shape[1], 1 << 30):
        page = 2
        keep = p.batch.page_table[1, page].clone()
        p.batch.page_table[1, page] = value
        out.fill_(77.0)
        p.cache.attend(q, p.batch, out=out)
        assert serving.paged_error() == 2
        assert torch.equal(out[rows[0]], good[rows[0]]) and torch.equal(out[rows[2]], good[rows[2]])
        p.batch.page_table[1, page] = keep
        # the same tokens made negligible: keys that give scores far below all others are as good as none
    last = (p.lengths[0] - 1) // 16
    keep = p.batch.page_table[0, last].clone()
    p.batch.page_table[0, last] = -3
    data = p.data.clone()
    k = randn(p.g, p.tokens, 2, 64).half()
    p.cache.append(k, k, None, None, p.batch)
    assert serving.paged_error() == 2
    assert torch.equal(p.data[:, p.table[0][last]], data[:, p.table[0][last]])
    p.batch.page_table[0, last] = keep


# ---------------------------------------------------------------- together, and around them

def test_layer_by_layer_decoding(serving):
    """A prompt, then tokens one by one, against the same tokens in one go: projections, cache and attention as a program uses
    them.  The integers of a page depend on the order of its tokens (its scale grows), so the two agree within the cache's steps."""
    g = gen(1)
    heads, hq, d, page, total = 2, 8, 64, 16, 75
    x = randn(g, total, 512).half()
    w = torch.randint(-127, 128, ((hq + 2 * heads) * d, 512), generator=g, device="cuda", dtype=torch.int8)
    linear = serving.QuantizedLinear(w, torch.full((w.shape[0],), 0.0006, device="cuda"))
    angle = torch.arange(total, device="cuda")[:, None] * 10000.0 ** (-torch.arange(d // 2, device="cuda") / (d // 2))
    cos, sin = angle.cos().float(), angle.sin().float()
    table = torch.tensor([[3, 0, 4, 1, 5]], dtype=torch.int32, device="cuda")

    def step(cache, lo, hi):
        y = linear(x[lo:hi])
        q, k, v = (y[:, a * d:b * d].unflatten(1, (-1, d)) for a, b in ((0, hq), (hq, hq + heads), (hq + heads, hq + 2 * heads)))
        batch = serving.PagedBatch(torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda"),
                                   torch.tensor([hi], dtype=torch.int32, device="cuda"), table, hi - lo, total)
        q = cache.append(k, v, cos, sin, batch, q=q)
        return q, v, cache.attend(q, batch)

    whole, piece = serving.PagedCache.empty(6, heads, page, d), serving.PagedCache.empty(6, heads, page, d)
    q, v, want = step(whole, 0, total)
    parts = [step(piece, lo, hi)[2] for lo, hi in [(0, 40), (40, 41), (41, 43)] + [(i, i + 1) for i in range(43, total)]]
    got = torch.cat(parts)
    # integers of 1 / 127 of a page's largest element; rescaled ones are off by up to a step per growth
    assert (got.float() - want.float()).abs().max() < 0.1 * v.abs().max()
    assert torch.nn.functional.cosine_similarity(got.float().flatten(), want.float().flatten(), dim=0) > 0.999


def test_capture_replay_and_other_streams(serving):
    """Each call captured into a graph and replayed on new contents gives what the call itself gives, from a stream of its own."""
    p = Paged(serving, 21, [(1, 130), (1, 700), (1, 20)], 2, 16, 64, wild=False)
    g, hq = p.g, 8
    linear = serving.QuantizedLinear(torch.randint(-127, 128, ((hq + 4) * 64, 256), generator=g, device="cuda", dtype=torch.int8),
                                     torch.full(((hq + 4) * 64,), 0.001, device="cuda"))
    x = randn(g, 3, 256).half()
    angle = torch.rand(700, 32, generator=g, device="cuda")
    cos, sin = angle.cos(), angle.sin()

    def layer():
        y = linear(x)
        q, k, v = y[:, :hq * 64].unflatten(1, (-1, 64)), y[:, hq * 64:(hq + 2) * 64].unflatten(1, (-1, 64)), y[:, (hq + 2) * 64:].unflatten(1, (-1, 64))
        return p.cache.attend(p.cache.append(k, v, cos, sin, p.batch, q=q), p.batch)

    first = (p.data.clone(), p.scales.clone())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = layer()
    torch.cuda.synchronize()
    for seed in (1, 2):
        x.copy_(randn(gen(seed), 3, 256).half())
        p.data.copy_(first[0]), p.scales.copy_(first[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = held.clone()
        p.data.copy_(first[0]), p.scales.copy_(first[1])
        assert torch.equal(layer(), replayed)


def test_capture_with_a_workspace(serving):
    """Two captured graphs of one long sequence each, whose parts lie in a workspace, replayed in turn and from two streams."""
    jobs = []
    for seed in (31, 32):
        p = Paged(serving, seed, [(1, 20000), (1, 30)], 2, 64, 128)
        q = query(p, 8, torch.bfloat16)[0]
        want = p.cache.attend(q, p.batch)
        graph = torch.cuda.CUDAGraph()
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            held = p.cache.attend(q, p.batch)
        jobs.append((graph, stream, want, held, p, q))
    assert any(v > 0 for v in jobs[0][4].batch._space.values()), "the case is meant to want a workspace"
    for _ in range(3):
        for graph, stream, *_ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, want, held, *_ in jobs:
        assert torch.equal(want, held)


def test_ordinary_launches_give_the_same(mlel, serving):
    """Without programmatic dependent launches."""
    lib = mlel.lib()
    p = Paged(serving, 41, [(1, 900), (1, 20000)], 2, 16, 64, wild=False)
    many = Paged(serving, 42, [(90, 400)], 2, 32, 128, wild=False)
    x = randn(gen(1), 40, 512).bfloat16()
    linear = serving.QuantizedLinear(torch.randint(-127, 128, (700, 512), generator=p.g, device="cuda", dtype=torch.int8), torch.ones(700, device="cuda"))
    q, q2 = query(p, 4, torch.float16)[0], query(many, 4, torch.float16)[0]
    got = []
    try:
        for value in (1, 0):
            assert lib.mlel_set_tuning(b"dependent_launch", value) == 0
            got.append((linear(x), p.cache.attend(q, p.batch), many.cache.attend(q2, many.batch)))
    finally:
        assert lib.mlel_set_tuning(b"dependent_launch", 1) == 0
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_nothing_to_do(serving):
    """No tokens, no sequences, sequences without new tokens."""
    linear = serving.QuantizedLinear(torch.zeros(5, 33, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"))
    assert linear(torch.zeros(0, 33, device="cuda")).shape == (0, 5)
    q, s = serving.quantize_rows(torch.zeros(0, 7, device="cuda"))
    assert q.shape == (0, 7) and s.shape == (0,)
    for sequences in ([], [(0, 20), (0, 0)]):
        p = Paged(serving, 1, sequences, 1, 16, 16, behind=2)
        x, out = query(p, 2, torch.float16)
        before = p.data.clone()
        p.cache.attend(x, p.batch, out=out)
        p.cache.append(x[:, :1].contiguous(), x[:, :1].contiguous(), None, None, p.batch)
        assert (out == 77).all() and torch.equal(p.data, before)


def test_page_table_of_a_larger_program(serving):
    """Rows of the page table apart from one another, lengths far below their bound, as a program's own tables have them."""
    p = Paged(serving, 51, [(1, 100), (3, 300), (1, 40)], 2, 16, 64)
    q, out = query(p, 4, torch.float16)
    check_attention(serving, p, q, out, torch.float16)
    wide = torch.full((3, 1000), -1, dtype=torch.int32, device="cuda")
    wide[:, :p.batch.page_table.shape[1]] = p.batch.page_table
    for bound in (1000 * 16, 600 * 16):
        other = serving.PagedBatch(p.batch.starts, p.batch.lengths, wide[:, :bound // 16], 7, bound)
        again = torch.full_like(out, 77.0)
        p.cache.attend(q, other, out=again)
        # another division of the keys: the same up to a rounding of the result
        assert ((again.float() - out.float()).abs() <= 2.0 ** -10 * out.float().abs() + 2.0 ** -9 * out.float().abs().amax()).all()
    wide_rows = serving.PagedBatch(p.batch.starts, p.batch.lengths, wide, 40, 16000)  # the kernel for many rows
    p.cache.attend(q, wide_rows, out=again)
    assert ((again.float() - out.float()).abs() <= 2.0 ** -10 * out.float().abs() + 2.0 ** -9 * out.float().abs().amax()).all()


def test_two_streams_at_once(serving):
    """Calls that run beside one another share nothing: the same results as one after another."""
    jobs = []
    for seed, sequences in enumerate(([(1, 900)] * 4, [(60, 600)], [(1, 3000)], [(3, 500)] * 3)):
        p = Paged(serving, seed, sequences, 2, 16, 128)
        jobs.append((p, query(p, 8, torch.float16)[0]))
    want = [p.cache.attend(q, p.batch) for p, q in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for _ in range(5):
        for s, (p, q) in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(p.cache.attend(q, p.batch))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(jobs)]), i


def test_operands_are_where_they_are_said_to_be(mlel, serving):
    """Host memory under a device tensor's name is refused before anything runs."""
    x = torch.zeros(4, 64)
    T, lib = mlel.device_tensor, mlel.lib()
    rc = lib.mlel_cuda_quantize_rows(ctypes.byref(T(x.data_ptr(), mlel.F32, (4, 64))), ctypes.byref(T(x.data_ptr(), mlel.I8, (4, 64))),
                                     ctypes.byref(T(x.data_ptr(), mlel.F32, (4,))), None)
    assert rc == -13 and b"current device" in ctypes.c_char_p(lib.mlel_last_error()).value


def test_what_is_described_stays(serving):
    """Objects hold descriptions of their tensors: values change in place, the tensors do not."""
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = serving.PagedBatch(torch.tensor([0, 1], **i32), torch.tensor([1], **i32), torch.tensor([[0]], **i32), 1, 16)
    cache = serving.PagedCache.empty(2, 1, 16, 64)
    linear = serving.QuantizedLinear(torch.ones(16, 32, dtype=torch.int8, device="cuda"), torch.ones(16, device="cuda"))
    for thing, name in ((batch, "lengths"), (batch, "max_new"), (cache, "data"), (linear, "weight"), (linear, "bias")):
        with pytest.raises(AttributeError, match="make a new"):
            setattr(thing, name, getattr(thing, name))
    x = torch.ones(2, 32, device="cuda")
    before = linear(x)
    linear.scales.mul_(2.0)
    linear.weight.neg_()
    assert torch.equal(linear(x), -2 * before)


def test_offsets_beyond_32_bits(serving):
    """A cache of over 4 GB: pages at both of its ends."""
    heads, page, d = 8, 256, 256
    pages = (1 << 32) // (heads * page * d) + 3
    data = torch.zeros(2, pages, heads, page, d, dtype=torch.int8, device="cuda")
    cache = serving.PagedCache(data, torch.zeros(2, pages, heads, device="cuda"))
    i32 = dict(dtype=torch.int32, device="cuda")
    for fresh in (1, 200):
        batch = serving.PagedBatch(torch.tensor([0, fresh, 2 * fresh], **i32), torch.tensor([fresh, fresh], **i32),
                                   torch.tensor([[0], [pages - 1]], **i32), fresh, fresh)
        k, v, q = (randn(gen(fresh + i), 2 * fresh, heads, d).half() for i in range(3))
        k[fresh:], v[fresh:], q[fresh:] = k[:fresh], v[:fresh], q[:fresh]
        cache.append(k, v, None, None, batch)
        y = cache.attend(q, batch)
        assert torch.equal(data[:, 0], data[:, -1]) and (data[:, 0, :, :fresh] != 0).any()
        assert torch.equal(y[:fresh], y[fresh:]) and y.abs().max() > 0


@pytest.mark.parametrize("sequences, group", [([(3, 300), (1, 40), (2, 2)], 3), ([(60, 300), (1, 700), (33, 33)], 8)], ids=["few", "many"])
@pytest.mark.parametrize("bound", [1 << 28, 1 << 30])
def test_loose_bounds_on_new_tokens(serving, sequences, group, bound):
    """Bounds far above the tokens there are, whose rows 32 bits would not count."""
    p = Paged(serving, 61, sequences, 2, 256, 64, skip=1, behind=2)
    wide = torch.full((3, bound // 256), -1, dtype=torch.int32, device="cuda")
    wide[:, :p.batch.page_table.shape[1]] = p.batch.page_table
    p.batch = serving.PagedBatch(p.batch.starts, p.batch.lengths, wide, bound, bound)
    q, out = query(p, 2 * group, torch.float16)
    check_attention(serving, p, q, out, torch.float16)
    k, v = randn(p.g, p.tokens, 2, 64).half(), randn(p.g, p.tokens, 2, 64).half()
    before = p.arrays()
    p.cache.append(k, v, None, None, p.batch)
    want, want_scales = ref.append(*before, ref.f64(k), ref.f64(v), None, None, False)
    assert np.array_equal(p.scales.cpu().numpy(), want_scales, equal_nan=True) and np.array_equal(p.data.cpu().numpy(), want)


def test_page_table_of_a_larger_program_with_many_rows(serving):
    """The kernel for many rows over rows of a page table that are wider than needed, and lengths far below their bound."""
    p = Paged(serving, 52, [(1, 100), (30, 300), (1, 40)], 2, 16, 64)
    wide = torch.full((3, 1000), -1, dtype=torch.int32, device="cuda")
    wide[:, :p.batch.page_table.shape[1]] = p.batch.page_table
    p.batch = serving.PagedBatch(p.batch.starts, p.batch.lengths, wide, 40, 16000)
    check_attention(serving, p, *query(p, 8, torch.float16), torch.float16)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("mixed", [False, True], ids=["alone", "mixed"])
@pytest.mark.parametrize("tiny", [1e-40, 1e-38, 1e-36, 4e-35])
@pytest.mark.parametrize("sequences, group, d", [([(1, 200), (1, 1000), (1, 9)], 4, 128), ([(3, 700), (2, 40)], 2, 64), ([(1, 20000)], 8, 64),
                                                 ([(130, 700), (1, 30)], 4, 128), ([(40, 300)], 2, 256), ([(70, 5000)], 1, 128)])
def test_attention_with_the_smallest_value_scales(serving, sequences, group, d, tiny, mixed, dtype):
    """Pages whose values are next to nothing, as the append leaves them: alone, and among ordinary ones."""
    t = DTYPES[dtype]
    p = Paged(serving, group + d, sequences, 1, 16, d, wild=False)
    small = torch.rand(p.scales[1].shape, generator=p.g, device="cuda") < (0.6 if mixed else 2.0)
    p.scales[1, small] = tiny
    check_attention(serving, p, *query(p, group, t, 0.2), t)


def test_attention_over_many_keys_with_the_smallest_value_scales(serving):
    """Thousands of equal weights: their sum and the smallest scale together leave the normal numbers, the result does not."""
    p = Paged(serving, 71, [(33, 4000)] * 10, 8, 16, 16, wild=False)
    p.scales[1] = 1e-38
    q, out = query(p, 8, torch.bfloat16, 0.0)
    p.data[1] = p.data[1].abs() // 2 + 60
    check_attention(serving, p, q, out, torch.bfloat16)


@pytest.mark.parametrize("loud", [1e3, 1e8, 1e16, 1e24])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("sequences, group, d, how", [([(4, 34), (3, 18)], 2, 64, {}), ([(8, 40), (6, 90)], 2, 128, {"window": 20}), ([(4, 19), (2, 33)], 4, 256, {}),
                                                      ([(4, 20002), (1, 40)], 2, 64, {}), ([(100, 160), (40, 300)], 4, 128, {}), ([(90, 200)], 3, 64, {"window": 33}),
                                                      ([(40, 70)], 2, 256, {"softcap": 9.0}), ([(70, 5000)], 1, 128, {})], ids=str)
def test_attention_values_that_a_row_does_not_see(serving, sequences, group, d, how, dtype, loud):
    """Pages whose values are far larger than all others, hidden from some rows: those rows are as exact as without them."""
    t = DTYPES[dtype]
    p = Paged(serving, 91 + d, sequences, 1, 16, d, wild=False)
    q, out = query(p, group, t)
    want, bound = ref.attend(*p.arrays(), ref.f64(q), d ** -0.5, True, how.get("window", 0), how.get("softcap", 0.0), t)
    pages = [[0 if "window" in how else (length - 1) // 16] for length in p.lengths]  # behind a window, or in front of the causal mask
    for b, of in enumerate(pages):
        p.scales[1, [p.table[b][i] for i in of]] *= loud
    got = ref.f64(p.cache.attend(q, p.batch, out=out, **how))
    unseen = 0
    for b, length in enumerate(p.lengths):
        for i in range(p.starts[b], p.starts[b + 1]):
            position = length - p.starts[b + 1] + i
            lo = max(0, position - how["window"] + 1) if "window" in how else 0
            if not any(page * 16 <= position and page * 16 + 16 > lo for page in pages[b]):
                assert (np.abs(got[i] - want[i]) <= bound[i]).all(), (b, i, np.abs(got[i] - want[i]).max())
                unseen += 1
    assert unseen > 0


@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("sequences, group, d", [([(1, 40), (3, 24)], 2, 64), ([(1, 5000)], 1, 128), ([(40, 60), (70, 90)], 4, 128), ([(30, 40)], 1, 256),
                                                 ([(50, 3000)], 1, 64)])
@pytest.mark.parametrize("side", [0, 1], ids=["keys", "values"])
def test_attention_with_an_infinite_scale(serving, sequences, group, d, side, softcap):
    """What attends to a page whose scale is infinite is no number, whatever the page's integers are; the rest does not notice."""
    p = Paged(serving, 81 + d, sequences, 1, 16, d, wild=False)
    q, out = query(p, group, torch.float16)
    p.data[side, :, :, ::2] = 0
    if side == 0:
        p.data[0] = torch.where(p.data[0] == 0, p.data[0], 1)  # and scores of one sign, below zero
        q.copy_(-q.abs())
    want, bound = ref.attend(*p.arrays(), ref.f64(q), d ** -0.5, True, 0, softcap, torch.float16)
    for b, length in enumerate(p.lengths):  # the page of each sequence's last token
        p.scales[side, p.table[b][(length - 1) // 16]] = float("inf")
    got = ref.f64(p.cache.attend(q, p.batch, out=out, softcap=softcap))
    for b, length in enumerate(p.lengths):
        for i in range(p.starts[b], p.starts[b + 1]):
            if length - p.starts[b + 1] + i >= (length - 1) // 16 * 16:
                assert np.isnan(got[i]).all(), (b, i)
            else:
                assert (np.abs(got[i] - want[i]) <= bound[i]).all(), (b, i)


@pytest.mark.parametrize("cap", [1e-42, 1e-20, 0.01, 1.0, 50.0, 300.0, 1e4, 1e6, 1e7, 1e20, 3e38])
@pytest.mark.parametrize("sequences, group, d", [([(1, 200), (1, 40)], 4, 64), ([(3, 300)], 2, 128), ([(1, 50), (2, 90)], 3, 256), ([(1, 9000)], 2, 64),
                                                 ([(130, 300), (20, 40)], 4, 128), ([(30, 100)], 2, 256), ([(60, 2500)], 1, 64)])
def test_attention_with_caps_of_every_size(serving, sequences, group, d, cap):
    """Capped scores are as exact as scores without a cap, from caps far below the scores to caps far above them."""
    p = Paged(serving, 95 + d, sequences, 1, 16, d, wild=False)
    q, out = query(p, group, torch.float16, 4.0)
    got = ref.f64(p.cache.attend(q, p.batch, out=out, softcap=cap))
    want, bound = ref.attend_capped(*p.arrays(), ref.f64(q), d ** -0.5, cap, torch.float16)
    inside = ~np.isnan(want)
    wrong = ~(np.abs(got - want) <= bound) & inside
    assert not wrong.any(), (int(wrong.sum()), np.argwhere(wrong)[:4].tolist(), float(np.nanmax(np.where(inside, np.abs(got - want) / bound, 0))))


@pytest.mark.parametrize("bad", [[0], [2], [0, 1, 2, 3], [11]], ids=str)
@pytest.mark.parametrize("fresh, group, d", [(1, 2, 64), (3, 2, 128), (4, 4, 256), (30, 4, 64), (150, 2, 128), (40, 1, 256)])
def test_tokens_of_a_page_outside_the_cache_are_not_attended_to(serving, fresh, group, d, bad):
    """What is left of the sequence is attended to as if those tokens did not exist; a row that has nothing left gives zeros."""
    p = Paged(serving, 97 + d, [(fresh, 170), (fresh, 190)], 2, 16, d, wild=False)
    q, out = query(p, 2 * group, torch.float16)
    for i, page in enumerate(bad):
        p.batch.page_table[1, page] = (-1, p.data.shape[1], 1 << 30, -(1 << 31))[i]
    got = ref.f64(p.cache.attend(q, p.batch, out=out))
    assert serving.paged_error() == 2
    want, bound = ref.attend_capped(*p.arrays(), ref.f64(q), d ** -0.5, 0.0, torch.float16, missing={(1, page) for page in bad})
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("fresh", [1, 5, 150])
def test_rows_without_any_page_are_zeros(serving, fresh):
    p = Paged(serving, 98, [(fresh, 160), (fresh, 150)], 2, 16, 64, wild=False)
    q, out = query(p, 4, torch.float16)
    p.batch.page_table[0] = -1
    p.cache.attend(q, p.batch, out=out)
    assert serving.paged_error() == 2
    assert (out[:fresh] == 0).all() and (out[fresh:] != 0).any()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1])
def test_windows_beyond_32_bits_hide_nothing(serving, mlel, window):
    p = Paged(serving, 99, [(1, 60), (3, 40)], 1, 16, 64, wild=False)
    q, out = query(p, 2, torch.float16)
    want = p.cache.attend(q, p.batch)
    assert torch.equal(p.cache.attend(q, p.batch, window=window)[:4], want[:4])
    with pytest.raises(mlel.MlelError, match="not negative"):
        p.cache.attend(q, p.batch, window=-window)


@pytest.mark.parametrize("mode", ["ordinary", "tiny", "zero"])
@pytest.mark.parametrize("sequences, group, d, how", [([(4, 34), (3, 18)], 2, 64, {}), ([(8, 40), (6, 90)], 2, 128, {"window": 20}), ([(4, 19), (2, 33)], 4, 256, {}),
                                                      ([(4, 20002), (1, 40)], 2, 64, {}), ([(100, 160), (40, 300)], 4, 128, {}), ([(90, 200)], 3, 64, {"window": 33}),
                                                      ([(40, 70)], 2, 256, {"softcap": 9.0}), ([(70, 5000)], 1, 128, {}), ([(33, 600)] * 4, 1, 64, {"window": 150})], ids=str)
def test_attention_over_the_whole_range_of_value_scales(serving, sequences, group, d, how, mode):
    """One page of each sequence as large as bf16 allows, the others ordinary, next to nothing in part, or zeros in part: rows that do not
    see the large page are as exact as without it, and rows that do are its values."""
    t = torch.bfloat16
    p = Paged(serving, 101 + d, sequences, 1, 16, d, wild=False)
    q, out = query(p, group, t)
    small = torch.rand(p.scales[1].shape, generator=p.g, device="cuda") < (0.0 if mode == "ordinary" else 0.5)
    if mode != "ordinary":
        p.scales[1, small] = 1e-38 if mode == "tiny" else 0.0
    if mode == "zero":
        p.data[1, small[:, 0]] = 0
    windowed = lambda b: 0 if "window" in how else (p.lengths[b] - 1) // 16
    args = d ** -0.5, True, how.get("window", 0), how.get("softcap", 0.0), t
    without, bound_without = ref.attend(*p.arrays(), ref.f64(q), *args)
    for b in range(len(sequences)):
        p.scales[1, p.table[b][windowed(b)]] = 3e38 / 127 / 4
    got = ref.f64(p.cache.attend(q, p.batch, out=out, **how))
    want, bound = ref.attend(*p.arrays(), ref.f64(q), *args)
    unseen = 0
    for b, length in enumerate(p.lengths):
        for i in range(p.starts[b], p.starts[b + 1]):
            position = length - p.starts[b + 1] + i
            lo = max(0, position - how["window"] + 1) if "window" in how else 0
            if windowed(b) * 16 <= position and windowed(b) * 16 + 16 > lo:
                assert (np.abs(got[i] - want[i]) <= bound[i]).all(), (b, i)
            else:
                assert (np.abs(got[i] - without[i]) <= bound_without[i]).all(), (b, i, np.abs(got[i] - without[i]).max())
                unseen += 1
    assert unseen > 0
