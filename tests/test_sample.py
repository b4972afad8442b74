"""Sampling with settings per row: the oracle's rules and the refusals on the CPU; the kernel's ids against 64 bits on a GPU."""
import math

import numpy as np
import pytest
import torch

from flyingfish_b200 import ops
from flyingfish_b200.ops import sample_ops
from flyingfish_b200.ops.lib import KernelError

BF16, F32 = torch.bfloat16, torch.float32


def _row(logits, u, t, k, p, m):
    """The definition for one row, in 64 bits, with sums that do not depend on an order (math.fsum where it decides little, numpy otherwise)."""
    l = np.where(np.isnan(logits), -np.inf, logits)
    top = l.max()
    if top == -np.inf:
        return 0, 0.0
    if not t > 0:
        return int(np.argmax(l)), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        away = np.where(l == top, 0.0, (l - top) / t)
    w = np.where(away < -1000 * math.log(2.0), 0.0, np.exp(away))          # a mass below 2^-1000 of the largest counts as none, by the operator's definition
    order = np.lexsort((np.arange(len(l)), -l))
    n = len(l) if k <= 0 else min(k, len(l))
    if p < 1:
        sums = np.cumsum(w[order])
        n = min(n, int(np.searchsorted(sums, max(p, 0.0) * sums[-1], side="left")) + 1)
    if m > 0:
        n = min(n, int((away >= math.log(min(m, 1.0))).sum()))
    ids = np.sort(order[:n])
    sums = np.cumsum(w[ids])
    u = min(u, 1 - 2.0 ** -24) if u > 0 else 0.0
    at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), int(np.nonzero(w[ids])[0][-1]))
    return int(ids[at]), float(w[ids[at]] / sums[-1])


def _want(logits, u, t, k, p, m):
    l = logits.double().cpu().numpy()
    get = lambda v, i, other: other if v is None else v[i].item()
    rows = [_row(l[i], u[i].item(), t[i].item(), get(k, i, 0), get(p, i, 1.0), get(m, i, 0.0)) for i in range(len(l))]
    return torch.tensor([r[0] for r in rows], dtype=torch.int32), torch.tensor([r[1] for r in rows], dtype=torch.float64)


def _check(logits, u, t, k=None, p=None, m=None):
    ids, probs = sample_ops.sample_tokens(logits, u, t, k, p, m)
    want, want_p = _want(logits, u, t, k, p, m)
    bad = torch.nonzero(ids.cpu() != want).flatten().tolist()
    assert not bad, f"rows {bad[:5]}: {ids.cpu()[bad[:5]].tolist()} for {want[bad[:5]].tolist()}"
    # rounded once from a quotient whose parts are held to a few 1e-12; below 2^-126 numbers lie 2^-149 apart, so half a step is 2^-150 whatever the value
    assert ((probs.double().cpu() - want_p).abs() <= want_p * (2.0 ** -24 + 1e-11) + 2.0 ** -150).all()


def _settings(rows, seed, device):
    g = torch.Generator().manual_seed(seed)
    pick = lambda options, dtype: torch.tensor(options, dtype=dtype)[torch.randint(len(options), (rows,), generator=g)]
    t = pick([0.0, 0.3, 0.7, 1.0, 1.3, 2.0, 50.0], F32)
    k = pick([0, 0, 1, 2, 20, 50, 1000, 10 ** 6], torch.int32)
    p = pick([1.0, 1.0, 0.999, 0.9, 0.5, 0.1, 0.0], F32)
    m = pick([0.0, 0.0, 0.0, 0.001, 0.05, 0.5, 1.0], F32)
    return [v.to(device) for v in (torch.rand(rows, generator=g), t, k, p, m)]


def _logits(kind, rows, vocab, dtype, seed, device):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g)
    if kind == "peaked":
        x = x * 2.5
        x[torch.arange(rows)[:, None], torch.randint(vocab, (rows, 20), generator=g)] += 12 * torch.rand(rows, 20, generator=g)
    elif kind == "equal":
        x = torch.full((rows, vocab), 1.7)
    elif kind == "steps":
        x = torch.randint(0, 4, (rows, vocab), generator=g).float() * 0.5
    elif kind == "masked":
        x = torch.where(torch.rand(rows, vocab, generator=g) < 0.9, torch.tensor(float("-inf")), x * 3)
    elif kind == "lowest":
        x = torch.where(torch.rand(rows, vocab, generator=g) < 0.9, torch.finfo(dtype).min, x * 3)
    elif kind == "tiny":
        x = x * 1e-30
    elif kind == "wide":
        x = x * 200
    return x.to(dtype).to(device)


KINDS = ["normal", "peaked", "equal", "steps", "masked", "lowest", "tiny", "wide"]


# ------------------------------------------------------------------------------------------
# CPU
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
def test_oracle_against_the_definition(kind):
    _check(_logits(kind, 24, 301, F32, 1, "cpu"), *_settings(24, 2, "cpu"))


def test_rules():
    l = torch.tensor([[0.0, 2.0, 2.0, 1.0]]).log_softmax(-1)
    one = lambda u, t=1.0, k=0, p=1.0, m=0.0: sample_ops.sample_tokens(l, torch.tensor([u]), torch.tensor([t]), torch.tensor([k], dtype=torch.int32), torch.tensor([p]),
                                                                       torch.tensor([m]))[0].item()
    assert one(0.99, t=0.0) == 1 and one(0.99, k=1) == 1 and one(0.99, k=2) == 2 and one(0.49, k=2) == 1
    assert one(0.99, p=0.0) == 1 and one(0.0) == 0 and one(0.999999) == 3 and one(0.6, m=1.0) == 2 and one(float("nan")) == 0 and one(2.0) == 3
    none = sample_ops.sample_tokens(torch.full((1, 4), -math.inf), torch.tensor([0.5]), torch.tensor([1.0]))
    assert none[0].item() == 0 and none[1].item() == 0
    inf = torch.tensor([[1.0, math.inf, math.nan, math.inf]])
    assert [sample_ops.sample_tokens(inf, torch.tensor([u]), torch.tensor([1.0]))[0].item() for u in (0.4, 0.6)] == [1, 3]


def test_refusals():
    l, v = torch.zeros(2, 8), torch.zeros(2)
    for args in ((l.double(), v, v), (l, v.double(), v), (l, v[:1], v), (l, v, v, v), (l, v, v, None, v.int()), (l.t(), torch.zeros(8), torch.zeros(8)), (l[:, :0], v, v)):
        with pytest.raises(KernelError):
            sample_ops.sample_tokens(*args)
    assert sample_ops.sample_tokens(l[:0], v[:0], v[:0])[0].shape == (0,)


# ------------------------------------------------------------------------------------------
# GPU
# ------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (40, 301), (17, 4099), (64, 50257), (9, 128256)])
def test_ids_of_64_bits(cuda, rows, vocab, kind, dtype):
    _check(_logits(kind, rows, vocab, dtype, rows + vocab, cuda), *_settings(rows, vocab, cuda))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(500, 1000, BF16), (300, 32000, F32), (150, 151936, BF16), (2, 600001, BF16), (3, 300007, F32), (120, 262144, BF16)])
def test_many_rows_and_wide_rows(cuda, rows, vocab, dtype):
    _check(_logits("peaked", rows, vocab, dtype, 5, cuda), *_settings(rows, 6, cuda))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "peaked", "steps", "equal"])
def test_single_filters(cuda, kind):
    """Each filter by itself, with the others absent; numbers next to 0 and 1."""
    rows, vocab = 32, 20011
    for dtype in (BF16, F32):
        l = _logits(kind, rows, vocab, dtype, 11, cuda)
        u, t, k, p, m = _settings(rows, 12, cuda)
        t = t.clamp(min=0.5)
        u[0], u[1], u[2], u[3] = 0.0, 1.0 - 2.0 ** -24, 2.0 ** -24, 0.5
        for args in ((None, None, None), (k, None, None), (None, p, None), (None, None, m), (k, p, None)):
            _check(l, u, t, *args)


@pytest.mark.gpu
def test_layouts_and_special_values(cuda):
    rows, vocab = 12, 5003
    base = torch.full((rows, vocab + 9), 1e4, dtype=BF16, device=cuda)
    base[:, 3:3 + vocab] = _logits("peaked", rows, vocab, BF16, 1, cuda)
    s = _settings(rows, 3, cuda)
    _check(base[:, 3:3 + vocab], *s)                                     # rows that start off a 16-byte boundary, in a wider buffer
    assert torch.equal(sample_ops.sample_tokens(base[:, 3:3 + vocab], *s)[0], sample_ops.sample_tokens(base[:, 3:3 + vocab].contiguous(), *s)[0])
    for dtype in (BF16, F32):
        l = _logits("peaked", rows, vocab, dtype, 2, cuda)
        l[0], l[1, ::3], l[2, 7], l[3, 5], l[3, 4000] = -math.inf, math.nan, math.inf, math.inf, math.inf
        l[4, 1:] = -math.inf
        l[5] = math.nan
        u, t, k, p, m = s
        _check(l, u, torch.ones_like(t))
        _check(l, u, torch.ones_like(t), k, p, m)
        t = t.clone()
        t[6], t[7], t[8] = -1.0, math.nan, 1e-40
        p, m, u = p.clone(), m.clone(), u.clone()
        p[9], m[9], m[10], u[11] = math.nan, math.nan, 7.0, math.nan
        _check(l, u, t, k, p, m)
        _check(l, u, torch.full_like(t, math.inf).fill_(1e30), k, p, m)


@pytest.mark.gpu
def test_frequencies(cuda):
    """Numbers spread evenly over [0, 1) draw every token as often as its probability says: off by at most one."""
    l = _logits("peaked", 1, 200, F32, 4, cuda)
    n = 4096
    u = (torch.arange(n, device=cuda) / n).float()
    ids, _ = sample_ops.sample_tokens(l.expand(n, 200), u, torch.ones(n, device=cuda), torch.full((n,), 40, dtype=torch.int32, device=cuda))
    top = torch.topk(l[0].double(), 40)
    share = torch.zeros(200, dtype=torch.float64, device=cuda)
    share[top.indices] = torch.softmax(top.values, 0)
    seen = torch.bincount(ids.long(), minlength=200).double()
    assert ((seen - share * n).abs() < 1.0 + 1e-6).all()


@pytest.mark.gpu
def test_captured_and_on_another_stream(cuda):
    l = _logits("peaked", 33, 32003, BF16, 1, cuda)
    s = _settings(33, 1, cuda)
    sample_ops.sample_tokens(l, *s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, probs = sample_ops.sample_tokens(l, *s)
    for seed in (2, 3):
        l.copy_(_logits("normal", 33, 32003, BF16, seed, cuda))
        for v, w in zip(s, _settings(33, seed, cuda)):
            v.copy_(w)
        graph.replay()
        want, want_p = sample_ops.sample_tokens(l, *s)
        assert torch.equal(ids, want) and torch.equal(probs, want_p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = sample_ops.sample_tokens(l, *s)
    here = sample_ops.sample_tokens(l, *s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[0], here[0]) and torch.equal(other[1], here[1])


@pytest.mark.gpu
def test_refusals_on_the_device(cuda):
    l, v = torch.zeros(2, 8, device=cuda), torch.zeros(2, device=cuda)
    with pytest.raises(KernelError):
        sample_ops.sample_tokens(l, v.cpu(), v)
    with pytest.raises(KernelError):
        sample_ops.sample_tokens(torch.zeros(1, 2_000_000, device=cuda), v[:1], v[:1])       # more than a cluster's shared memory holds
    ops.check_status(cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["normal", "peaked", "steps"])
def test_long_prefixes_at_extreme_temperatures(cuda, kind, dtype):
    """Prefixes of more tokens than a list holds, whose last ones weigh nothing, next to nothing, or as much as the first."""
    rows, vocab = 24, 30011
    l = _logits(kind, rows, vocab, dtype, 21, cuda)
    f = lambda v: torch.tensor([v[i % len(v)] for i in range(rows)], device=cuda)
    for min_p in (None, f([0.0, 1e-30, 1e-3])):
        for top_p in (None, f([0.9999999, 1.0])):
            _check(l, f([0.0, 0.3, 0.99999, 0.7, 0.999999]), f([1e-6, 1e-3, 0.05, 1.0, 40.0, 1e6, 3e-39]), f([1500, 5000, 30010, 1025]).to(torch.int32), top_p, min_p)


@pytest.mark.gpu
def test_rows_that_no_shared_memory_holds_are_refused(cuda):
    one = lambda: torch.zeros(1, device=cuda)
    for vocab, dtype in ((786433, BF16), (393217, F32)):
        with pytest.raises(KernelError):
            sample_ops.sample_tokens(torch.zeros(1, vocab, dtype=dtype, device=cuda), one(), one())
        ids, p = sample_ops.sample_tokens(torch.zeros(1, vocab - 1, dtype=dtype, device=cuda), one() + 0.5, one() + 1)
        assert abs(int(ids[0]) - (vocab - 1) // 2) <= 1 and float(p[0]) == pytest.approx(1 / (vocab - 1), rel=1e-6)


def _zeros(rows, vocab, dtype, device):
    """Zeros of both signs among smaller logits."""
    g = torch.Generator().manual_seed(rows)
    pick = torch.randint(0, 4, (rows, vocab), generator=g)
    return torch.tensor([0.0, -0.0, -2.0, -0.5])[pick].to(dtype).to(device)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_zeros_of_both_signs_are_equal_for_the_oracle(dtype):
    l = torch.tensor([[-0.0, 0.0, -0.0, -1.0]], dtype=dtype)
    one = lambda u, k: sample_ops.sample_tokens(l, torch.tensor([u]), torch.tensor([1.0]), torch.tensor([k], dtype=torch.int32))[0].item()
    assert one(0.9, 1) == 0 and one(0.9, 2) == 1 and one(0.9, 3) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [4, 301, 50257])
def test_zeros_of_both_signs_are_equal(cuda, vocab, dtype):
    rows = 24
    l = _zeros(rows, vocab, dtype, cuda)
    f = lambda v, t=F32: torch.tensor([v[i % len(v)] for i in range(rows)], dtype=t, device=cuda)
    u, t = f([0.1, 0.5, 0.99, 0.0, 0.999]), f([1.0, 0.5])
    for k in (f([1, 2, 3, 5, 100, vocab // 3 + 1], torch.int32), None):
        for p in (f([0.3, 0.05, 0.9, 0.6]), None):
            ids, _ = sample_ops.sample_tokens(l, u, t, k, p)
            want, _ = _want(l, u, t, k, p, None)
            for r in torch.nonzero(ids.cpu() != want).flatten().tolist():
                # Weights 1, w, 1, w and the number 0.5: the half of the mass ends with a token, and 0.5 (2 + 2 w) against 1 + w is decided by the last bit of either sum.
                # Sums of n weights in 64 bits are off by n 2^-53 of themselves at most: within that the draw may fall on either side.
                low, high = sorted((int(ids[r]), int(want[r])))
                w = torch.exp((l[r].double().cpu() - l[r].double().cpu().max()) / float(t[r]))
                order = torch.argsort(l[r].double().cpu(), descending=True, stable=True)
                n = vocab if k is None else min(vocab, int(k[r]))
                if p is not None:
                    n = min(n, int((torch.cumsum(w[order], 0) < float(p[r]) * w.sum()).sum()) + 1)
                kept = torch.zeros_like(w)
                kept[order[:n]] = w[order[:n]]
                sums = torch.cumsum(kept, 0)
                assert kept[low] > 0 and kept[high] > 0 and not kept[low + 1: high].any(), (r, low, high)
                assert abs(sums[low] - float(u[r]) * sums[-1]) <= vocab * 2.0 ** -52 * sums[-1], (r, low, high)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("top", [25.0, 3e4, -7.5, 1e-3])
def test_neighbouring_numbers_at_temperatures_that_part_them(cuda, top, dtype):
    """Logits a step or a few below the largest, at temperatures where a step is from less than an octave to thousands of them."""
    rows, vocab = 30, 5003
    start = torch.tensor(top, dtype=dtype)
    steps = [start]
    for _ in range(6):
        steps.append(torch.nextafter(steps[-1], torch.tensor(-float("inf"), dtype=dtype)))
    gap = float(steps[0]) - float(steps[1])
    g = torch.Generator().manual_seed(3)
    l = torch.stack(steps)[torch.randint(0, 7, (rows, vocab), generator=g)].to(cuda)
    f = lambda v, t=F32: torch.tensor([v[i % len(v)] for i in range(rows)], dtype=t, device=cuda)
    t = f([gap * s for s in (1e-6, 1e-4, 4e-4, 7e-4, 1.1e-3, 1.44e-3, 1.6e-3, 3e-3, 0.1, 3.0)])
    u = f([0.0, 0.3, 0.999, 0.7, 0.9999999])
    for k, p in ((None, None), (f([3000, 700, 20], torch.int32), None), (None, f([0.9, 0.4])), (f([3000, 700, 20], torch.int32), f([0.9, 0.4]))):
        _check(l, u, t, k, p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(24, 4099), (140, 4099), (24, 9001), (9, 20011), (3, 128256)])
def test_borders_in_a_bin_of_many_tokens(cuda, rows, vocab, dtype):
    """One large logit far above thousands within a thousandth of one another: the border's bin holds them all, and is divided by key until a list holds what is left (FP32:
    thousands of keys) or one key is (BF16: a few). All CTAs of a row have to come to the same keys, each time."""
    g = torch.Generator().manual_seed(rows + vocab)
    l = torch.rand(rows, vocab, generator=g) * (1e-3 if dtype == F32 else 0.05) + 1.0
    l[torch.arange(rows), torch.randint(vocab, (rows,), generator=g)] = 31.0
    l = l.to(dtype).to(cuda)
    f = lambda v, t=F32: torch.tensor([v[i % len(v)] for i in range(rows)], dtype=t, device=cuda)
    u, t, k, p = torch.rand(rows, generator=g).to(cuda), f([50.0, 20.0, 100.0]), f([1500, vocab // 2, vocab - 1100, 2600], torch.int32), f([0.9, 0.55, 0.3])
    for args in ((k, None), (None, p), (k, p)):
        _check(l, u, t, *args)
        first = sample_ops.sample_tokens(l, u, t, *args)
        for _ in range(30):
            again = sample_ops.sample_tokens(l, u, t, *args)
            assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def _nearly_zero(rows, vocab, dtype, device):
    """Logits from 1e-28 down to subnormal ones, by rows, with zeros of both signs, values far below and masked ones among them."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g, dtype=torch.float64) * torch.tensor([1e-28, 1e-33, 1e-38, 1e-40, 1e-42, 0.0], dtype=torch.float64)[torch.arange(rows) % 6][:, None]
    what = torch.randint(0, 20, (rows, vocab), generator=g)
    for i, v in enumerate((0.0, -0.0, -1.0, -3e38, -math.inf)):
        x[what == i] = v
    x[torch.arange(rows) % 5 == 4, 7] = math.nan
    return x.to(F32).to(dtype).to(device)


def _freezing(rows, device):
    f = lambda v, t=F32: torch.tensor([v[i % len(v)] for i in range(rows)], dtype=t, device=device)
    return (f([0.0, 0.3, 0.999, 0.7, 0.9999999]), f([1e-25, 1e-29, 3e-31, 1e-35, 1e-40, 2e-42, 1e-45]),
            ((None, None, None), (f([40, 3, 2000], torch.int32), None, None), (None, f([0.9, 0.4]), None), (f([3000, 900, 20], torch.int32), f([0.97, 0.4]), f([0.0, 0.2, 1e-9]))))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_temperatures_next_to_zero_for_the_oracle(dtype):
    u, t, settings = _freezing(42, "cpu")
    for args in settings:
        _check(_nearly_zero(42, 301, dtype, "cpu"), u, t, *args)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [301, 5003, 60013])
def test_temperatures_next_to_zero(cuda, vocab, dtype):
    """Logits whose differences such temperatures still part: what is 2^-1000 of the largest counts as none, what is more has its weight."""
    u, t, settings = _freezing(42, cuda)
    for args in settings:
        _check(_nearly_zero(42, vocab, dtype, cuda), u, t, *args)


def _far_apart(rows, vocab, dtype, device):
    """Logits whose distance from the largest passes the largest number of their type, and infinite temperatures, which make them all alike."""
    g = torch.Generator().manual_seed(vocab + rows)
    low = torch.finfo(dtype).min
    x = torch.randn(rows, vocab, generator=g).clamp(-3, 3) * 1e38
    x = torch.where(torch.rand(rows, vocab, generator=g) < torch.tensor([0.9, 0.1, 0.5])[torch.arange(rows) % 3][:, None], torch.tensor(low), x)
    f = lambda v, t=F32: torch.tensor([v[i % len(v)] for i in range(rows)], dtype=t, device=device)
    t = f([math.inf, 1e38, 1.0, 3e38, 1e36, math.inf, 1e30])
    k, p = f([1500, vocab // 2, vocab - 40, 3001, 30], torch.int32), f([0.9, 0.6, 0.31])
    return x.to(dtype).to(device), f([0.3, 0.0, 0.777, 0.9999]), t, ((None, None, None), (k, None, None), (None, p, None), (k, p, f([0.0, 0.01, 0.2, 0.0])))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logits_far_apart_for_the_oracle(dtype):
    l, u, t, settings = _far_apart(24, 5003, dtype, "cpu")
    for args in settings:
        _check(l, u, t, *args)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [5003, 30011])
def test_logits_far_apart(cuda, vocab, dtype):
    l, u, t, settings = _far_apart(24, vocab, dtype, cuda)
    for args in settings:
        _check(l, u, t, *args)


@pytest.mark.gpu
def test_batches_on_two_streams_at_once(cuda):
    cases = [(_logits(kind, rows, 32003, BF16, 1, cuda), *_settings(rows, rows, cuda)) for kind, rows in (("normal", 40), ("peaked", 100))]
    want = [sample_ops.sample_tokens(*c) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[] for _ in cases]
    for _ in range(20):
        for s, c, out in zip(streams, cases, got):
            with torch.cuda.stream(s):
                out.append(sample_ops.sample_tokens(*c))
    torch.cuda.synchronize()
    for out, w in zip(got, want):
        assert all(torch.equal(o[0], w[0]) and torch.equal(o[1], w[1]) for o in out)
