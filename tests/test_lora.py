"""Adapters of many requests beside a projection: packing, refusals and the oracle on the CPU; the kernels against 64 bits on a GPU."""
import pytest
import torch

from flyingfish_b200 import ops
from flyingfish_b200.ops import lora_ops, ref
from flyingfish_b200.ops.lib import KernelError

BF16 = torch.bfloat16


def _case(m, k, n, r, count, seed=0, device="cpu", dtype=BF16, pad=0):
    g = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g)
    x = torch.zeros(m, k + pad, dtype=dtype)
    x[:, :k] = new(m, k)
    ranks = torch.tensor([(r, max(r // 2, 1), 0, 5)[i % 4] if count > 1 else r for i in range(count)], dtype=torch.int32)
    live = torch.arange(r)[None] < ranks[:, None]
    a = (new(count, r, k) * k ** -0.5 * live[:, :, None]).to(dtype)
    b = (new(count, n, r) * 0.1 * live[:, None]).to(dtype)
    scale = torch.rand(count, generator=g) + 0.5
    ids = torch.randint(-1, count, (m,), generator=g, dtype=torch.int32)
    to = lambda t: t.to(device)
    return to(x)[:, :k], to((new(n, k) * k ** -0.5).to(dtype)), lora_ops.AdapterStack(to(a), to(b), to(scale), to(ranks)), to(ids)


def _exact(x, w, st, ids):
    """(y, bound of a sum's error before the last rounding) in 64 bits. FP32 sums of 16-element instructions lose at most 2^-23 of the absolute sum per
    instruction and per partial sum that is joined; t is held to 2^-17 of itself."""
    x, w = x.double().cpu(), w.double().cpu()
    k, r = x.shape[1], st.a.shape[1]
    y, size = x @ w.T, (k / 16 + 64) * 2.0 ** -23 * (x.abs() @ w.abs().T)
    for i in range(st.a.shape[0]):
        rows = torch.nonzero(ids.cpu() == i).flatten()
        if rows.numel():
            a, b, s = st.a[i].double().cpu(), st.b[i].double().cpu(), float(st.scale[i])
            y[rows] += s * (x[rows] @ a.T) @ b.T
            size[rows] += ((k / 16 + r / 8 + 80) * 2.0 ** -23 + 2.0 ** -17) * s * (x[rows].abs() @ a.abs().T) @ b.abs().T
    return y, size


def _assert_near(got, y, size):
    got = got.double().cpu()
    off = (got - y).abs() - (size + (y.abs() + size) * 2.0 ** -8)
    assert torch.isfinite(got).all() and off.max() <= 0, f"{off.max():.3g} over the bound"


# ------------------------------------------------------------------------------------------
# CPU
# ------------------------------------------------------------------------------------------
def test_oracle_is_the_formula():
    x, w, st, ids = _case(37, 64, 48, 16, 5, dtype=torch.float32)
    y = lora_ops.linear_lora(x, w, st, ids)
    for r in range(37):
        want = w.double() @ x[r].double()
        if ids[r] >= 0:
            i = int(ids[r])
            want = want + float(st.scale[i]) * st.b[i].double() @ (st.a[i].double() @ x[r].double())
        assert torch.allclose(y[r].double(), want, rtol=1e-5, atol=1e-5)


def test_packed_parts_are_the_parts():
    """A fused projection's stack gives each part's own result, side by side and interleaved; missing parts give none."""
    g = torch.Generator().manual_seed(1)
    k, cols = 64, [256, 64, 64]
    mk = lambda c, r, s: (torch.randn(r, k, generator=g), torch.randn(c, r, generator=g), s)
    adapters = [[mk(256, 8, 2.0), None, mk(64, 20, 2.0)], [mk(256, 3, 0.5), mk(64, 17, 0.25), mk(64, 3, 0.5)], [None, None, None]]
    st = lora_ops.pack_stack(adapters, k, cols, "cpu", torch.float32)
    assert st.a.shape == (3, 96, k) and st.step == 32 and st.ranks.tolist() == [96, 96, 0] and st.part_of.tolist() == [0, 0, 0, 0, 1, 2]
    x = torch.randn(6, k, generator=g)
    ids = torch.tensor([0, 1, 2, -1, 1, 0], dtype=torch.int32)
    got = lora_ops.linear_lora(x, torch.zeros(384, k), st, ids)
    for r, i in enumerate(ids.tolist()):
        want = torch.cat([torch.zeros(c) if i < 0 or p is None else p[2] * (p[1] @ (p[0] @ x[r])) for p, c in zip(adapters[i], cols)])
        assert torch.allclose(got[r], want, rtol=1e-4, atol=1e-4)
    gate, up = mk(128, 8, 1.0), mk(128, 16, 1.0)
    st = lora_ops.pack_stack([[gate, up]], k, [128, 128], "cpu", torch.float32, interleave=True)
    got = lora_ops.linear_lora(x, torch.zeros(256, k), st, torch.zeros(6, dtype=torch.int32))
    want = [torch.cat([p[1] @ (p[0] @ x[r]) for p in (gate, up)]) for r in range(6)]
    want = torch.stack([ref.interleave_gate_up(v[:128, None], v[128:, None])[:, 0] for v in want])
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-4) and st.part_of.tolist() == [0, 1, 0, 1]
    # b is zero where a part's columns do not look
    for i, p in enumerate(st.part_of.tolist()):
        for s in range(st.a.shape[1] // st.step):
            if s % st.parts != p:
                assert not st.b[:, 64 * i: 64 * i + 64, st.step * s: st.step * (s + 1)].any()


def test_refusals():
    x, w, st, ids = _case(4, 64, 48, 16, 2)
    bad = [(st._replace(a=st.a[:, :, :56]), ids), (st._replace(b=st.b[:, :40]), ids), (st._replace(scale=st.scale.double()), ids),
           (st._replace(a=st.a[:, :8], b=st.b[:, :, :8]), ids), (st._replace(ranks=st.ranks.long()), ids), (st, ids.long()), (st, ids[:3]),
           (st._replace(b=st.b.float()), ids), (st._replace(a=st.a.transpose(0, 1).contiguous().transpose(0, 1)), ids),
           (st._replace(part_of=torch.zeros(0, dtype=torch.int32)), ids), (st._replace(part_of=torch.zeros(1, dtype=torch.int32), step=32), ids)]
    for stack, i in bad:
        with pytest.raises(KernelError):
            lora_ops.linear_lora(x, w, stack, i)
    part = (torch.randn(4, 64), torch.randn(48, 4), 1.0)
    for adapters, cols in (([], [48]), ([[part, part]], [48]), ([[(part[0], part[1][:40], 1.0)]], [48]), ([[(part[0] * float("inf"), part[1], 1.0)]], [48]),
                           ([[part, part]], [48, 48]), ([[(torch.zeros(1040, 64), torch.zeros(48, 1040), 1.0)]], [48])):
        with pytest.raises(KernelError):
            lora_ops.pack_stack(adapters, 64, cols, "cpu")


def test_a_stack_without_rows():
    x, w, st, ids = _case(0, 64, 48, 16, 2)
    assert lora_ops.linear_lora(x, w, st, ids).shape == (0, 48)


# ------------------------------------------------------------------------------------------
# GPU
# ------------------------------------------------------------------------------------------
SIZES = [(1, 64, 64, 16, 1), (1, 4096, 1000, 32, 3), (2, 72, 8, 16, 2), (7, 2048, 520, 48, 9), (31, 520, 384, 16, 40), (33, 4096, 256, 64, 4),
         (64, 1024, 4096, 16, 64), (100, 264, 200, 80, 7), (113, 512, 28672, 16, 5), (128, 4096, 6144, 16, 128), (128, 1032, 136, 256, 2),
         (129, 64, 64, 16, 3), (200, 2048, 1000, 32, 200), (257, 136, 72, 48, 2), (300, 4096, 512, 128, 6), (1000, 1024, 2048, 16, 3), (1500, 512, 264, 64, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,r,count", SIZES)
def test_against_64_bits(cuda, m, k, n, r, count):
    x, w, st, ids = _case(m, k, n, r, count, seed=m + n, device=cuda, pad=16 * (m % 3))
    y, size = _exact(x, w, st, ids)
    got = lora_ops.linear_lora(x, w, st, ids)
    _assert_near(got, y, size)
    bare = ids < 0
    assert torch.equal(got[bare], ops.linear(x, w)[bare])               # rows without an adapter: the product's own bits
    # requests of several rows each: tiles with one adapter, two, and none
    runs = torch.sort(ids).values
    y, size = _exact(x, w, st, runs)
    _assert_near(lora_ops.linear_lora(x, w, st, runs), y, size)
    wide = torch.zeros(m, n + 8, dtype=BF16, device=cuda)
    assert torch.equal(lora_ops.linear_lora(x, w, st._replace(ranks=None), runs, out=wide[:, :n]), lora_ops.linear_lora(x, w, st, runs))
    assert not wide[:, n:].any()
    for i in (-1, count - 1):
        same = torch.full_like(ids, i)
        y, size = _exact(x, w, st, same)
        _assert_near(lora_ops.linear_lora(x, w, st, same), y, size)
    ops.check_status(cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("m,r", [(128, 96), (120, 80), (97, 256), (128, 1024), (100, 1008), (300, 512)])
def test_an_adapter_for_every_row(cuda, m, r):
    """As many units as a tile can have: passes as wide as shared memory allows."""
    x, w, st, _ = _case(m, 256, 192, r, m, seed=r, device=cuda)
    ids = torch.arange(m, dtype=torch.int32, device=cuda).flip(0).contiguous()
    y, size = _exact(x, w, st, ids)
    _assert_near(lora_ops.linear_lora(x, w, st, ids), y, size)
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 64, 128, 300, 700])
def test_a_row_does_not_depend_on_its_neighbours(cuda, m):
    x, w, st, ids = _case(m, 1024, 768, 32, 6, seed=3, device=cuda)
    whole = lora_ops.linear_lora(x, w, st, ids)
    other = ids.clone()
    other[1:] = torch.randint(-1, 6, (m - 1,), device=cuda, dtype=torch.int32)
    assert torch.equal(lora_ops.linear_lora(x, w, st, other)[0], whole[0])
    if m <= 128:
        for row in (0, m // 2, m - 1):
            assert torch.equal(lora_ops.linear_lora(x[row: row + 1], w, st, ids[row: row + 1])[0], whole[row])
    # an adapter whose weights are not finite, and rows that are not, reach their own rows only
    st.a[1, 0, 0], st.b[2, 5, 1] = float("inf"), float("nan")
    x = x.clone()
    x[m // 2] = float("inf")
    got = lora_ops.linear_lora(x, w, st, ids)
    fine = (ids != 1) & (ids != 2)
    fine[m // 2] = False
    assert torch.equal(got[fine], whole[fine])


@pytest.mark.gpu
def test_ids_past_the_stack_are_reported(cuda):
    for m in (4, 200):
        x, w, st, ids = _case(m, 128, 64, 16, 3, device=cuda)
        ids[1] = 3
        got = lora_ops.linear_lora(x, w, st, ids)
        with pytest.raises(ops.DeviceStatusError):
            ops.check_status(cuda)
        assert torch.equal(got[1], ops.linear(x, w)[1])
        ids[1] = -7
        assert torch.equal(lora_ops.linear_lora(x, w, st, ids), got)
        ops.check_status(cuda)
        st.ranks[:] = 1000                                                   # ranks past the stack's are cut, negative ones are none
        full = lora_ops.linear_lora(x, w, st, ids)
        assert torch.equal(full, got)
        st.ranks[:] = -5
        assert torch.equal(lora_ops.linear_lora(x, w, st, ids), ops.linear(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 64, 128, 200, 600])
def test_fused_projections(cuda, m):
    """Gate and up with the activation, q / k / v with rotation and cache write: what the product and the separate kernels give."""
    g = torch.Generator().manual_seed(m)
    k, f, hq, hkv = 512, 384, 4, 2
    new = lambda *s: torch.randn(*s, generator=g)
    x = new(m, k).to(BF16).to(cuda)
    ids = torch.randint(-1, 3, (m,), generator=g, dtype=torch.int32).to(cuda)
    wgu = (new(2 * f, k) * k ** -0.5).to(BF16).to(cuda)
    part = lambda c, r: ((new(r, k) * k ** -0.5).to(BF16), (new(c, r) * 0.2).to(BF16), 1.0)
    gu = lora_ops.pack_stack([[part(f, 16), part(f, 8)], [part(f, 24), None], [None, part(f, 16)]], k, [f, f], cuda, interleave=True)
    y, size = _exact(x, wgu, gu, ids)
    _assert_near(lora_ops.linear_lora(x, wgu, gu, ids), y, size)
    _assert_near(lora_ops.linear_lora(x, wgu, gu._replace(part_of=None), ids), y, size)
    for mode, limit in ((0, 0.0), (3, 0.0), (5, 1.5), (1, 0.0)):
        got = lora_ops.linear_swiglu_lora(x, wgu, gu, ids, mode=mode, limit=limit)
        want = ops.silu_mul_interleaved(lora_ops.linear_lora(x, wgu, gu, ids), None, mode, limit).double()
        # Either way rounds gate g, up u, the activation and the result to BF16 at most once each: with |act(g)| <= |g| and |act'| <= 1.2 that is at
        # most 2^-8 |g| (|u| + 1) (1.2 + 1 + 1 + 1) for each of the two, second orders included in 9 for both
        near = (y.abs() + 8 * size).view(m, f // 64, 2, 64)
        bound = 2.0 ** -8 * 9 * (near[:, :, 0] * (near[:, :, 1] + 1)).reshape(m, f)
        assert ((got.double() - want).abs().cpu() <= bound).all(), mode
        assert torch.equal(got[ids < 0], ops.linear_swiglu(x, wgu, mode=mode, limit=limit)[ids < 0])
    d, n = 128, (hq + 2 * hkv) * 128
    wqkv = (new(n, k) * k ** -0.5).to(BF16).to(cuda)
    qkv = lora_ops.pack_stack([[part(hq * d, 16), part(hkv * d, 8), part(hkv * d, 16)], [part(hq * d, 32), None, part(hkv * d, 4)], [None, None, None]], k,
                              [hq * d, hkv * d, hkv * d], cuda)
    positions = torch.arange(m, dtype=torch.int32, device=cuda)
    slots = torch.randperm(16 * 64, generator=g)[:m].to(torch.int32).to(cuda)
    slots[m // 2] = -1
    caches = lambda: [torch.zeros(16, hkv, 64, d, dtype=BF16, device=cuda) for _ in range(2)]
    kc, vc = caches()
    got = lora_ops.linear_rope_kv_lora(x, wqkv, qkv, ids, positions, slots, kc, vc, hq, hkv, d, 1e4)
    ka, va = caches()
    apart = lora_ops.linear_lora(x, wqkv, qkv, ids)
    ops.rope_kv_paged(apart, positions, slots, ka, va, hq, hkv, d, 1e4)
    # the two products may split K differently: one rounding's difference, turned (two terms) and rounded three times
    for one, two in ((got, apart), (kc, ka), (vc, va)):
        bound = 2.0 ** -8 * 8 * two.double().abs().max()
        assert ((one.double() - two.double()).abs() <= bound).all() and (one != two).double().mean() < 0.2
    kb, vb = caches()
    plain = ops.linear_rope_kv(x, wqkv, positions, slots, kb, vb, hq, hkv, d, 1e4)
    assert torch.equal(got[ids < 0], plain[ids < 0])
    ops.check_status(cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [8, 200])
def test_captured_and_on_other_streams(cuda, m):
    x, w, st, ids = _case(m, 512, 1024, 16, 8, seed=5, device=cuda)
    x, w = x.clone(), w.clone()
    first = lora_ops.linear_lora(x, w, st, ids)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        mid = lora_ops.linear_lora(x, w, st, ids)
        out = lora_ops.linear_lora(mid[:, :512], w, st, ids)
    for seed in (7, 8):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(m, 512, generator=g))
        ids.copy_(torch.randint(-1, 8, (m,), generator=g, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, lora_ops.linear_lora(lora_ops.linear_lora(x, w, st, ids)[:, :512], w, st, ids))
    g = torch.Generator().manual_seed(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = lora_ops.linear_lora(x, w, st, ids)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, lora_ops.linear_lora(x, w, st, ids)) and first.shape == other.shape
    ops.check_status(cuda)


@pytest.mark.gpu
def test_refusals_on_the_device(cuda):
    x, w, st, ids = _case(4, 64, 48, 16, 2, device=cuda)
    for args in ((x.float(), w, st, ids), (x, w.float(), st, ids), (x, w, st, ids.cpu()), (x, w, st._replace(scale=st.scale.cpu()), ids), (x, w[:, :56], st, ids)):
        with pytest.raises(KernelError):
            lora_ops.linear_lora(*args)
    with pytest.raises(KernelError):
        lora_ops.linear_lora(x, w, st, ids, out=torch.zeros(4, 40, dtype=BF16, device=cuda))
    x, w, st, ids = _case(200, 64, 44, 16, 2, device=cuda)                   # prompts' products want columns in eights, as ops.linear does
    with pytest.raises(KernelError):
        lora_ops.linear_lora(x, w, st, ids)
    ops.check_status(cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 7, 64, 113, 200, 300, 600])
def test_inputs_written_just_before(cuda, m):
    """X and the ids come from kernels that end just before the call, over and over into the same memory, eagerly and replayed: every call reads its own. Some calls
    have rows without adapters only, or a stack none of whose live steps has columns."""
    k, n, count = 1024, 1536, 5
    _, w, st, _ = _case(m, k, n, 32, count, seed=m, device=cuda)
    blind = st._replace(part_of=torch.ones(n // 64, dtype=torch.int32, device=cuda), parts=2, step=16, ranks=torch.full_like(st.ranks, 16))
    g = torch.Generator().manual_seed(m)
    rounds = 24
    raw = torch.randn(rounds, m, k, generator=g).to(BF16).to(cuda)
    who = torch.randint(-1, count, (rounds, m), generator=g, dtype=torch.int32)
    who[::5] = -1
    who = who.to(cuda)
    gain = torch.ones(k, dtype=BF16, device=cuda)
    stacks = [blind if i % 7 == 3 else st for i in range(rounds)]
    want = []
    for i in range(rounds):
        x = ops.rmsnorm(raw[i], gain, 1e-6)
        torch.cuda.synchronize()
        want.append(lora_ops.linear_lora(x, w, stacks[i], who[i]))
        torch.cuda.synchronize()
    x, ids = torch.empty(m, k, dtype=BF16, device=cuda), torch.empty(m, dtype=torch.int32, device=cuda)

    def run():
        out = []
        for i in range(rounds):
            ids.copy_(who[i])
            x.copy_(ops.rmsnorm(raw[i], gain, 1e-6))
            out.append(lora_ops.linear_lora(ops.rmsnorm(x, gain, 0.0) if i % 2 else x, w, stacks[i], ids))
            x.fill_(float("nan"))                        # behind the call
            ids.fill_(0)
        return out
    again = [lora_ops.linear_lora(ops.rmsnorm(ops.rmsnorm(raw[i], gain, 1e-6), gain, 0.0), w, stacks[i], who[i]) if i % 2 else want[i] for i in range(rounds)]
    torch.cuda.synchronize()
    for i, y in enumerate(run()):
        assert torch.equal(y, again[i]), i
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        graph.replay()
        for i, y in enumerate(out):
            assert torch.equal(y, again[i]), i
    ops.check_status(cuda)


def _parts_of_several_scales(k, cols, scales, device, seed=0):
    """One adapter of rank 1 per scale set, whose A picks element 3 of x."""
    g = torch.Generator().manual_seed(seed)
    pick = torch.zeros(1, k)
    pick[0, 3] = 1.0
    return [[None if s is None else (pick.to(BF16), torch.randn(c, 1, generator=g).to(BF16), s) for c, s in zip(cols, row)] for row in scales]


def test_no_matrix_takes_a_scale_into_itself():
    cols, scales = [128, 64, 64], [(1.0, 41 / 32, 0.7), (0.3, 0.3, None), (None, None, None), (0.0, 2.0, 1e-3)]
    parts = _parts_of_several_scales(64, cols, scales, "cpu")
    for stack, one in ((lora_ops.pack_stack(parts, 64, cols, "cpu"), False), (lora_ops.pack_stack(parts[1:3], 64, cols, "cpu"), True)):
        assert stack.scale.shape == ((2,) if one else (4, stack.a.shape[1]))
        for i, row in enumerate(parts[1:3] if one else parts):
            at = 0
            for j, p in enumerate(row):
                if p is not None:
                    assert torch.equal(stack.b[i, at: at + cols[j], j * stack.step], p[1][:, 0])
                    s = stack.scale[i] if one else stack.scale[i, j * stack.step]
                    assert float(s) == pytest.approx(p[2], rel=2.0 ** -24)
                at += cols[j]
    from flyingfish_b200.loaders.adapters import _one_part
    small = [[(torch.ones(1, 8, dtype=BF16), torch.tensor([[1.1], [0.3]]).to(BF16), s) for s in row] for row in ((0.7, 0.9), (0.7, 0.7))]
    stack = lora_ops.pack_stack(_one_part(small, [2, 2]), 8, [4], "cpu")
    assert torch.equal(stack.b[:, :2, 0], stack.b[:, 2:, 1]) and torch.equal(stack.b[0, :2, 0], small[0][0][1][:, 0])
    assert stack.scale[0, :2].tolist() == torch.tensor([0.7, 0.9]).tolist() and stack.scale[1, :2].tolist() == torch.tensor([0.7, 0.7]).tolist()
    with pytest.raises(KernelError):                     # what BF16 has no number for
        lora_ops.pack_stack([[(torch.full((1, 8), 3.4e38), torch.ones(2, 1), 1.0)]], 8, [2], "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 128, 200, 600])
@pytest.mark.parametrize("adapters", [3, 200])
def test_scales_of_parts_cost_no_rounding(cuda, m, adapters):
    """Rank-1 adapters of one element x, so that a delta is B s x with 8 + 6 + 8 bits: rounded once, it is within half a step of BF16 (and what FP32 sums of the two
    words of t leave, 2^-22 of itself). B rounded with its scale first would be off by up to a whole step."""
    k, cols = 64, [256, 128, 128]
    sets = [(1.0, 41 / 32, 25 / 32), (37 / 32, 1.0, None), (0.5, 0.5, 0.5)]
    stack = lora_ops.pack_stack(_parts_of_several_scales(k, cols, [sets[i % 3] for i in range(adapters)], cuda, m), k, cols, cuda)
    assert stack.scale.dim() == 2
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, k, generator=g).to(BF16).to(cuda)
    ids = torch.randint(-1, adapters, (m,), generator=g, dtype=torch.int32).to(cuda)
    got = lora_ops.linear_lora(x, torch.zeros(sum(cols), k, dtype=BF16, device=cuda), stack, ids).double()
    a, b, s = stack.a.double(), stack.b.double(), stack.scale.double()
    safe = ids.long().clamp(min=0)
    t = s[safe] * torch.einsum("mk,mrk->mr", x.double(), a[safe])
    want = torch.einsum("mr,mnr->mn", t, b[safe]) * (ids >= 0)[:, None]
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=1e-30))) - 7)
    assert ((got - want).abs() <= step / 2 * (1 + 2.0 ** -12)).all()
    ops.check_status(cuda)


@pytest.mark.gpu
def test_prompts_on_two_streams_at_once(cuda):
    """Calls of more than 128 rows share nothing: each has its own t and its own word behind it."""
    cases = [_case(m, 1024, 1536, 32, 5, seed=m, device=cuda) for m in (300, 200, 700)]
    want = [lora_ops.linear_lora(*c) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[] for _ in cases]
    for _ in range(20):
        for s, c, out in zip(streams, cases, got):
            with torch.cuda.stream(s):
                out.append(lora_ops.linear_lora(*c))
    torch.cuda.synchronize()
    for out, w in zip(got, want):
        assert all(torch.equal(o, w) for o in out)
    ops.check_status(cuda)
