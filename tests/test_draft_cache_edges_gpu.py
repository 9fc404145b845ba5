"""Edges of the operators of a cache that is drafted into and thinned out, against plain forms in 64 bits."""
import math
import random

import pytest
import torch

from tests import test_draft_cache_gpu as G
from tests.plain import draft_cache_plain as P
from tests.test_draft_cache_gpu import DTYPES, Requests, check_rows, dev, i32, run_mass, run_tree, spread_mask, tree_sees, trees

pytestmark = pytest.mark.gpu
ops = G.ops


def same_mass(r, mass):
    """Sums of weights, NaN and infinite ones among them, against 64 bits (the bound of check_mass)."""
    for s, n in enumerate(r.rows):
        q, k, v = r.of(s)
        sees = torch.cat([torch.ones((n, r.held[s]), dtype=torch.bool), torch.ones((n, n), dtype=torch.bool).tril()], 1)
        _, w = P.attention(q, k, v, sees, r.scale)
        sums = w.reshape(r.hkv, -1, w.shape[-1]).sum(1)
        have = mass[:, r.slots[s]].double()
        assert torch.equal(have.isnan(), sums.isnan()), (s, have.isnan().sum(), sums.isnan().sum())
        fine = ~sums.isnan()
        rel = 2 * P.score_error(q, k, r.scale) + (n * r.hq // r.hkv + len(r.slots[s]) + 16) * 2.0 ** -24 + 2.0 ** -20
        assert bool(((have - sums).abs()[fine] <= rel * sums[fine]).all()), s


def causal(r):
    return [torch.cat([torch.ones((n, h), dtype=torch.bool), torch.ones((n, n), dtype=torch.bool).tril()], 1) for h, n in zip(r.held, r.rows)]


@pytest.fixture
def rows_at_once(monkeypatch):
    """The plain attention without its loop over rows, for values that are finite (a masked score is replaced, whatever it is)."""

    def attention(q, k, v, sees, scale):
        q, k, v = q.double(), k.double(), v.double()
        assert bool(v.isfinite().all())
        kk, vv = (x.repeat_interleave(q.shape[1] // k.shape[1], 1).transpose(0, 1) for x in (k, v))
        x = torch.where(sees, q.transpose(0, 1) @ kk.transpose(1, 2) * scale, -math.inf)
        weights = torch.where(sees.any(1)[:, None], torch.softmax(x, -1), 0.0)
        return (weights @ vv).transpose(0, 1), weights

    monkeypatch.setattr(P, "attention", attention)


HEADS = [(14, 2, 64), (12, 2, 128), (3, 1, 32), (8, 8, 64)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [1, 37, 200, 3]], ids=["single", "portions"])
def test_rows_that_score_minus_infinity_everywhere(ops, rows_at_once, dtype, heads, rows):
    """A row that sees keys and scores minus infinity with all of them has no softmax: NaN in its result and in what its keys receive, as
    in 64 bits.  The others are as ever; a head of queries that looks the other way sees plus infinity, which is NaN as well."""
    held = [0, 5, 700, 130]
    r = Requests(held, rows, heads, dtype, 16, 201)
    r.q[:, :, 0] = r.q[:, :, 0].abs() + 0.5
    for s in (0, 2):
        r.k[r.slots[s], 0, 0] = -math.inf          # the first kv head of two requests
    got, mass = run_mass(ops, r, None)
    check_rows(r, got, causal(r))
    same_mass(r, mass)
    nan = mass[:, r.slots[2]].isnan()
    assert bool(nan[0].all()) and not bool(nan[1:].any())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_drafted_rows_that_score_minus_infinity_everywhere(ops, rows_at_once, dtype, heads):
    """In a tree, too, whether its request holds keys or not; a row without any key to see is zeros beside them."""
    r = Requests([0, 0, 900, 31], [7, 150, 20, 5], heads, dtype, 16, 202)
    mask = spread_mask(ops, r, trees(random.Random(1), r.rows))
    empty = [r.first[0] + 3, r.first[1] + 9, r.first[1] + 140]
    mask[empty] = 0
    r.q[:, :, 0] = r.q[:, :, 0].abs() + 0.5
    for s in (0, 1, 2):
        r.k[r.slots[s], 0, 0] = -math.inf
    got = run_tree(ops, r, mask)
    check_rows(r, got, tree_sees(r, mask))
    group = r.hq // r.hkv
    for s in (0, 1, 2):
        rows = [i for i in range(r.first[s], r.first[s] + r.rows[s]) if i not in empty]
        assert bool(got[rows, :group].isnan().all())
    assert bool((got[empty] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", HEADS + [(28, 4, 128), (5, 1, 64), (43, 1, 64)], ids=str)
@pytest.mark.parametrize("held,n", [(0, 300), (500, 130), (900, 1)])
def test_a_key_that_scores_minus_infinity(ops, rows_at_once, dtype, heads, held, n):
    """It receives nothing from any row (nothing, not a NaN), and changes nothing else."""
    r = Requests([held, 40], [n, 3 if n > 1 else 1], heads, dtype, 16, 203)
    r.q[:, :, 1] = r.q[:, :, 1].abs() + 0.5
    at = [2 if n > 1 or held else 0, (held + n) // 2] if held + n > 3 else []
    r.k[[r.slots[0][j] for j in at], :, 1] = -math.inf
    got, mass = run_mass(ops, r, None)
    # (a portion's rows that see only such keys have none here: key 0 is a common one)
    check_rows(r, got, causal(r))
    same_mass(r, mass)
    assert bool((mass[:, [r.slots[0][j] for j in at]] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(3, 1, 64), (4, 2, 128), (5, 1, 20)], ids=str)
def test_single_tokens_behind_many_bad_pages(ops, dtype, heads):
    """A table may name more places outside the cache than the cache has rows: the keys that there are receive their weights all the same."""
    hq, hkv, hd = heads
    page, S, held = 16, 3, [1500, 77, 2303]
    g = torch.Generator().manual_seed(204)
    slots = 8 * page
    k, v = (torch.randn((slots, hkv, hd), generator=g).to(dtype) for _ in range(2))
    q = torch.randn((S, hq, hd), generator=g).to(dtype)
    table = [[-1] * 150 for _ in range(S)]
    good = {0: {3: 5, 80: 0, 93: 7}, 1: {0: 1, 4: 2}, 2: {60: 3, 143: 6, 142: 4}}
    for s, pages in good.items():
        for at, p in pages.items():
            table[s][at] = p
    mass_in = torch.rand((hkv, slots), generator=g)
    mass, out = torch.full((hkv, slots), -5.0, device=dev()), torch.full((S, hq * hd), 7.0, dtype=dtype, device=dev())
    ops.paged_attention_mass(q.reshape(S, -1).to(dev()), k.to(dev()), v.to(dev()), out, mass, i32([0, 1, 2]), i32([1] * S), i32(held), i32(table), page,
                             hq, hkv, hd, hd ** -0.5, 1, mass_in=mass_in.to(dev()))
    ops.check_async_errors(dev())
    have, out = mass.cpu().double(), out.cpu().double().reshape(S, hq, hd)
    for s in range(S):
        kk, vv = (torch.zeros((held[s] + 1, hkv, hd), dtype=dtype) for _ in range(2))
        here = {}
        for at, p in good[s].items():
            for o in range(page):
                if at * page + o <= held[s]:
                    kk[at * page + o], vv[at * page + o] = k[p * page + o], v[p * page + o]
                    here[at * page + o] = p * page + o
        want, w = P.attention(q[s:s + 1], kk, vv, torch.ones((1, held[s] + 1), dtype=torch.bool), hd ** -0.5)
        sums = w.reshape(hkv, -1, w.shape[-1]).sum(1)
        rel = 2 * P.score_error(q[s:s + 1], kk, hd ** -0.5) + (hq // hkv + held[s] + 17) * 2.0 ** -24 + 2.0 ** -20
        for j, slot in here.items():
            before = mass_in[:, slot].double() if j < held[s] else 0.0
            assert bool(((have[:, slot] - before - sums[:, j]).abs() <= rel * sums[:, j] + 2.0 ** -23 * before).all()), (s, j)
        # (a bf16 result's bound as in Requests.tolerance)
        top = float(vv.double().abs().max())
        step = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
        assert bool(((out[s] - want[0]).abs() <= (rel + (step if dtype == torch.bfloat16 else 0.0)) * top + step * want[0].abs()).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_scratch_goes_by_what_the_requests_can_hold(ops, dtype):
    """One token behind few keys in a pool of two million rows: its call asks for no memory in proportion to the pool."""
    hq, hkv, hd, page, slots = 16, 1, 64 if dtype == torch.bfloat16 else 8, 16, 1 << 21
    k, v = (torch.zeros((slots, hkv, hd), dtype=dtype, device=dev()) for _ in range(2))
    q, out = torch.ones((1, hq * hd), dtype=dtype, device=dev()), torch.zeros((1, hq * hd), dtype=dtype, device=dev())
    mass = torch.full((hkv, slots), -5.0, device=dev())
    table = i32([[slots // page - 1 - i for i in range(40)]])
    args = (i32([0]), i32([1]), i32([600]), table, page, hq, hkv, hd, hd ** -0.5, 1)
    ops.paged_attention_mass(q, k, v, out, mass, *args)          # (the flag of errors and the like are there afterwards)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    ops.paged_attention_mass(q, k, v, out, mass, *args)
    torch.cuda.synchronize()
    # scores of at most 640 places and the pieces' ends, partial results of up to 512 blocks of two parts of 128 rows (of bf16 heads; 16
    # rows of float32) and their maxima
    rows = 256 if dtype == torch.bfloat16 else 64
    bound = 4 * (2 * 512 * rows * (hd + 4) + 2 * 512 * 128 + (640 + 4 * 128 * 5) * hq + 65536)
    assert torch.cuda.max_memory_allocated() - before <= bound
    assert torch.cuda.max_memory_allocated() - before < 4 * slots * hq // 2
    slots_of = torch.tensor([int(table[0, j // page]) * page + j % page for j in range(601)])
    weights = mass.cpu()[0, slots_of].double()
    assert torch.allclose(weights, torch.full_like(weights, hq / 601), rtol=1e-5)
    assert int((mass != -5.0).sum()) == 601


def test_results_over_other_memory_of_a_call(ops):
    """Refused, with nothing written; memory that lies side by side is fine."""
    r = Requests([40, 7], [3, 5], (4, 2, 64), torch.float32, 16, 205)
    q, k, v = r.q.reshape(r.T, -1).to(dev()), r.k.to(dev()), r.v.to(dev())
    want, sums = run_mass(ops, r, None)
    planes = torch.full((3 * r.hkv * r.num_slots,), -5.0, device=dev())
    plane = lambda at: planes[at:at + r.hkv * r.num_slots].view(r.hkv, r.num_slots)  # noqa: E731
    n = r.hkv * r.num_slots
    out = torch.full_like(q, 7.0)
    for at in (1, n - 1):
        with pytest.raises(ops.KernelError, match="mass must not lie over mass_in"):
            ops.paged_attention_mass(q, k, v, out, plane(at), *r.args(), 5, mass_in=plane(0))
    with pytest.raises(ops.KernelError, match="out must not lie over k_cache"):
        ops.paged_attention_mass(q, k, v, k.view(-1)[:q.numel()].view_as(q), plane(0), *r.args(), 5)
    mask = spread_mask(ops, r, trees(random.Random(1), r.rows)).to(dev())
    with pytest.raises(ops.KernelError, match="out must not lie over v_cache"):
        ops.tree_attention(q, k, v, v.view(-1)[-q.numel():].view_as(q), mask, *r.args())
    assert bool((out == 7.0).all()) and bool((planes == -5.0).all())
    plane(0).zero_()
    ops.paged_attention_mass(q, k, v, out, plane(n), *r.args(), 5, mass_in=plane(0))          # side by side
    assert torch.equal(out.cpu().view_as(want), want) and torch.equal(plane(n).cpu(), sums) and bool((planes[2 * n:] == -5.0).all())
    # two layers of weights, written one layer further on
    kl, vl = (x.expand(2, *x.shape).contiguous() for x in (k, v))
    mass, pos = torch.rand((3, r.hkv, r.num_slots), device=dev()), torch.zeros((3, r.hkv, r.num_slots), dtype=torch.int32, device=dev())
    spans = r.spans()
    before = [x.clone() for x in (kl, vl, mass, pos)]
    with pytest.raises(ops.KernelError, match="mass_out must not lie over mass"):
        ops.cache_evict(kl, vl, mass[:2], pos[:2], i32([43, 12]), i32([43, 12]), spans[3], 16, 10, 0, 0, mass_out=mass[1:], positions_out=pos[1:])
    ids = i32([0] * r.T)
    path, count = i32([[0] * 4] * 2), i32([0, 0])
    with pytest.raises(ops.KernelError, match="next_token must not lie over tokens"):
        ops.tree_commit(ids, ids.clone(), ids.clone(), kl, vl, *spans, 16, path, count, ids[:2])
    with pytest.raises(ops.KernelError, match="k_cache must not lie over v_cache"):
        ops.tree_commit(ids, ids.clone(), ids.clone(), kl.view(-1, 2, 64)[:-1], kl.view(-1, 2, 64)[1:], *spans, 16, path, count, i32([0, 0]))
    assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip((kl, vl, mass, pos), before))


def decode(ops, q, k, v, out, pos, table, page, heads, fresh, nsplit=4):
    hq, hkv, hd = heads
    S = q.shape[0]
    iota, zeros = i32(list(range(S))), i32([0] * S)
    return lambda f=fresh: ops.paged_decode_mma(q, k, v, out, iota, zeros, S, iota, pos, table, table.shape[1], page, hq, hkv, hd, 0, hd ** -0.5, nsplit, None,
                                                fresh=f)


@pytest.mark.parametrize("held", [1500, 5000], ids=["registers", "large tables"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)], ids=str)
def test_a_decode_step_right_behind_an_eviction(ops, heads, held):
    """Decode attention asks for the keys of earlier steps before it waits for the launch before it: the moved ones are there, eager and
    from a graph."""
    hq, hkv, hd = heads
    S, page, budget = 24, 16, 1024
    r, k, v, mass, pos, ends = evict_inputs(held, S, heads, page)
    k0, v0, m0, p0 = (x.to(dev()) for x in (k, v, mass, pos))
    k1, v1, m1, p1 = (torch.empty_like(x) for x in (k0, v0, m0, p0))
    q = torch.randn((S, hq * hd), generator=torch.Generator().manual_seed(207)).bfloat16().to(dev())
    out, table, lengths, end = torch.zeros_like(q), r.spans()[3], i32([held] * S), i32(ends)
    step = decode(ops, q, k1, v1, out, i32([budget - 1] * S), table, page, heads, 1)

    def run():
        for a, b in ((k1, k0), (v1, v0), (m1, m0), (p1, p0)):
            a.copy_(b)
        ops.cache_evict(k1, v1, m1, p1, lengths, end, table, page, budget, 4, 100)

    run()
    torch.cuda.synchronize()
    step(0)
    torch.cuda.synchronize()
    want, rows = out.clone(), k1.clone()
    assert not torch.equal(rows, k0)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run()
        step()
    for i in range(40):
        out.zero_()
        if i % 2:
            graph.replay()
        else:
            run()
            step()
        torch.cuda.synchronize()
        assert torch.equal(k1, rows) and torch.equal(out, want), i


def evict_inputs(held, S, heads, page):
    r, k, v, mass, pos, ends = G.evict_case([held] * S, heads, torch.bfloat16, page, 0, 206)
    return r, k[0].contiguous(), v[0].contiguous(), mass[0].contiguous(), pos[0].contiguous(), ends


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)], ids=str)
def test_a_decode_step_right_behind_a_commit(ops, heads):
    """The same of confirmed drafted tokens: every other node of a long chain moves up, over several tiles of keys."""
    hq, hkv, hd = heads
    S, page, n, held = 24, 16, 400, 300
    r = Requests([held] * S, [n] * S, heads, torch.bfloat16, page, 208, gap=0)
    parents = [-1] + [max(0, i - 2) for i in range(1, n)]
    tokens, targets = [i % 2 for i in range(n)], [0] * n          # (even nodes go on with even ones)
    flat = [i32(x * S) for x in (tokens, parents, targets)]
    k0, v0 = r.k.to(dev()), r.v.to(dev())
    k1, v1 = torch.empty_like(k0), torch.empty_like(v0)
    path, count, nxt = i32([[0] * n] * S), i32([0] * S), i32([0] * S)
    took, _ = P.commit(tokens, parents, targets, n)
    assert len(took) == n // 2
    q = r.q[:S].reshape(S, -1).to(dev())
    out, spans = torch.zeros_like(q), r.spans()
    step = decode(ops, q, k1, v1, out, i32([held + len(took) - 1] * S), spans[3], page, heads, 1)

    def run():
        k1.copy_(k0), v1.copy_(v0)
        ops.tree_commit(*flat, k1, v1, *spans, page, path, count, nxt)

    run()
    torch.cuda.synchronize()
    assert count.tolist() == [len(took)] * S
    step(0)
    torch.cuda.synchronize()
    want = out.clone()
    assert bool(want.isfinite().all())
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run()
        step()
    for i in range(40):
        out.zero_()
        if i % 2:
            graph.replay()
        else:
            run()
            step()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def shifted(t, by):
    """The same numbers in memory that begins ``by`` numbers behind a boundary of 16 bytes."""
    room = torch.empty(t.numel() + 16, dtype=t.dtype, device=dev())
    assert room.data_ptr() % 16 == 0
    return room[by:by + t.numel()].view(t.shape).copy_(t)


ODD = [(3, 1, 5), (4, 2, 18), (6, 2, 67), (12, 4, 130), (2, 1, 255), (7, 7, 1)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", ODD, ids=str)
def test_odd_heads(ops, dtype, heads):
    """Heads of no whole groups of four numbers: trees, portions and single tokens, uncut jobs and cut ones."""
    rng = random.Random(11)
    held, rows = [0, 1, 63, 200, 17, 1500], [5, 1, 37, 90, 0, 3]
    r = Requests(held, rows, heads, dtype, 16, 301)
    mask = spread_mask(ops, r, trees(rng, rows))
    check_rows(r, run_tree(ops, r, mask), tree_sees(r, mask))
    mass_in = torch.rand((r.hkv, r.num_slots), generator=torch.Generator().manual_seed(302))
    for n in (rows, [1] * 6, [2, 1, 2, 0, 1, 2]):
        r = Requests(held, n, heads, dtype, 16, 303)
        mass_in = torch.rand((r.hkv, r.num_slots), generator=torch.Generator().manual_seed(304))
        got, mass = run_mass(ops, r, mass_in)
        G.check_mass(r, got, mass, mass_in, torch.full_like(mass_in, -5.0))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (6, 2, 67), (5, 1, 20)], ids=str)
@pytest.mark.parametrize("by", [1, 2, 4, 5])
@pytest.mark.parametrize("which", ["q", "k", "v", "out", "all"])
def test_addresses_behind_a_boundary(ops, dtype, heads, by, which):
    """Operands that begin 2, 4, 8 or more bytes behind 16: each of them alone, and all, with little and much to do."""
    for held, rows in (([0, 90, 1100], [6, 40, 3]), ([33, 2, 700], [1, 1, 1])):
        r = Requests(held, rows, heads, dtype, 16, 305)
        at = lambda name, t: shifted(t, by) if which in (name, "all") else t.to(dev())  # noqa: E731
        q, k, v = at("q", r.q.reshape(r.T, -1)), at("k", r.k), at("v", r.v)
        mask = spread_mask(ops, r, trees(random.Random(2), rows))
        out = at("out", torch.full((r.T, r.hq * r.hd), 7.0, dtype=dtype))
        ops.tree_attention(q, k, v, out, mask.to(dev()), *r.args())
        check_rows(r, out.cpu().reshape(r.T, r.hq, r.hd), tree_sees(r, mask))
        mass_in = torch.rand((r.hkv, r.num_slots), generator=torch.Generator().manual_seed(306))
        mass, out = shifted(torch.full_like(mass_in, -5.0), 1), at("out", torch.full((r.T, r.hq * r.hd), 7.0, dtype=dtype))
        ops.paged_attention_mass(q, k, v, out, mass, *r.args(), max(rows), mass_in=shifted(mass_in, 3))
        G.check_mass(r, out.cpu().reshape(r.T, r.hq, r.hd), mass.cpu(), mass_in, torch.full_like(mass_in, -5.0))
    ops.check_async_errors(dev())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (5, 1, 20)], ids=str)
def test_scales_below_zero(ops, dtype, heads):
    """Scores of the queries turned round, and of a scale of nothing: every key that a row sees weighs the same."""
    for held, rows in (([0, 90, 1100], [6, 40, 3]), ([33, 2, 700], [1, 1, 1])):
        r = Requests(held, rows, heads, dtype, 16, 307)
        q, scale = r.q, r.scale
        mask = spread_mask(ops, r, trees(random.Random(3), rows))
        r.q, r.scale = -q, -scale
        tree, (got, mass) = run_tree(ops, r, mask), run_mass(ops, r, None)
        r.q, r.scale = q, scale
        check_rows(r, tree, tree_sees(r, mask))
        G.check_mass(r, got, mass, None, torch.full_like(mass, -5.0))
        r.scale = 0.0
        check_rows(r, run_tree(ops, r, mask), tree_sees(r, mask))
        got, mass = run_mass(ops, r, None)
        G.check_mass(r, got, mass, None, torch.full_like(mass, -5.0))


@pytest.mark.parametrize("heads", [(3, 1, 4), (4, 2, 2), (2, 1, 20), (5, 5, 12), (2, 1, 33)], ids=str)
@pytest.mark.parametrize("layers", [0, 3])
def test_rows_of_other_widths_move(ops, heads, layers):
    """Rows of 8 bytes and of eights, fours and twos of them."""
    G.test_commit(ops, torch.bfloat16, heads, layers)
    for held, budget in (([33, 5, 200, 0], 32), ([129, 128], 128), ([3000, 77], 1000)):
        for apart in (False, True):
            G.test_evict(ops, torch.bfloat16, heads, held, budget, 3, 8, apart, False)


@pytest.mark.parametrize("by", [1, 2, 4])
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("held", [600, 5000])
def test_planes_behind_a_boundary_move(ops, by, dtype, held):
    """Rows of a whole number of 16 bytes in planes that begin between them (K alone, V alone, both): what aligned planes have afterwards."""
    S, L, budget = 3, 2, 500
    r, k, v, mass, pos, ends = G.evict_case([held] * S, (8, 4, 16), dtype, 16, L, 308)
    planes = lambda a, b: (shifted(k, by) if a else k.to(dev()), shifted(v, by) if b else v.to(dev()), shifted(mass, 1), shifted(pos, 3))  # noqa: E731
    spans, args = r.spans(), (i32([held] * S), i32(ends), r.spans()[3], 16, budget, 4, 100)
    want = (k.to(dev()), v.to(dev()), mass.to(dev()), pos.to(dev()))
    ops.cache_evict(*want, *args)
    parents = [-1] + [max(0, i - 2) for i in range(1, 40)]
    tokens = [i % 2 for i in range(40)]
    trees_of = [i32(x * S) for x in (tokens, parents, [0] * 40)]
    row, length, at = i32([0, 40, 80]), i32([40] * S), i32([held - 40] * S)
    for planes_at in ((1, 0), (0, 1), (1, 1)):
        got = planes(*planes_at)
        ops.cache_evict(*got, *args)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    commit = lambda a, b: ops.tree_commit(*trees_of, a, b, row, length, at, spans[3], 16, i32([[0] * 30] * S), i32([0] * S), i32([0] * S))  # noqa: E731
    want = (k.to(dev()), v.to(dev()))
    commit(*want)
    assert not torch.equal(want[0].cpu(), k)
    for planes_at in ((1, 0), (0, 1), (1, 1)):
        got = planes(*planes_at)[:2]
        commit(*got)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_captured_eviction_into_other_planes(ops):
    """A replay's weights and positions, in planes of their own, against the plain form, for other lengths, tables and weights of the same sizes."""
    heads, page, budget = (4, 2, 16), 16, 64
    graph, args, planes = torch.cuda.CUDAGraph(), None, None
    for i, held in enumerate(([100, 64, 200, 65], [300, 20, 64, 90], [63, 70, 80, 299])):
        r, k, v, mass, pos, ends = G.evict_case(held, heads, torch.bfloat16, page, 2, 310 + i)
        slots, width = 80 * page, 24
        fill = lambda t, axis: torch.cat([t, t.new_zeros([n if d != axis else slots - t.shape[axis] for d, n in enumerate(t.shape)])], axis).to(dev())  # noqa: E731
        new = (fill(k, 1), fill(v, 1), fill(mass, 2), fill(pos, 2))
        table = i32([row + [-1] * (width - len(row)) for row in r.table])
        if planes is None:
            planes, args = [x.clone() for x in new], (i32(held), i32(ends), table)
            mo, po = torch.empty_like(planes[2]), torch.empty_like(planes[3])
            with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
                ops.cache_evict(*planes, *args, page, budget, 4, 20, mass_out=mo, positions_out=po)
        for a, b in zip((*planes, *args), (*new, i32(held), i32(ends), table)):
            a.copy_(b)
        mo.fill_(-3.0), po.fill_(-3)
        graph.replay()
        torch.cuda.synchronize()
        want_m, want_p = torch.full_like(mass, -3.0), torch.full_like(pos, -3)
        for l in range(2):
            for h in range(r.hkv):
                for s, n in enumerate(held):
                    at = r.slots[s]
                    stay = at[:min(n, budget)]
                    want_m[l, h, stay], want_p[l, h, stay] = mass[l, h, stay], pos[l, h, stay]
                    for a, b in P.evict(mass[l, h, at].tolist(), pos[l, h, at].tolist(), ends[s], budget, 4, 20):
                        want_m[l, h, at[a]], want_p[l, h, at[a]] = mass[l, h, at[b]], pos[l, h, at[b]]
                        k[l, at[a], h], v[l, at[a], h] = k[l, at[b], h].clone(), v[l, at[b], h].clone()
        n = r.num_slots
        assert torch.equal(mo[:, :, :n].cpu(), want_m) and torch.equal(po[:, :, :n].cpu(), want_p)
        assert torch.equal(planes[0][:, :n].cpu(), k) and torch.equal(planes[1][:, :n].cpu(), v)
        assert bool((mo[:, :, n:] == -3.0).all()) and bool((po[:, :, n:] == -3).all())


class Served:
    """One layer's cache of three requests as a served model steps over it, with lengths on the device: portions and single tokens whose keys'
    weights are counted, thinning, drafted trees and what of them is confirmed, decode steps.  ``look`` is called behind every step."""
    BUDGET, PAGE, WIDTH, LENS, TREES = 96, 16, 16, [140, 40, 97], [9, 5, 12]

    def __init__(self, ops, heads, dtype, look):
        self.ops, self.heads, self.look = ops, heads, look
        hq, hkv, hd = heads
        g, rng = torch.Generator().manual_seed(401), random.Random(401)
        S = len(self.LENS)
        order = torch.randperm(S * self.WIDTH + 2, generator=g).tolist()
        self.table = i32([order[s * self.WIDTH:(s + 1) * self.WIDTH] for s in range(S)])
        slots = len(order) * self.PAGE
        self.k, self.v = (torch.full((slots, hkv, hd), math.nan, dtype=dtype, device=dev()) for _ in range(2))
        self.mass, self.pos = torch.full((hkv, slots), math.nan, device=dev()), torch.zeros((hkv, slots), dtype=torch.int32, device=dev())
        self.held, self.ends = i32([0] * S), i32([0] * S)
        self.inv = (10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float().to(dev())
        self.rounds = []
        for n in (self.LENS, [1] * S, [1] * S):
            parents = trees(rng, self.TREES)
            tokens = [[rng.randrange(3) for _ in t] for t in parents]
            targets = [[rng.randrange(3) for _ in t] for t in parents]
            depth = []
            for t in parents:
                d = []
                for p in t:
                    d.append(d[p] + 1 if p >= 0 else 0)
                depth += d
            qkv = [torch.randn((sum(rows), (hq + 2 * hkv) * hd), generator=g).to(dtype).to(dev()) for rows in (n, self.TREES, [1] * S)]
            flat = [i32([x for t in lists for x in t]) for lists in (tokens, parents, targets)]
            self.rounds.append((n, parents, tokens, targets, i32(depth), qkv, flat, ops.tree_mask(parents).to(dev())))
        self.first = {str(n): i32([sum(n[:s]) for s in range(S)]) for n in (self.LENS, self.TREES, [1] * S)}
        self.row = {str(n): (torch.tensor([s for s in range(S) for _ in range(n[s])], device=dev()), torch.tensor([i for s in range(S) for i in range(n[s])], device=dev()))
                    for n in (self.LENS, self.TREES, [1] * S)}
        self.lengths = {str(n): i32(n) for n in (self.LENS, self.TREES, [1] * S)}
        self.outs = [torch.zeros((sum(n), hq * hd), dtype=dtype, device=dev()) for r in self.rounds for n in (r[0], self.TREES, [1] * S)]
        self.paths = [(i32([[0] * 12] * S), i32([0] * S), i32([0] * S)) for _ in self.rounds]

    def places(self, req, at):
        return (self.table[req, at // self.PAGE] * self.PAGE + at % self.PAGE).long()

    def bring(self, n, qkv, depth=None):
        """The rows' keys and values, rotated by their positions, behind what the requests hold; the rotated queries."""
        hq, hkv, hd = self.heads
        req, i = self.row[str(n)]
        slot = self.places(req, self.held[req] + i)
        position = (self.ends[req] + (i if depth is None else depth)).int()
        q = torch.empty((qkv.shape[0], hq * hd), dtype=qkv.dtype, device=dev())
        self.ops.rope_kv_write(qkv, position, slot.int(), self.inv, hd, False, q, self.k, self.v, hq, hkv, hd)
        return q, slot, position

    def run(self):
        ops, (hq, hkv, hd), S = self.ops, self.heads, len(self.LENS)
        outs = iter(self.outs)
        for (n, parents, tokens, targets, depth, qkv, flat, mask), (path, count, nxt) in zip(self.rounds, self.paths):
            args = (self.table, self.PAGE, hq, hkv, hd, hd ** -0.5)
            # a portion of each, or a token
            q, slot, position = self.bring(n, qkv[0])
            self.pos[:, slot] = position
            self.look("bring", self)
            out = next(outs)
            ops.paged_attention_mass(q, self.k, self.v, out, self.mass, self.first[str(n)], self.lengths[str(n)], self.held, *args, max(n), mass_in=self.mass)
            self.look("mass", self, n, q, out)
            self.held += self.lengths[str(n)]
            self.ends += self.lengths[str(n)]
            ops.cache_evict(self.k, self.v, self.mass, self.pos, self.held, self.ends, self.table, self.PAGE, self.BUDGET, 4, 16)
            self.look("evict", self)
            self.held.clamp_(max=self.BUDGET)
            # drafted trees
            n = self.TREES
            q, _, _ = self.bring(n, qkv[1], depth)
            out, spans = next(outs), (self.first[str(n)], self.lengths[str(n)], self.held)
            ops.tree_attention(q, self.k, self.v, out, mask, *spans, *args)
            self.look("tree", self, n, q, out, parents)
            ops.tree_commit(*flat, self.k, self.v, *spans, self.table, self.PAGE, path, count, nxt)
            self.look("commit", self, tokens, parents, targets, path, count, nxt)
            d = torch.arange(12, device=dev())
            req = torch.arange(S, device=dev())[:, None].expand(S, 12)
            slot = torch.where(d < count[:, None], self.places(req, self.held[:, None] + d), self.places(req[:, :1], self.held[:, None]))
            self.mass.index_fill_(1, slot.reshape(-1), 0.0)
            self.pos[:, slot] = torch.where(d < count[:, None], self.ends[:, None] + d, self.ends[:, None]).int()
            self.held += count
            self.ends += count
            # a token each
            n = [1] * S
            q, slot, position = self.bring(n, qkv[2])
            self.mass.index_fill_(1, slot.reshape(-1), 0.0)
            self.pos[:, slot] = position
            q, slot, position = self.bring(n, qkv[2])          # (again, so that no other launch lies between the write and the decode)
            out = next(outs)
            iota, zeros = self.first[str(n)], self.first[str(n)] * 0
            ops.paged_decode_mma(q, self.k, self.v, out, iota, zeros, S, iota, self.held, self.table, self.WIDTH, self.PAGE, hq, hkv, hd, 0, hd ** -0.5, 2, None,
                                 fresh=1)
            self.look("decode", self, n, q, out)
            self.held += 1
            self.ends += 1

    def state(self):
        return [self.k, self.v, self.mass, self.pos, self.held, self.ends, *self.outs, *(x for p in self.paths for x in p)]


class Looker:
    """The plain forms beside every step, from what the caches held before it."""

    def __init__(self):
        self.calls = 0

    def of(self, a, s, more):
        at = torch.arange(self.held[s] + more)
        return (a.table.cpu()[s, at // a.PAGE] * a.PAGE + at % a.PAGE).long()

    def attend(self, a, n, q, out, sees):
        r = Requests([0], [1], a.heads, q.dtype, 16, 0)
        for s, rows in enumerate(n):
            first = sum(n[:s])
            slots = self.of(a, s, rows)
            mine = q.cpu().view(-1, a.heads[0], a.heads[2])[first:first + rows], a.k.cpu()[slots], a.v.cpu()[slots]
            want, w = P.attention(*mine, sees(s, rows), a.heads[2] ** -0.5)
            r.of, r.slots = lambda _: mine, [slots.tolist()]
            got = out.cpu().double().view(-1, a.heads[0], a.heads[2])[first:first + rows]
            assert bool(((got - want).abs() <= r.tolerance(0, want)).all()), (self.calls, s)
            yield s, slots, mine, w

    def causal(self, s, rows):
        return torch.cat([torch.ones((rows, self.held[s]), dtype=torch.bool), torch.ones((rows, rows), dtype=torch.bool).tril()], 1)

    def __call__(self, what, a, *more):
        self.calls += 1
        torch.cuda.synchronize()
        self.held = a.held.tolist()          # (as the step was given it)
        if what == "mass":
            n, q, out = more
            for s, slots, (mq, mk, _), w in self.attend(a, n, q, out, self.causal):
                sums = w.reshape(a.heads[1], -1, w.shape[-1]).sum(1)
                before = torch.zeros_like(sums)
                before[:, :self.held[s]] = self.mass[:, slots[:self.held[s]]].double()
                rel = 2 * P.score_error(mq, mk, a.heads[2] ** -0.5) + (n[s] * a.heads[0] // a.heads[1] + len(slots) + 16) * 2.0 ** -24 + 2.0 ** -20
                assert bool(((a.mass.cpu()[:, slots].double() - before - sums).abs() <= rel * sums + 2.0 ** -23 * before).all())
        elif what == "tree":
            n, q, out, parents = more
            list(self.attend(a, n, q, out, lambda s, rows: torch.cat([torch.ones((rows, self.held[s]), dtype=torch.bool), P.ancestors(parents[s])], 1)))
        elif what == "decode":
            n, q, out = more
            list(self.attend(a, n, q, out, self.causal))
        elif what == "evict":
            for s in range(3):
                at, ends = self.of(a, s, 0), a.ends.tolist()
                for h in range(a.heads[1]):
                    for hole, filler in P.evict(self.new_mass[h, at].tolist(), self.new_pos[h, at].tolist(), ends[s], a.BUDGET, 4, 16):
                        for t in (self.k, self.v):
                            t[at[hole], h] = t[at[filler], h].clone()
                        for t in (self.new_mass, self.new_pos):
                            t[h, at[hole]] = t[h, at[filler]].clone()
            for got, want in ((a.k, self.k), (a.v, self.v), (a.mass, self.new_mass), (a.pos, self.new_pos)):
                assert torch.equal(got.cpu().nan_to_num(9.0), want.nan_to_num(9.0))
        elif what == "commit":
            tokens, parents, targets, path, count, nxt = more
            for s in range(3):
                took, last = P.commit(tokens[s], parents[s], targets[s], 12)
                assert path[s].tolist() == took + [-1] * (12 - len(took)) and int(count[s]) == len(took) and int(nxt[s]) == last
                slots = self.of(a, s, 12)[self.held[s]:]
                for t in (self.k, self.v):
                    t[slots[:len(took)]] = t[slots[took]].clone()
            assert torch.equal(a.k.cpu().nan_to_num(9.0), self.k.nan_to_num(9.0)) and torch.equal(a.v.cpu().nan_to_num(9.0), self.v.nan_to_num(9.0))
        # what the next step finds
        self.k, self.v, self.new_mass, self.new_pos = a.k.cpu(), a.v.cpu(), a.mass.cpu(), a.pos.cpu()
        self.mass = self.new_mass


@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128)], ids=str)
def test_served_steps_in_bf16(ops, heads):
    """Cache writes, counted attention, thinning, drafted trees, their commit and decode steps behind one another: every step against the plain
    forms, then all of them without a look between, eager and as one graph, with equal bits."""
    look = Looker()
    a = Served(ops, heads, torch.bfloat16, look)
    a.run()
    ops.check_async_errors(dev())
    assert look.calls == 18 and a.held.tolist() != a.ends.tolist()
    want = [x.clone() for x in a.state()]
    b = Served(ops, heads, torch.bfloat16, lambda *_: None)
    start = [x.clone() for x in b.state()]
    b.run()
    torch.cuda.synchronize()
    assert all(torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0)) for x, y in zip(b.state(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        b.run()
    for _ in range(3):
        for x, y in zip(b.state(), start):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0)) for x, y in zip(b.state(), want))
    ops.check_async_errors(dev())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (5, 1, 20)], ids=str)
@pytest.mark.parametrize("held", [0, 40, 700])
def test_infinite_values_of_keys_that_weigh_next_to_nothing(ops, dtype, heads, held):
    """A weight of less than 32 bits show times infinity is infinity (or, with a weight of 0, NaN): it shows in the rows that see the key, and in no
    others."""
    r = Requests([held, 9], [30, 6], heads, dtype, 16, 209)
    r.q[:, :, 0] = r.q[:, :, 0].abs() + 1.0
    at = held + 11
    r.k[r.slots[0][at], :, 0] = -300.0 / r.scale          # scores of -300 and less
    r.v[r.slots[0][at], :, 2] = math.inf
    mask = spread_mask(ops, r, trees(random.Random(8), r.rows))
    sees = tree_sees(r, mask)
    assert bool(sees[0][:, at].any()) and not bool(sees[0][:, at].all())
    got = run_tree(ops, r, mask)[r.first[0]:r.first[0] + 30]
    assert torch.equal(~got.isfinite()[:, :, 2], sees[0][:, at, None].expand(30, r.hq)) and bool(got[:, :, :2].isfinite().all())
    got, mass = run_mass(ops, r, None)
    got = got[r.first[0]:r.first[0] + 30]
    assert torch.equal(~got.isfinite()[:, :, 2], causal(r)[0][:, at, None].expand(30, r.hq)) and bool(got[:, :, :2].isfinite().all())
    # (a row that sees no key but this one gives it everything: there is none here)
    assert bool((mass[:, r.slots[0][at]] == 0).all())
