"""Attention of drafted trees, their commit, attention that counts keys' weights and eviction, against plain forms in 64 bits."""
import math
import random

import pytest
import torch

from tests.plain import draft_cache_plain as P

pytestmark = pytest.mark.gpu
HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (4, 2, 16), (3, 1, 32), (8, 8, 64), (16, 1, 128), (5, 1, 20), (2, 1, 256), (64, 1, 64)]
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from lightllm_b200.csrc import ops as o
    o.lib()
    return o


def dev():
    return torch.device("cuda:0")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=dev())


class Requests:
    """Requests of ``held`` keys and ``rows`` new rows each in shuffled pages; what no request owns is NaN, and rows of no request lie
    between the requests' rows."""

    def __init__(self, held, rows, heads, dtype, page, seed, gap=1):
        self.held, self.rows, self.page, self.dtype = held, rows, page, dtype
        self.hq, self.hkv, self.hd = heads
        g = torch.Generator().manual_seed(seed)
        S = len(held)
        need = [-(-(h + n) // page) for h, n in zip(held, rows)]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g).tolist()
        width = max(need + [1]) + 1
        table, at = [], 0
        for n in need:
            table.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.table = table
        self.slots = [[table[s][j // page] * page + j % page for j in range(held[s] + rows[s])] for s in range(S)]
        self.num_slots = pages * page
        self.k, self.v = (torch.full((self.num_slots, self.hkv, self.hd), math.nan) for _ in range(2))
        for s in range(S):
            for c in (self.k, self.v):
                c[self.slots[s]] = torch.randn((len(self.slots[s]), self.hkv, self.hd), generator=g)
        self.first = [sum(rows[:s]) + gap * (s + 1) for s in range(S)]
        self.T = sum(rows) + gap * (S + 1)
        self.q = torch.randn((self.T, self.hq, self.hd), generator=g)
        self.k, self.v, self.q = (x.to(dtype) for x in (self.k, self.v, self.q))
        self.scale = self.hd ** -0.5

    def spans(self):
        return i32(self.first), i32(self.rows), i32(self.held), i32(self.table).reshape(len(self.held), len(self.table[0]) if self.table else 1)

    def args(self):
        return (*self.spans(), self.page, self.hq, self.hkv, self.hd, self.scale)

    def of(self, s):
        return self.q[self.first[s]:self.first[s] + self.rows[s]], self.k[self.slots[s]], self.v[self.slots[s]]

    def tolerance(self, s, want):
        """Scores are off by score_error, and so (twice: in the weight and in the sum) are weights in proportion; sums of so many weights
        by half a step of 32 bits a term at most; with bf16 every weight is rounded for the product with the values, and the result."""
        q, k, v = self.of(s)
        rel = 2 * P.score_error(q, k, self.scale) + (len(self.slots[s]) + 8) * 2.0 ** -24 + 2.0 ** -21
        top = float(v.double().abs().nan_to_num(0.0, 0.0, 0.0).max()) if v.numel() else 0.0
        if self.dtype == torch.bfloat16:
            return (rel + 2.0 ** -8) * top + 2.0 ** -8 * want.abs()
        return rel * top + 2.0 ** -24 * want.abs()


def trees(rng, rows):
    return [[-1] + [rng.randrange(max(0, i - 5), i) for i in range(1, n)] if n else [] for n in rows]


def run_tree(ops, r, mask):
    out = torch.full((r.T, r.hq * r.hd), 7.0, dtype=r.dtype, device=dev())
    ops.tree_attention(r.q.reshape(r.T, -1).to(dev()), r.k.to(dev()), r.v.to(dev()), out, mask.to(dev()), *r.args())
    ops.check_async_errors(dev())
    return out.cpu().reshape(r.T, r.hq, r.hd)


def check_rows(r, got, sees):
    """All rows of all requests, and that rows of no request were left alone."""
    mine = torch.zeros(r.T, dtype=torch.bool)
    for s, n in enumerate(r.rows):
        if not n:
            continue
        q, k, v = r.of(s)
        want, _ = P.attention(q, k, v, sees[s], r.scale)
        rows = got[r.first[s]:r.first[s] + n].double()
        mine[r.first[s]:r.first[s] + n] = True
        assert torch.equal(rows.isfinite(), want.isfinite())
        off = (rows - want).abs() - r.tolerance(s, want)
        off = off[want.isfinite()]
        assert not off.numel() or float(off.max()) <= 0, (s, float(off.max()))
    assert bool((got[~mine] == 7.0).all())


def tree_sees(r, mask):
    sees = []
    for s, n in enumerate(r.rows):
        bits = torch.ones((n, r.held[s] + n), dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                bits[i, r.held[s] + j] = j // 64 < mask.shape[1] and bool((int(mask[r.first[s] + i, j // 64]) >> (j % 64)) & 1)
        sees.append(bits)
    return sees


def spread_mask(ops, r, parents):
    m = ops.tree_mask(parents)
    mask = torch.full((r.T, m.shape[1]), -1, dtype=torch.int64)
    at = 0
    for s, n in enumerate(r.rows):
        mask[r.first[s]:r.first[s] + n] = m[at:at + n]
        at += n
    return mask


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("page", [8, 16])
def test_trees_of_many_sizes(ops, dtype, heads, page):
    """Requests of no keys and of many, trees of one node to more than a mask's word, a request without rows among them."""
    rng = random.Random(3)
    held = [0, 1, 63, 64, 65, 127, 128, 300, 17, 1000]
    rows = [5, 1, 19, 37, 2, 9, 64, 0, 70, 3]
    r = Requests(held, rows, heads, dtype, page, 11)
    mask = spread_mask(ops, r, trees(rng, rows))
    check_rows(r, run_tree(ops, r, mask), tree_sees(r, mask))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (3, 1, 32)], ids=str)
@pytest.mark.parametrize("held", [1, 127, 129, 2000, 5003])
@pytest.mark.parametrize("n", [1, 8, 21, 64])
def test_one_request(ops, dtype, heads, held, n):
    """A single request's keys are shared by all blocks."""
    r = Requests([held], [n], heads, dtype, 16, 12, gap=0)
    mask = spread_mask(ops, r, trees(random.Random(held + n), [n]))
    check_rows(r, run_tree(ops, r, mask), tree_sees(r, mask))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (3, 1, 32)], ids=str)
def test_any_mask(ops, dtype, heads):
    """Masks that are no trees: random bits (those beyond the request's nodes among them), rows that see no drafted node and, in
    requests that hold no keys, nothing at all: zeros."""
    g = torch.Generator().manual_seed(5)
    held, rows = [0, 0, 40, 130], [3, 66, 30, 90]
    r = Requests(held, rows, heads, dtype, 16, 13)
    mask = torch.randint(-2 ** 63, 2 ** 63 - 1, (r.T, 3), generator=g)
    mask[::3] = 0
    got, sees = run_tree(ops, r, mask), tree_sees(r, mask)
    check_rows(r, got, sees)
    empty = [r.first[s] + i for s in (0, 1) for i in range(rows[s]) if not sees[s][i].any()]
    assert empty and bool((got[empty] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (3, 1, 32)], ids=str)
@pytest.mark.parametrize("held", [0, 50, 1000])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_masked_is_nothing(ops, dtype, heads, held, bad):
    """A node's keys or values that are no finite numbers show in the rows that see it and in no others."""
    r = Requests([held, 9], [40, 6], heads, dtype, 16, 14)
    parents = trees(random.Random(8), r.rows)
    mask = spread_mask(ops, r, parents)
    r.v[r.slots[0][held + 7], 0, 3] = bad
    r.v[r.slots[0][held + 31], :, :] = bad
    if bad != math.inf:
        r.k[r.slots[0][held + 22], 0, :] = math.nan
    got, sees = run_tree(ops, r, mask), tree_sees(r, mask)
    assert not sees[0][:, held + 7].all() and not sees[0][:, held + 22].all()
    check_rows(r, got, sees)


def test_keys_whose_scores_stand_out(ops):
    """The running maximum rises late and by much, in the last tile and among the drafted nodes."""
    for dtype in DTYPES:
        for heads in ((14, 2, 64), (12, 2, 128)):
            r = Requests([700, 1500], [20, 3], heads, dtype, 16, 15)
            for s in range(2):
                for j, x in ((100, 4.0), (650, 9.0), (r.held[s], 14.0)):
                    r.k[r.slots[s][j]] = x * torch.sign(r.q[r.first[s], 0]).to(dtype)
            mask = spread_mask(ops, r, trees(random.Random(9), r.rows))
            check_rows(r, run_tree(ops, r, mask), tree_sees(r, mask))


def run_mass(ops, r, mass_in, max_len=None, in_place=False):
    out = torch.full((r.T, r.hq * r.hd), 7.0, dtype=r.dtype, device=dev())
    mass = mass_in.to(dev()) if in_place else torch.full((r.hkv, r.num_slots), -5.0, device=dev())
    given = mass if in_place else None if mass_in is None else mass_in.to(dev())
    ops.paged_attention_mass(r.q.reshape(r.T, -1).to(dev()), r.k.to(dev()), r.v.to(dev()), out, mass, *r.args(),
                             max(r.rows) if max_len is None else max_len, mass_in=given)
    ops.check_async_errors(dev())
    return out.cpu().reshape(r.T, r.hq, r.hd), mass.cpu()


def check_mass(r, got, mass, mass_in, left):
    sees = [torch.cat([torch.ones((n, h), dtype=torch.bool), torch.ones((n, n), dtype=torch.bool).tril()], 1) for h, n in zip(r.held, r.rows)]
    check_rows(r, got, sees)
    touched = torch.zeros(r.num_slots, dtype=torch.bool)
    for s, n in enumerate(r.rows):
        if not n:
            continue
        q, k, v = r.of(s)
        _, w = P.attention(q, k, v, sees[s], r.scale)
        sums = w.reshape(r.hkv, -1, w.shape[-1]).sum(1)
        before = torch.zeros_like(sums)
        if mass_in is not None:
            before[:, :r.held[s]] = mass_in[:, r.slots[s][:r.held[s]]].double()
        have = mass[:, r.slots[s]].double()
        # a weight's score and its row's sum are off by score_error each; the exponential, the logarithm and so many additions by half
        # a step or a few of 32 bits
        rel = 2 * P.score_error(q, k, r.scale) + (n * r.hq // r.hkv + len(r.slots[s]) + 16) * 2.0 ** -24 + 2.0 ** -20
        assert bool(((have - before - sums).abs() <= rel * sums + 2.0 ** -23 * before.abs()).all()), (s, float((have - before - sums).abs().max()))
        touched[r.slots[s]] = True
    assert torch.equal(mass[:, ~touched], left[:, ~touched])


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("rows", ["single", "portions"])
def test_mass(ops, dtype, heads, rows):
    """One token of every request, and portions of several lengths beside single tokens, onto sums of before."""
    held = [0, 1, 15, 63, 64, 127, 128, 333, 1500]
    n = [1] * len(held) if rows == "single" else [7, 1, 130, 20, 64, 1, 3, 0, 40]
    r = Requests(held, n, heads, dtype, 16, 21)
    mass_in = torch.rand((r.hkv, r.num_slots), generator=torch.Generator().manual_seed(22))
    left = torch.full_like(mass_in, -5.0)
    got, mass = run_mass(ops, r, mass_in)
    check_mass(r, got, mass, mass_in, left)
    again, mass2 = run_mass(ops, r, mass_in.clone(), in_place=True)
    check_mass(r, again, mass2, mass_in, mass_in)
    assert torch.equal(got, again)
    got, mass = run_mass(ops, r, None)
    check_mass(r, got, mass, None, left)
    # a longer most than any request has is no other result
    got2, mass3 = run_mass(ops, r, None, max_len=max(n) + 70)
    check_mass(r, got2, mass3, None, left)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (3, 1, 32)], ids=str)
@pytest.mark.parametrize("held,n", [(0, 1), (5000, 1), (0, 300), (250, 257), (3000, 2)])
def test_mass_of_one_request(ops, dtype, heads, held, n):
    r = Requests([held], [n], heads, dtype, 8, 23, gap=0)
    mass_in = torch.rand((r.hkv, r.num_slots), generator=torch.Generator().manual_seed(24))
    got, mass = run_mass(ops, r, mass_in)
    check_mass(r, got, mass, mass_in, torch.full_like(mass_in, -5.0))


def test_mass_sums_to_the_rows(ops):
    """Every row's weights add up to one: all keys' together to rows times the group."""
    r = Requests([100, 2000], [77, 1], (14, 2, 64), torch.bfloat16, 16, 25)
    _, mass = run_mass(ops, r, None)
    for s, n in enumerate(r.rows):
        assert torch.allclose(mass[:, r.slots[s]].double().sum(1), torch.full((2,), 7.0 * n, dtype=torch.float64), rtol=1e-5)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (4, 2, 16), (3, 1, 5), (28, 4, 128)], ids=str)
@pytest.mark.parametrize("layers", [0, 1, 5])
def test_commit(ops, dtype, heads, layers):
    """Paths of all lengths, several children with the right token (the first goes on), requests without rows, a width that cuts."""
    rng = random.Random(31)
    held = [0, 5, 16, 31, 100, 7, 64]
    rows = [1, 9, 40, 0, 70, 26, 3]
    r = Requests(held, rows, heads, dtype, 16, 32)
    parents = trees(rng, rows)
    for width in (1, 4, 70):
        tokens = [[rng.randrange(4) for _ in t] for t in parents]
        targets = [[rng.randrange(4) for _ in t] for t in parents]
        for t, k, g in zip(parents, tokens, targets):          # most nodes go on
            for i in range(1, len(t)):
                if rng.random() < 0.5:
                    g[t[i]] = k[i]
        flat = [torch.full((r.T,), 99, dtype=torch.int32) for _ in range(3)]
        for x, lists in zip(flat, (tokens, parents, targets)):
            for s, v in enumerate(lists):
                x[r.first[s]:r.first[s] + rows[s]] = torch.tensor(v, dtype=torch.int32)
        shape = ((layers,) if layers else ()) + tuple(r.k.shape)
        g = torch.Generator().manual_seed(33)
        k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        kd, vd = k.to(dev()), v.to(dev())
        path = torch.full((len(held), width), 5, dtype=torch.int32, device=dev())
        count, nxt = i32([9] * len(held)), i32([9] * len(held))
        ops.tree_commit(*(x.to(dev()) for x in flat), kd, vd, *r.spans(), r.page, path, count, nxt)
        for s in range(len(held)):
            want, last = P.commit(tokens[s], parents[s], targets[s], width)
            assert path[s].tolist() == want + [-1] * (width - len(want))
            assert int(count[s]) == len(want) and int(nxt[s]) == last
            src = [r.slots[s][held[s] + a] for a in want]
            dst = [r.slots[s][held[s] + d] for d in range(len(want))]
            for c in (k, v):
                c[..., dst, :, :] = c[..., src, :, :].clone()
        assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


def evict_case(held, heads, dtype, page, layers, seed, ties=False):
    g = torch.Generator().manual_seed(seed)
    r = Requests(held, [0] * len(held), heads, torch.float32, page, seed)
    L = max(1, layers)
    k, v = (torch.randn((L, r.num_slots, r.hkv, r.hd), generator=g).to(dtype) for _ in range(2))
    mass = torch.exp(2.0 * torch.randn((L, r.hkv, r.num_slots), generator=g))
    if ties:
        mass = torch.randint(0, 5, mass.shape, generator=g).float() * torch.where(torch.rand(mass.shape, generator=g) < 0.1, -1.0, 1.0)
        mass[torch.rand(mass.shape, generator=g) < 0.02] = math.nan
        mass[torch.rand(mass.shape, generator=g) < 0.02] = math.inf
        mass[torch.rand(mass.shape, generator=g) < 0.02] = -math.inf
    pos = torch.zeros((L, r.hkv, r.num_slots), dtype=torch.int32)
    for s, n in enumerate(held):
        for l in range(L):
            for h in range(r.hkv):
                pos[l, h, r.slots[s]] = torch.randperm(n + 20, generator=g)[:n].to(torch.int32)
    return r, k, v, mass, pos, [n + 20 for n in held]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (4, 2, 16), (3, 1, 5)], ids=str)
@pytest.mark.parametrize("held,budget,first,latest", [
    ([33, 5, 200, 1, 0, 64], 32, 4, 8), ([129, 128, 127, 130], 128, 0, 0), ([1, 2, 3], 1, 0, 1), ([3000, 77, 2500], 1000, 4, 128),
    ([500], 499, 0, 0), ([700, 20], 10, 3, 7), ([4097], 2048, 100, 100)])
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("ties", [False, True])
def test_evict(ops, dtype, heads, held, budget, first, latest, apart, ties):
    """One place and many, equal worths, budgets that are all first and latest places, in place and into other planes."""
    layers = 2 if len(held) > 1 else 0
    r, k, v, mass, pos, ends = evict_case(held, heads, dtype, 16, layers, 41, ties)
    pick = (lambda x: x) if layers else (lambda x: x[0])
    kd, vd, md, pd = (pick(x).contiguous().to(dev()) for x in (k, v, mass, pos))
    mo, po = (torch.full_like(md, -3.0), torch.full_like(pd, -3)) if apart else (None, None)
    ops.cache_evict(kd, vd, md, pd, i32(held), i32(ends), r.spans()[3], r.page, budget, first, latest, mass_out=mo, positions_out=po)
    want_m, want_p = (torch.full_like(mass, -3.0), torch.full_like(pos, -3)) if apart else (mass.clone(), pos.clone())
    before_m, before_p = mass.clone(), pos.clone()
    for l in range(mass.shape[0]):
        for h in range(r.hkv):
            for s, n in enumerate(held):
                at = r.slots[s]
                moves = P.evict(before_m[l, h, at].tolist(), before_p[l, h, at].tolist(), ends[s], budget, first, latest)
                stay = at[:min(n, budget)]
                want_m[l, h, stay], want_p[l, h, stay] = before_m[l, h, stay], before_p[l, h, stay]
                for hole, filler in moves:
                    a, b = at[hole], at[filler]
                    k[l, a, h], v[l, a, h] = k[l, b, h].clone(), v[l, b, h].clone()
                    want_m[l, h, a], want_p[l, h, a] = before_m[l, h, b], before_p[l, h, b]
    assert torch.equal(kd.cpu(), pick(k)) and torch.equal(vd.cpu(), pick(v))
    for got, want in (((mo if apart else md).cpu(), pick(want_m)), ((po if apart else pd).cpu(), pick(want_p))):
        assert torch.equal(got.nan_to_num(1e30, 2e30, -2e30) if got.is_floating_point() else got,
                           want.nan_to_num(1e30, 2e30, -2e30) if want.is_floating_point() else want)
    if apart:
        assert torch.equal(pd.cpu(), pick(pos))


@pytest.mark.parametrize("layers", [1, 4, 8, 15, 30])          # 8, 4, 2 blocks a (layer, request, kv head), and one
@pytest.mark.parametrize("held", [[900, 1500, 601], [513, 513, 40], [9000, 5000, 1]], ids=str)
@pytest.mark.parametrize("apart", [False, True])
def test_evict_shared_by_blocks(ops, layers, held, apart):
    """Few (layer, request, kv head) triples: several blocks share the moves of one."""
    r, k, v, mass, pos, ends = evict_case(held, (4, 2, 16), torch.bfloat16, 16, layers, 43)
    kd, vd, md, pd = (x.to(dev()) for x in (k, v, mass, pos))
    mo, po = (torch.full_like(md, -3.0), torch.full_like(pd, -3)) if apart else (None, None)
    ops.cache_evict(kd, vd, md, pd, i32(held), i32(ends), r.spans()[3], r.page, 512, 4, 100, mass_out=mo, positions_out=po)
    want_m, want_p = (torch.full_like(mass, -3.0), torch.full_like(pos, -3)) if apart else (mass.clone(), pos.clone())
    for l in range(layers):
        for h in range(r.hkv):
            for s, n in enumerate(held):
                at = r.slots[s]
                moves = P.evict(mass[l, h, at].tolist(), pos[l, h, at].tolist(), ends[s], 512, 4, 100)
                stay = at[:min(n, 512)]
                want_m[l, h, stay], want_p[l, h, stay] = mass[l, h, stay], pos[l, h, stay]
                if moves:
                    a, b = (torch.tensor([at[m[i]] for m in moves]) for i in (0, 1))
                    k[l, a, h], v[l, a, h] = k[l, b, h], v[l, b, h]
                    want_m[l, h, a], want_p[l, h, a] = mass[l, h, b], pos[l, h, b]
    for got, want in ((kd, k), (vd, v), (mo if apart else md, want_m), (po if apart else pd, want_p)):
        assert torch.equal(got.cpu(), want)


def test_evict_more_places_than_shared_memory_holds(ops):
    held = [30000, 20001]
    r, k, v, mass, pos, ends = evict_case(held, (2, 1, 4), torch.float32, 16, 1, 42)
    kd, vd, md, pd = (x.to(dev()) for x in (k, v, mass, pos))
    ops.cache_evict(kd, vd, md, pd, i32(held), i32(ends), r.spans()[3], r.page, 9000, 4, 500)
    for s in range(2):
        at = r.slots[s]
        for hole, filler in P.evict(mass[0, 0, at].tolist(), pos[0, 0, at].tolist(), ends[s], 9000, 4, 500):
            for c in (k, v):
                c[0, at[hole]] = c[0, at[filler]].clone()
            mass[0, 0, at[hole]], pos[0, 0, at[hole]] = mass[0, 0, at[filler]].clone(), pos[0, 0, at[filler]].clone()
    for got, want in ((kd, k), (vd, v), (md, mass), (pd, pos)):
        assert torch.equal(got.cpu(), want)


def test_pages_outside_the_cache(ops):
    """A table that names no page of the cache inside a request: its keys read as zeros, its rows are not moved and not written."""
    for dtype in DTYPES:
        r = Requests([100], [9], (4, 2, 64), dtype, 16, 51)
        r.k[r.slots[0][32:48]], r.v[r.slots[0][32:48]] = 0, 0
        for page in (-1, 10 ** 6, 2 ** 31 - 1):
            r.table[0][2] = page
            mask = spread_mask(ops, r, trees(random.Random(1), r.rows))
            check_rows(r, run_tree(ops, r, mask), tree_sees(r, mask))
            got, mass = run_mass(ops, r, None)
            assert bool((mass[:, r.slots[0][32:48]] == -5.0).all())
            kd, vd = r.k.to(dev()), r.v.to(dev())
            md, pd = torch.rand((2, r.num_slots), device=dev()), torch.zeros((2, r.num_slots), dtype=torch.int32, device=dev())
            keep = kd[r.slots[0][32:48]].clone()
            ops.cache_evict(kd, vd, md, pd, i32([100]), i32([200]), r.spans()[3], 16, 40, 0, 0)
            assert torch.equal(kd[r.slots[0][32:48]], keep)


def test_captured(ops):
    """One graph of all four, replayed for other trees, lengths and tables of the same sizes, on a stream of its own; eager calls of the
    same operators run between the replays."""
    heads, page, dtype = (14, 2, 64), 16, torch.bfloat16
    rng = random.Random(61)
    cases = []
    for seed in range(3):
        rows = [rng.randrange(1, 9) for _ in range(3)]
        rows.append(20 - sum(rows) if 0 < 20 - sum(rows) < 9 else 1)
        held = [rng.randrange(0, 300) for _ in rows]
        cases.append((held, rows))
    T, slots, width = 40, 100 * page, 24
    z = lambda *s, d=torch.int32: torch.zeros(s, dtype=d, device=dev())  # noqa: E731
    q, k, v = (torch.randn(s, device=dev()).to(dtype) for s in ((T, 14 * 64), (slots, 2, 64), (slots, 2, 64)))
    row, length, held_d, table, mask = z(4), z(4), z(4), z(4, width), z(T, 1, d=torch.int64)
    tokens, parents, targets, path, count, nxt = z(T), z(T), z(T), z(4, 9), z(4), z(4)
    out, out2, mass, pos, ends = torch.zeros_like(q), torch.zeros_like(q), z(2, slots, d=torch.float32), z(2, slots), z(4)
    k2, v2, mass2, pos2 = (torch.empty_like(x) for x in (k, v, mass, pos))

    def step():
        ops.tree_attention(q, k, v, out, mask, row, length, held_d, table, page, *heads, 0.125)
        ops.paged_attention_mass(q, k, v, out2, mass, row, length, held_d, table, page, *heads, 0.125, 9)
        k2.copy_(k), v2.copy_(v)
        ops.tree_commit(tokens, parents, targets, k2, v2, row, length, held_d, table, page, path, count, nxt)
        ops.cache_evict(k2, v2, mass, pos, held_d, ends, table, page, 64, 2, 16, mass_out=mass2, positions_out=pos2)

    def load(case, seed):
        held, rows = case
        g = torch.Generator().manual_seed(seed)
        order = torch.randperm(100, generator=g).tolist()
        t, at = [], 0
        for h, n in zip(held, rows):
            need = -(-(h + n) // page)
            t.append(order[at:at + need] + [-1] * (width - need))
            at += need
        row.copy_(i32([sum(rows[:s]) for s in range(4)])), length.copy_(i32(rows)), held_d.copy_(i32(held)), table.copy_(i32(t))
        parent = trees(random.Random(seed), rows)
        m = ops.tree_mask(parent)
        mask[:m.shape[0]] = m.to(dev())
        flat = [p for t in parent for p in t]
        parents[:len(flat)] = i32(flat)
        tokens.copy_(torch.randint(0, 2, (T,), generator=g)), targets.copy_(torch.randint(0, 2, (T,), generator=g))
        pos.copy_(torch.randint(0, 400, pos.shape, generator=g)), ends.copy_(i32([h + 30 for h in held]))

    def results():
        torch.cuda.synchronize()
        return [x.clone() for x in (out, out2, mass, k2, v2, path, count, nxt)]

    def clear():
        for x in (out, out2, mass, k2, v2, path, count, nxt, mass2, pos2):
            x.zero_()

    load(cases[0], 70)
    step()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for i, case in enumerate(cases * 2):
        load(case, 71 + i)
        clear()
        step()
        want = results()
        clear()
        graph.replay()
        got = results()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    ops.check_async_errors(dev())


def test_a_run_of_them(ops):
    """Requests as they would be served, one layer: a prompt with its keys' weights, then steps that draft a tree, attend to it, confirm a
    path, and thin the cache to a budget; the plain forms go the same way beside it."""
    hq, hkv, hd, page, dtype, budget = 14, 2, 64, 16, torch.float32, 96
    g, rng = torch.Generator().manual_seed(81), random.Random(81)
    S, width, slots = 3, 12, 40 * page
    order = torch.randperm(36, generator=g).tolist()
    table = [order[s * width:(s + 1) * width] for s in range(S)]
    slot = lambda s, j: table[s][j // page] * page + j % page  # noqa: E731
    kc, vc = (torch.full((slots, hkv, hd), math.nan, device=dev()) for _ in range(2))
    mass, pos = torch.full((hkv, slots), math.nan, device=dev()), torch.zeros((hkv, slots), dtype=torch.int32, device=dev())
    rn = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    lens = [140, 40, 97]
    # what each request holds, in its places' order, for the plain side: lists per kv head of (key, value, mass, position)
    plain = [[[] for _ in range(hkv)] for _ in range(S)]
    held, ends = [0] * S, [0] * S

    def bring(rows):
        q, k, v = (rn(sum(rows), h, hd) for h in (hq, hkv, hkv))
        first = [sum(rows[:s]) for s in range(S)]
        for s in range(S):
            for i in range(rows[s]):
                kc[slot(s, held[s] + i)], vc[slot(s, held[s] + i)] = k[first[s] + i].to(dev()), v[first[s] + i].to(dev())
        return q, k, v, first

    def plain_rows(s, q, k, v, sees):
        out, weights = [], []
        for h in range(hkv):
            pk = torch.stack([e[0] for e in plain[s][h]] + list(k[:, h])) if plain[s][h] else k[:, h]
            pv = torch.stack([e[1] for e in plain[s][h]] + list(v[:, h])) if plain[s][h] else v[:, h]
            o, w = P.attention(q[:, h * 7:(h + 1) * 7], pk[:, None], pv[:, None], sees, hd ** -0.5)
            out.append(o)
            weights.append(w.sum((0, 1)))
        return torch.cat(out, 1), weights

    rows = lens
    for step in range(5):
        q, k, v, first = bring(rows)
        out = torch.zeros((sum(rows), hq * hd), device=dev())
        spans = (i32(first), i32(rows), i32(held), i32(table))
        if step % 2 == 0:          # a portion, or one token each
            ops.paged_attention_mass(q.reshape(-1, hq * hd).to(dev()), kc, vc, out, mass, *spans, page, hq, hkv, hd, hd ** -0.5, max(rows), mass_in=mass)
            for s, n in enumerate(rows):
                sees = torch.cat([torch.ones((n, held[s]), dtype=torch.bool), torch.ones((n, n), dtype=torch.bool).tril()], 1)
                a = slice(first[s], first[s] + n)
                want, w = plain_rows(s, q[a], k[a], v[a], sees)
                assert torch.allclose(out[a].cpu().double().reshape(n, hq, hd), want, atol=2e-5)
                for h in range(hkv):
                    for j, e in enumerate(plain[s][h]):
                        e[2] += float(w[h][j])
                    for i in range(n):
                        plain[s][h].append([k[first[s] + i, h], v[first[s] + i, h], float(w[h][held[s] + i]), ends[s] + i])
                for i in range(n):
                    pos[:, slot(s, held[s] + i)] = ends[s] + i
            held, ends = [h + n for h, n in zip(held, rows)], [e + n for e, n in zip(ends, rows)]
            for s in range(S):
                have = mass[:, [slot(s, j) for j in range(held[s])]].cpu().double()
                want = torch.tensor([[e[2] for e in plain[s][h]] for h in range(hkv)], dtype=torch.float64)
                assert torch.allclose(have, want, rtol=1e-4, atol=1e-6)
            ops.cache_evict(kc, vc, mass, pos, i32(held), i32(ends), i32(table), page, budget, 4, 16)
            for s in range(S):
                for h in range(hkv):
                    at = [slot(s, j) for j in range(held[s])]
                    # (the plain side's own sums: equal choices need sums further apart than the rounding, which random ones are)
                    for a, b in P.evict([e[2] for e in plain[s][h]], [e[3] for e in plain[s][h]], ends[s], budget, 4, 16):
                        plain[s][h][a] = list(plain[s][h][b])
                    del plain[s][h][budget:]
                    n = min(held[s], budget)
                    assert pos[h, at[:n]].tolist() == [e[3] for e in plain[s][h]]
                    assert torch.equal(kc[at[:n], h].cpu(), torch.stack([e[0] for e in plain[s][h]]))
            held = [min(h, budget) for h in held]
            rows = [9, 5, 12]
        else:
            parents = trees(rng, rows)
            tokens = [[rng.randrange(3) for _ in t] for t in parents]
            targets = [[rng.randrange(3) for _ in t] for t in parents]
            ops.tree_attention(q.reshape(-1, hq * hd).to(dev()), kc, vc, out, ops.tree_mask(parents).to(dev()), *spans, page, hq, hkv, hd, hd ** -0.5)
            path, count, nxt = i32([[0] * 12] * S), i32([0] * S), i32([0] * S)
            flat = [i32([x for t in lists for x in t]) for lists in (tokens, parents, targets)]
            ops.tree_commit(*flat, kc, vc, *spans, page, path, count, nxt)
            for s, n in enumerate(rows):
                a = slice(first[s], first[s] + n)
                sees = torch.cat([torch.ones((n, held[s]), dtype=torch.bool), P.ancestors(parents[s])], 1)
                want, _ = plain_rows(s, q[a], k[a], v[a], sees)
                assert torch.allclose(out[a].cpu().double().reshape(n, hq, hd), want, atol=2e-5)
                took, last = P.commit(tokens[s], parents[s], targets[s], 12)
                assert path[s].tolist()[:len(took)] == took and int(count[s]) == len(took) and int(nxt[s]) == last
                for d, node in enumerate(took):
                    for h in range(hkv):
                        plain[s][h].append([k[first[s] + node, h], v[first[s] + node, h], 0.0, ends[s] + d])
                    mass[:, slot(s, held[s] + d)] = 0.0
                    pos[:, slot(s, held[s] + d)] = ends[s] + d
                held[s], ends[s] = held[s] + len(took), ends[s] + len(took)
            rows = [1, 1, 1]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128)], ids=str)
@pytest.mark.parametrize("page", [4, 24, 32, 128])
def test_other_pages(ops, dtype, heads, page):
    """Pages that a tile of keys holds a part of, one of, or no whole number of."""
    held, rows = [0, 5, 131, 400, 23], [3, 1, 20, 7, 64]
    r = Requests(held, rows, heads, dtype, page, 91)
    mask = spread_mask(ops, r, trees(random.Random(6), rows))
    check_rows(r, run_tree(ops, r, mask), tree_sees(r, mask))
    mass_in = torch.rand((r.hkv, r.num_slots), generator=torch.Generator().manual_seed(92))
    got, mass = run_mass(ops, r, mass_in)
    check_mass(r, got, mass, mass_in, torch.full_like(mass_in, -5.0))
    r = Requests(held, [1] * 5, heads, dtype, page, 93)
    got, mass = run_mass(ops, r, None)
    check_mass(r, got, mass, None, torch.full((r.hkv, r.num_slots), -5.0))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_many_requests(ops, dtype):
    """More requests than a warp has lanes, and more jobs than there are blocks."""
    rng = random.Random(7)
    held, rows = [rng.randrange(0, 90) for _ in range(333)], [rng.choice([0, 1, 1, 2, 5, 11]) for _ in range(333)]
    r = Requests(held, rows, (14, 2, 64), dtype, 16, 94, gap=0)
    mask = spread_mask(ops, r, trees(rng, rows))
    check_rows(r, run_tree(ops, r, mask), tree_sees(r, mask))
    for n in (rows, [1] * 333):
        r = Requests(held, n, (14, 2, 64), dtype, 16, 95, gap=0)
        got, mass = run_mass(ops, r, None)
        check_mass(r, got, mass, None, torch.full((2, r.num_slots), -5.0))


def test_nothing_to_do(ops):
    for dtype in DTYPES:
        r = Requests([7, 9], [0, 0], (4, 2, 64), dtype, 16, 96)
        mask = torch.zeros((r.T, 1), dtype=torch.int64)
        assert bool((run_tree(ops, r, mask) == 7.0).all())
        got, mass = run_mass(ops, r, None, max_len=1)
        assert bool((got == 7.0).all()) and bool((mass == -5.0).all())
        got, mass = run_mass(ops, r, None, max_len=4)
        assert bool((got == 7.0).all()) and bool((mass == -5.0).all())
        r = Requests([], [], (4, 2, 64), dtype, 16, 97)
        assert run_tree(ops, r, torch.zeros((r.T, 1), dtype=torch.int64)).shape[0] == r.T


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_spans_beyond_their_tensors(ops, dtype):
    """Lengths that the rows, the mask, max_len or the block table have no room for are cut to what there is."""
    heads = (4, 2, 64)
    r = Requests([20], [12], heads, dtype, 16, 98, gap=0)
    mask = spread_mask(ops, r, trees(random.Random(1), r.rows))
    want, sees = run_tree(ops, r, mask), tree_sees(r, mask)
    r.rows = [4000]
    assert torch.equal(run_tree(ops, r, mask), want)
    r.rows, r.held = [12], [40]          # (two pages and one that is not there: 48 places)
    got = run_tree(ops, r, mask)
    assert bool((got[8:] == 7.0).all()) and bool((got[:8] != 7.0).any())
    r.rows, r.held = [12], [20]
    full, mass = run_mass(ops, r, None)
    r2 = Requests([20], [12], heads, dtype, 16, 98, gap=0)
    cut, mass_cut = run_mass(ops, r2, None, max_len=5)
    assert bool((cut[5:] == 7.0).all()) and bool((cut[:5] != 7.0).any())
    assert bool((mass_cut[:, r2.slots[0][25:]] == -5.0).all()) and bool((mass_cut[:, r2.slots[0][:25]] > 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_two_calls_at_once(ops, dtype):
    """Calls on two streams, and on another stream than the current one was, have scratch of their own."""
    rs = [Requests([900, 33], [20, 5], (12, 2, 128), dtype, 16, 101), Requests([1500, 77], [9, 40], (12, 2, 128), dtype, 16, 102)]
    masks = [spread_mask(ops, r, trees(random.Random(2), r.rows)) for r in rs]
    want = [run_tree(ops, r, m) for r, m in zip(rs, masks)]
    want_mass = [run_mass(ops, r, None) for r in rs]
    streams = [torch.cuda.Stream() for _ in rs]
    on = [[x.to(dev()) for x in (r.q.reshape(r.T, -1), r.k, r.v, m)] for r, m in zip(rs, masks)]
    args = [r.args() for r in rs]
    outs = [[torch.full((r.T, r.hq * r.hd), 7.0, dtype=dtype, device=dev()) for _ in range(2)] for r in rs]
    sums = [torch.full((r.hkv, r.num_slots), -5.0, device=dev()) for r in rs]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                q, k, v, m = on[i]
                ops.tree_attention(q, k, v, outs[i][0], m, *args[i])
                ops.paged_attention_mass(q, k, v, outs[i][1], sums[i], *args[i], max(rs[i].rows))
    torch.cuda.synchronize()
    ops.check_async_errors(dev())
    for i, r in enumerate(rs):
        assert torch.equal(outs[i][0].cpu().reshape(want[i].shape), want[i])
        assert torch.equal(outs[i][1].cpu().reshape(want[i].shape), want_mass[i][0]) and torch.equal(sums[i].cpu(), want_mass[i][1])


def test_one_request_twice(ops):
    """Requests that share their pages, as two drafts of one sequence do: reading is no matter."""
    r = Requests([300, 300], [9, 9], (14, 2, 64), torch.bfloat16, 16, 103)
    r.table[1], r.slots[1] = r.table[0], r.slots[0]
    rng = random.Random(3)
    mask = spread_mask(ops, r, trees(rng, r.rows))
    check_rows(r, run_tree(ops, r, mask), tree_sees(r, mask))


def test_strided_tensors_are_refused(ops):
    r = Requests([30], [4], (4, 2, 64), torch.bfloat16, 16, 104, gap=0)
    q, k, v = (x.to(dev()) for x in (r.q.reshape(4, -1), r.k, r.v))
    mask = ops.tree_mask([[-1, 0, 0, 1]]).to(dev())
    out = torch.empty((8, 256), dtype=torch.bfloat16, device=dev())[::2]
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.tree_attention(q, k, v, out, mask, *r.args())
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.cache_evict(k, v, torch.zeros((r.num_slots, 2), device=dev()).t(), torch.zeros((2, r.num_slots), dtype=torch.int32, device=dev()), i32([34]), i32([34]),
                        r.spans()[3], 16, 8, 0, 0)
    with pytest.raises(ops.KernelError, match="query heads a kv head"):
        ops.tree_attention(torch.zeros((4, 65 * 16), device=dev()), torch.zeros((r.num_slots, 1, 16), device=dev()), torch.zeros((r.num_slots, 1, 16), device=dev()),
                           torch.zeros((4, 65 * 16), device=dev()), mask, *r.spans(), 16, 65, 1, 16, 1.0)
    with pytest.raises(ops.KernelError, match="head size 260"):
        ops.tree_attention(torch.zeros((4, 260), device=dev()), torch.zeros((r.num_slots, 1, 260), device=dev()), torch.zeros((r.num_slots, 1, 260), device=dev()),
                           torch.zeros((4, 260), device=dev()), mask, *r.spans(), 16, 1, 1, 260, 1.0)


def test_caches_of_more_than_2_to_the_31_numbers(ops):
    """Pages at the end of planes whose offsets pass 32 bits."""
    hq, hkv, hd, page, dtype = 16, 8, 128, 16, torch.bfloat16
    r = Requests([300, 40], [9, 1], (hq, hkv, hd), dtype, page, 105)
    slots = (1 << 21) + (1 << 14)          # 2.2e9 numbers a plane
    move = slots // page - r.num_slots // page
    k, v = (torch.empty((slots, hkv, hd), dtype=dtype, device=dev()) for _ in range(2))
    k[-r.num_slots:], v[-r.num_slots:] = r.k.to(dev()), r.v.to(dev())
    table = i32([[p + move if p >= 0 else -1 for p in row] for row in r.table])
    args = (*r.spans()[:3], table, page, hq, hkv, hd, r.scale)
    q, out = r.q.reshape(r.T, -1).to(dev()), torch.full((r.T, hq * hd), 7.0, dtype=dtype, device=dev())
    parents = trees(random.Random(4), r.rows)
    mask = spread_mask(ops, r, parents)
    ops.tree_attention(q, k, v, out, mask.to(dev()), *args)
    check_rows(r, out.cpu().reshape(r.T, hq, hd), tree_sees(r, mask))
    mass, out = torch.full((hkv, slots), -5.0, device=dev()), torch.full_like(out, 7.0)
    ops.paged_attention_mass(q, k, v, out, mass, *args, 9)
    check_mass(r, out.cpu().reshape(r.T, hq, hd), mass[:, -r.num_slots:].cpu(), None, torch.full((hkv, r.num_slots), -5.0))
    held, ends = [309, 41], [400, 41]
    pos = torch.arange(slots, dtype=torch.int32, device=dev()).expand(hkv, slots).contiguous() % 300
    kr, vr, mr, pr = k[-r.num_slots:].cpu(), v[-r.num_slots:].cpu(), mass[:, -r.num_slots:].cpu(), pos[:, -r.num_slots:].cpu()
    ops.cache_evict(k, v, mass, pos, i32(held), i32(ends), table, page, 100, 4, 20)
    for h in range(hkv):
        for s, n in enumerate(held):
            at = r.slots[s][:n]
            for a, b in P.evict(mr[h, at].tolist(), pr[h, at].tolist(), ends[s], 100, 4, 20):
                for c in (kr, vr):
                    c[at[a], h] = c[at[b], h].clone()
    assert torch.equal(k[-r.num_slots:].cpu().nan_to_num(9.0), kr.nan_to_num(9.0)) and torch.equal(v[-r.num_slots:].cpu().nan_to_num(9.0), vr.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (3, 1, 32)], ids=str)
@pytest.mark.parametrize("what", ["query", "key"])
def test_weights_beside_a_row_of_nan(ops, dtype, heads, what):
    """A row whose scores are no numbers gives none to the keys that it sees, and leaves the other keys alone."""
    held, n, at = 90, 150, 77
    r = Requests([held, 20], [n, 3], heads, dtype, 16, 111)
    if what == "query":
        r.q[r.first[0] + at, 0] = math.nan
    else:
        r.k[r.slots[0][held + at], 0] = math.nan          # seen by the rows from its own on
    got, mass = run_mass(ops, r, None)
    for s in range(2):
        q, k, v = r.of(s)
        sees = torch.cat([torch.ones((r.rows[s], r.held[s]), dtype=torch.bool), torch.ones((r.rows[s],) * 2, dtype=torch.bool).tril()], 1)
        out, w = P.attention(q, k, v, sees, r.scale)
        sums = w.reshape(r.hkv, -1, w.shape[-1]).sum(1)
        have = mass[:, r.slots[s]].double()
        assert torch.equal(have.isnan(), sums.isnan()) and bool(have.isnan().any()) == (s == 0)
        fine = ~sums.isnan()
        # (the bound of the tests above, with the rows' number for the terms of a sum)
        rel = 2 * P.score_error(q, k, r.scale) + (r.rows[s] * r.hq // r.hkv + len(r.slots[s]) + 16) * 2.0 ** -24 + 2.0 ** -20
        assert bool(((have - sums).abs()[fine] <= rel * sums[fine]).all())
        rows = got[r.first[s]:r.first[s] + r.rows[s]].double()
        assert torch.equal(rows.isnan(), out.isnan())
