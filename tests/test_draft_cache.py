"""What the operators of a cache that is drafted into and thinned out refuse, and the masks of trees; no GPU needed."""
import pytest
import torch

from lightllm_b200.csrc import ops
from tests.plain import draft_cache_plain as P


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def tree_args(**kw):
    a = dict(q=torch.zeros(6, 4 * 16), k=torch.zeros(32, 2, 16), v=torch.zeros(32, 2, 16), out=torch.zeros(6, 64), mask=torch.zeros((6, 1), dtype=torch.int64),
             row=i32(2), len=i32(2), pos=i32(2), table=i32(2, 3), page=8, hq=4, hkv=2, hd=16, scale=0.25)
    a.update(kw)
    return list(a.values())


def mass_args(**kw):
    a = dict(q=torch.zeros(6, 64), k=torch.zeros(32, 2, 16), v=torch.zeros(32, 2, 16), out=torch.zeros(6, 64), mass=torch.zeros(2, 32),
             row=i32(2), len=i32(2), pos=i32(2), table=i32(2, 3), page=8, hq=4, hkv=2, hd=16, scale=0.25, max_len=3, mass_in=None)
    a.update(kw)
    return list(a.values())


def commit_args(**kw):
    a = dict(tokens=i32(6), parents=i32(6), targets=i32(6), k=torch.zeros(3, 32, 2, 16), v=torch.zeros(3, 32, 2, 16), row=i32(2), len=i32(2), pos=i32(2),
             table=i32(2, 3), page=8, path=i32(2, 4), count=i32(2), next=i32(2))
    a.update(kw)
    return list(a.values())


def evict_args(**kw):
    a = dict(k=torch.zeros(3, 32, 2, 16), v=torch.zeros(3, 32, 2, 16), mass=torch.zeros(3, 2, 32), positions=i32(3, 2, 32), lengths=i32(2), ends=i32(2),
             table=i32(2, 3), page=8, budget=8, first=2, latest=4, mass_out=None, positions_out=None)
    a.update(kw)
    return list(a.values())


MASK = torch.zeros((6, 1), dtype=torch.int64)


@pytest.mark.parametrize("call,args,word", [
    (ops.tree_attention, tree_args(hq=3), "multiple"), (ops.tree_attention, tree_args(out=torch.zeros(5, 64)), "q and out"),
    (ops.tree_attention, tree_args(out=torch.zeros(6, 64).bfloat16()), "q and out"), (ops.tree_attention, tree_args(k=torch.zeros(32, 2, 8)), "caches"),
    (ops.tree_attention, tree_args(v=torch.zeros(32, 2, 16).bfloat16()), "caches"), (ops.tree_attention, tree_args(mask=MASK.int()), "mask"),
    (ops.tree_attention, tree_args(mask=MASK[:5]), "mask"), (ops.tree_attention, tree_args(mask=MASK[:, :0]), "mask"),
    (ops.tree_attention, tree_args(row=i32(3)), "index arrays"), (ops.tree_attention, tree_args(pos=i32(2).long()), "index arrays"),
    (ops.tree_attention, tree_args(table=i32(3, 3)), "block_table"), (ops.tree_attention, tree_args(page=0), "page size"),
    (ops.tree_attention, tree_args(q=torch.zeros(6, 64).half(), out=torch.zeros(6, 64).half(), k=torch.zeros(32, 2, 16).half(), v=torch.zeros(32, 2, 16).half()), "float16"),
    (ops.tree_attention, tree_args(), "no CPU path"),
    (ops.paged_attention_mass, mass_args(mass=torch.zeros(32, 2)), "weights"), (ops.paged_attention_mass, mass_args(mass=torch.zeros(2, 32).double()), "weights"),
    (ops.paged_attention_mass, mass_args(mass_in=torch.zeros(2, 31)), "weights"), (ops.paged_attention_mass, mass_args(max_len=0), "max_len"),
    (ops.paged_attention_mass, mass_args(), "no CPU path"),
    (ops.tree_commit, commit_args(tokens=i32(6).long()), "tokens"), (ops.tree_commit, commit_args(parents=i32(5)), "tokens"),
    (ops.tree_commit, commit_args(path=i32(3, 4)), "path"), (ops.tree_commit, commit_args(v=torch.zeros(2, 32, 2, 16)), "one shape"),
    (ops.tree_commit, commit_args(count=i32(1)), "count"), (ops.tree_commit, commit_args(), "no CPU path"),
    (ops.cache_evict, evict_args(mass=torch.zeros(2, 32)), "mass is float32"), (ops.cache_evict, evict_args(positions=torch.zeros(3, 2, 32)), "positions int32"),
    (ops.cache_evict, evict_args(budget=5), "does not hold"), (ops.cache_evict, evict_args(budget=0, first=0, latest=0), "does not hold"),
    (ops.cache_evict, evict_args(first=-1), "does not hold"), (ops.cache_evict, evict_args(mass_out=torch.zeros(3, 2, 32)), "both or neither"),
    (ops.cache_evict, evict_args(k=torch.zeros(32, 2, 16)), "one shape"), (ops.cache_evict, evict_args(), "no CPU path"),
])
def test_refusals(call, args, word):
    with pytest.raises(ops.KernelError, match=word):
        call(*args)


def test_shared_planes_are_refused():
    k = torch.zeros(3, 32, 2, 16)
    with pytest.raises(ops.KernelError, match="planes of their own"):
        ops.tree_commit(*commit_args(k=k, v=k))
    with pytest.raises(ops.KernelError, match="planes of their own"):
        ops.cache_evict(*evict_args(k=k, v=k))


@pytest.mark.parametrize("call,args", [(ops.tree_attention, tree_args), (ops.paged_attention_mass, mass_args)])
def test_results_over_the_queries_are_refused(call, args):
    """Blocks read a job's queries at different times, some of them when others have written its results."""
    both = torch.zeros(7, 64)
    for q, out in ((both[:6], both[:6]), (both[:6], both[1:]), (both[1:], both[:6])):
        with pytest.raises(ops.KernelError, match="must not lie over q"):
            call(*args(q=q, out=out))
    twice = torch.zeros(12, 64)
    with pytest.raises(ops.KernelError, match="no CPU path"):          # side by side is fine
        call(*args(q=twice[:6], out=twice[6:]))


@pytest.mark.parametrize("call,args,word", [
    (ops.tree_attention, tree_args(page=1 << 40), "page size"), (ops.paged_attention_mass, mass_args(page=1 << 40), "page size"),
    (ops.tree_commit, commit_args(page=1 << 40), "page size"), (ops.cache_evict, evict_args(page=1 << 40), "page size"),
    (ops.cache_evict, evict_args(budget=1 << 40), "32 bits"), (ops.paged_attention_mass, mass_args(max_len=1 << 40), "no CPU path"),
])
def test_numbers_of_more_than_32_bits(call, args, word):
    """No count is cut to 32 bits: it is refused, or (rows a request) means no more than the rows that there are."""
    with pytest.raises(ops.KernelError, match=word):
        call(*args)


def test_tree_masks():
    trees = [[-1], [-1, 0, 0, 1, 3], [], [-1] + list(range(129))]
    mask = ops.tree_mask(trees)
    assert mask.shape == (136, 3) and mask.dtype == torch.int64
    at = 0
    for tree in trees:
        sees = P.ancestors(tree)
        for i in range(len(tree)):
            for j in range(192):
                assert bool((int(mask[at + i, j // 64]) >> (j % 64)) & 1) == (j < len(tree) and bool(sees[i, j]))
        at += len(tree)
    for bad in ([[0]], [[-1, 1]], [[-1, -1]], [[-1, 2, 0]]):
        with pytest.raises(ValueError, match="parent"):
            ops.tree_mask(bad)
    assert ops.tree_mask([]).shape == (0, 1)
