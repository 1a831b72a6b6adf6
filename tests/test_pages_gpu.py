"""Copies of pages, kept tokens and the pages' bookkeeping, to the bit against the definitions on lists."""

import random

import pytest
import torch

import draft_oracle as oracle
import fa
from fa import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF, BF, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cache(gen, pages, page, heads, d, dtype, spread=5):
    x = [torch.randn(pages, heads, page, d, generator=gen, device=DEV) for _ in "kv"]
    if dtype != E4M3:
        return fa.PagedKVCache(*(t.to(dtype) for t in x))
    scales = [2.0 ** torch.randint(-spread, spread, (pages, heads), generator=gen, device=DEV).float() for _ in "kv"]
    return fa.PagedKVCache(*((t * 40).to(E4M3) for t in x), *scales)


def _bits(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t.view(torch.int16)


# ----------------------------------------------------------------------------------------- keep


def _check_keep(cache, table, lengths, kept, tokens, counts=None, status=0):
    want = [oracle.keep(x, s, table, lengths, kept, counts, tokens) for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    new = fa.keep_tokens(cache, table, lengths, kept, tokens, counts=counts)
    assert new.tolist() == want[0][2] and new.dtype == torch.int32
    for (pool, scale, _), got, got_scale in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert scale is None or torch.equal(got_scale, scale)
        assert torch.equal(_bits(got), _bits(pool))
    assert _C.device_status(0, clear=True) == status


@pytest.mark.parametrize("dtype", [HALF, E4M3])
@pytest.mark.parametrize("page,heads,d,tokens,lengths,counts", [
    (16, 1, 64, 1, [1, 17], None), (8, 2, 128, 9, [9, 10, 16], None), (16, 3, 64, 61, [100, 61, 0, 90], [61, 30, 0, 1]),
    (64, 2, 128, 64, [64, 65, 127, 300], None), (8, 1, 64, 256, [256, 1000], [256, 200]), (256, 2, 128, 256, [400, 511], None),
    (32, 2, 128, 33, [50, 2000], [7, 33]),
])
def test_paths(page, heads, d, tokens, lengths, counts, dtype):
    gen, rng = torch.Generator(DEV).manual_seed(page + tokens), random.Random(tokens)
    per = -(-max(lengths) // page) + 1
    cache = _cache(gen, len(lengths) * per + 2, page, heads, d, dtype)
    table = torch.randperm(len(lengths) * per + 2, generator=gen, device=DEV)[: len(lengths) * per].view(-1, per).int()
    each = counts or [tokens] * len(lengths)
    for share in (0.1, 0.6, 1.0):  # few, many (sources among the targets), all: nothing moves
        kept = [sorted(rng.sample(range(n), int(round(share * n)))) for n in each]
        most = max(map(len, kept)) + (share < 1)
        if most == 0:
            continue
        kept = _ints([x + [-1] * (most - len(x)) for x in kept])
        _check_keep(cache, table, _ints(lengths), kept, tokens, None if counts is None else _ints(counts))


def test_no_path_and_no_tokens():
    cache = _cache(torch.Generator(DEV).manual_seed(0), 4, 16, 1, 64, E4M3)
    table, lengths = _ints([[0, 1], [2, 3]]), _ints([20, 5])
    _check_keep(cache, table, lengths, _ints([[-1, 3], [-1, -1]]), 4)
    assert fa.keep_tokens(cache, table, lengths, _ints([[], []]), 4).tolist() == [16, 1]
    assert fa.keep_tokens(cache, table, lengths, _ints([[], []]), 4, counts=_ints([9, -2])).tolist() == [16, 5]
    none = torch.empty(0, 2, dtype=torch.int32, device=DEV)
    assert fa.keep_tokens(cache, none, lengths[:0], none, 4).shape == (0,)


def test_bad_paths_end_and_are_reported():
    cache = _cache(torch.Generator(DEV).manual_seed(0), 6, 16, 2, 64, E4M3)
    table, lengths = _ints([[0, 1], [2, 3], [4, 5]]), _ints([20, 30, 31])
    for row in ([1, 3, 3, 5], [2, 1, -1, -1], [4, 8, -1, -1], [-7, 1, 2, 3], [0, 2**31 - 1, 3, 4]):
        _check_keep(cache, table, lengths, _ints([row, [1, 2, -1, -1], [0, 1, 2, 3]]), 8, status=32)


def test_places_that_do_not_exist_are_skipped():
    for dtype in (HALF, E4M3):
        cache = _cache(torch.Generator(DEV).manual_seed(0), 6, 16, 2, 64, dtype)
        kept = _ints([[1, 18, 30], [3, 20, 31], [0, 2, 20], [3, 20, 31]])
        # A page outside the pool, a missing one, more tokens than the table has places, fewer tokens than nodes.
        table, lengths = _ints([[0, 99], [-1, 1], [2, 3], [4, 5]]), _ints([32, 32, 50, 20])
        _check_keep(cache, table, lengths, kept, 32, status=32)
        _check_keep(cache, table, _ints([-(2**31), 2**31 - 1, 0, 32]), kept, 32, status=32)


def test_strided_pools_and_one_path_for_all():
    gen = torch.Generator(DEV).manual_seed(1)
    both = (torch.randn(7, 2, 3, 16, 64, generator=gen, device=DEV) * 40).to(E4M3)
    scales = [2.0 ** torch.randint(-3, 3, (7, 3), generator=gen, device=DEV).float() for _ in "kv"]
    cache = fa.PagedKVCache(both[:, 0], both[:, 1], *scales)
    _check_keep(cache, _ints([[6, 2, 0], [1, 3, 5]]), _ints([40, 47]), _ints([1, 4, 9, 20, -1]).expand(2, 5), 24)


def test_keep_in_a_graph():
    gen = torch.Generator(DEV).manual_seed(2)
    cache = _cache(gen, 6, 16, 2, 64, E4M3)
    table, lengths, kept = _ints([[0, 1, 2], [3, 4, 5]]), _ints([40, 30]), _ints([[2, 7], [1, -1]])
    fa.keep_tokens(cache, table, lengths, kept, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = fa.keep_tokens(cache, table, lengths, kept, 8)
    for seed in (3, 4):
        lengths.copy_(_ints([33 + seed, 20 * (seed - 2)]))
        kept.copy_(_ints([[0, seed], [seed, 7]]))
        want = [oracle.keep(x, s, table, lengths, kept, None, 8) for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
        graph.replay()
        assert new.tolist() == want[0][2] and torch.equal(_bits(cache.k), _bits(want[0][0])) and torch.equal(_bits(cache.v), _bits(want[1][0]))


# ----------------------------------------------------------------------------------------- copy


@pytest.mark.parametrize("dtype,page,heads,d,n", [(HALF, 8, 1, 64, 1), (BF, 16, 3, 64, 7), (E4M3, 8, 2, 64, 5), (E4M3, 64, 8, 128, 40), (HALF, 256, 2, 128, 3)])
def test_copies(dtype, page, heads, d, n):
    gen = torch.Generator(DEV).manual_seed(n)
    cache = _cache(gen, 2 * n + 3, page, heads, d, dtype)
    order = torch.randperm(2 * n + 3, generator=gen, device=DEV).int()
    src, dst = order[:n].contiguous(), order[n : 2 * n].contiguous()
    src[0] = src[n // 2]  # one page to several
    if n > 4:
        src[2], dst[3] = -1, -5
    pools = [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    want = [t.clone() for t in pools]
    for a, z in zip(src.tolist(), dst.tolist()):
        for t in want:
            if a >= 0 and z >= 0:
                (t.view(torch.uint8) if t.dtype == E4M3 else t)[z] = (t.view(torch.uint8) if t.dtype == E4M3 else t)[a]
    fa.copy_pages(cache, src, dst)
    assert all(torch.equal(t.view(torch.uint8), w.view(torch.uint8)) for t, w in zip(pools, want)) and _C.device_status(0, clear=True) == 0
    src[0] = 2 * n + 3
    before = cache.k.clone()
    fa.copy_pages(cache, src[:1], dst[:1])
    fa.copy_pages(cache, dst[:1], src[:1])
    fa.copy_pages(cache, src[:0], dst[:0])
    assert torch.equal(cache.k.view(torch.uint8), before.view(torch.uint8)) and _C.device_status(0, clear=True) == 32


def test_copy_between_strided_pages():
    both = torch.randn(5, 2, 3, 16, 64, device=DEV).to(HALF)
    want = both.clone()
    want[4] = both[1]
    fa.copy_pages(fa.PagedKVCache(both[:, 0], both[:, 1]), _ints([1]), _ints([4]))
    assert torch.equal(both, want)


# ---------------------------------------------------------------------------------- bookkeeping


def _same(refs, pages, table, rows):
    assert refs.tolist() == pages.refs and table.tolist() == rows


@pytest.mark.parametrize("seed,num_pages,batch,width,page,tokens", [
    (0, 40, 3, 8, 8, 1), (1, 300, 9, 20, 16, 5), (2, 64, 4, 12, 8, 40), (3, 9000, 700, 12, 8, 3), (4, 5000, 1500, 3, 256, 2), (5, 100000, 40, 300, 16, 2100),
])
def test_steps_of_many_sequences(seed, num_pages, batch, width, page, tokens):
    """Random forks, frees and reservations, scarce pages among them, against the lists."""
    rng = random.Random(seed)
    refs = torch.zeros(num_pages, dtype=torch.int32, device=DEV)
    pages = oracle.Pages(refs.tolist())
    rows = [[-1] * width for _ in range(batch)]
    table = _ints(rows)
    lengths = [0] * batch
    for step in range(12):
        counts = [rng.randint(0, tokens) if step % 3 else min(tokens, 1) for _ in range(batch)]
        counts = [min(c, width * page - n) for c, n in zip(counts, lengths)]
        wanted = [n + c for n, c in zip(lengths, counts)]
        got = fa.reserve_pages(refs, table, _ints(wanted), tokens, page, counts=_ints(counts))
        want = pages.reserve(rows, wanted, tokens, page, counts)
        assert [x.tolist() for x in got] == [*want] and got[0].dtype == torch.bool
        _same(refs, pages, table, rows)
        lengths = [w if ok else n for w, n, ok in zip(wanted, lengths, want[0])]
        if step % 4 == 1:  # new sequences from old ones, the old ones given back
            parents = [rng.randrange(-1, batch) for _ in range(batch)]
            new, new_rows = fa.fork_pages(refs, table, _ints(parents)), pages.fork(rows, parents)
            _same(refs, pages, new, new_rows)
            fa.free_pages(refs, table)
            pages.free(rows)
            _same(refs, pages, table, rows)
            table, rows, lengths = new, new_rows, [lengths[p] if p >= 0 else 0 for p in parents]
        if step % 4 == 3:  # some shortened
            lengths = [rng.choice([n, n // 2, 0]) for n in lengths]
            keep = [-(-n // page) for n in lengths]
            fa.free_pages(refs, table, _ints(keep))
            pages.free(rows, keep)
            _same(refs, pages, table, rows)
    assert _C.device_status(0, clear=True) == 0


def test_a_long_prompt():
    """Thousands of entries of one row, some of them shared, beside rows that need one or none."""
    refs, table = torch.zeros(9000, dtype=torch.int32, device=DEV), torch.full((3, 6500), -1, dtype=torch.int32, device=DEV)
    refs[5], refs[7000], refs[17] = 2, 3, 1
    table[1, 0], table[1, 6000], table[0, 0] = 5, 7000, 17
    pages, rows, lengths, counts = oracle.Pages(refs.tolist()), table.tolist(), [9, 6400 * 8 + 3, 40], [1, 6400 * 8, 0]
    got = fa.reserve_pages(refs, table, _ints(lengths), 6400 * 8, 8, counts=_ints(counts))
    want = pages.reserve(rows, lengths, 6400 * 8, 8, counts)
    assert [x.tolist() for x in got] == [*want] and all(want[0]) and want[1][1] == 5
    _same(refs, pages, table, rows)


def test_too_few_pages():
    refs, table = _ints([0, 1, 0, 0, 1]), _ints([[1, -1, -1], [4, -1, -1], [-1, -1, -1], [-1, -1, -1]])
    # Two pages, none, two of the one that is left, and one.
    granted, src, dst = fa.reserve_pages(refs, table, _ints([24, 5, 16, 3]), 20, 8, counts=_ints([18, 1, 16, 3]))
    assert granted.tolist() == [True, True, False, False] and table.tolist() == [[1, 0, 2], [4, -1, -1], [-1] * 3, [-1] * 3]
    assert refs.tolist() == [1, 1, 1, 0, 1] and src.tolist() == dst.tolist() == [-1] * 4
    assert fa.reserve_pages(refs, table, _ints([24, 5, 16, 3]), 20, 8, counts=_ints([0, 0, 0, 3]))[0].all()
    assert table[3].tolist() == [3, -1, -1] and _C.device_status(0, clear=True) == 0


def test_rows_that_do_not_fit_and_bad_entries():
    refs, table = _ints([0, 0, 1, 0]), _ints([[2, 77], [-9, -1], [-1, -1], [-1, -1]])
    granted, src, dst = fa.reserve_pages(refs, table, _ints([12, 3, 17, 2]), 4, 8, counts=_ints([4, 3, 3, 3]))
    assert granted.tolist() == [True, True, False, False] and table.tolist() == [[2, 0], [1, -1], [-1, -1], [-1, -1]]
    assert refs.tolist() == [1, 1, 1, 0] and src.tolist() == dst.tolist() == [-1] * 4 and _C.device_status(0, clear=True) == 32
    extreme = fa.reserve_pages(refs, table, _ints([2**31 - 1, -(2**31), -1, 0]), 4, 8)[0]
    assert not extreme.any() and refs.tolist() == [1, 1, 1, 0] and _C.device_status(0, clear=True) == 32
    forked = fa.fork_pages(refs, _ints([[2, 9], [-2, 3]]), _ints([0, 1, 2, -1, -3]))
    assert forked.tolist() == [[2, -1], [-1, 3], [-1, -1], [-1, -1], [-1, -1]] and refs.tolist() == [1, 1, 2, 1]
    assert _C.device_status(0, clear=True) == 32
    twice = _ints([[3, 3, 2], [2, 2, 44]])
    fa.free_pages(refs, twice)
    assert refs.tolist() == [1, 1, 0, 0] and (twice == -1).all() and _C.device_status(0, clear=True) == 32


def test_two_children_share_a_page():
    """Both get copies of it; it is free for the next call, not for this one."""
    refs, table = _ints([0, 2, 0, 0]), _ints([[1, -1], [1, -1]])
    granted, src, dst = fa.reserve_pages(refs, table, _ints([6, 5]), 1, 8)
    assert granted.all() and src.tolist() == [1, 1] and dst.tolist() == [0, 2] and table[:, 0].tolist() == [0, 2]
    assert refs.tolist() == [1, 0, 1, 0]
    assert fa.reserve_pages(refs, table, _ints([16, 16]), 8, 8)[0].all() and table.tolist() == [[0, 1], [2, 3]]


def test_bookkeeping_in_a_graph():
    refs, table, lengths, rows = torch.zeros(64, dtype=torch.int32, device=DEV), torch.full((4, 6), -1, dtype=torch.int32, device=DEV), _ints([7, 9, 1, 0]), _ints([0, 0, 2, 1])

    def step():
        lengths.add_(3)
        granted, src, dst = fa.reserve_pages(refs, table, lengths, 3, 8)
        new = fa.fork_pages(refs, table, rows)
        fa.free_pages(refs, table)
        table.copy_(new)
        return granted, src, dst

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        granted, src, dst = step()
    pages, lists, now = oracle.Pages(refs.tolist()), table.tolist(), lengths.tolist()
    for _ in range(4):
        graph.replay()
        now = [n + 3 for n in now]
        want = pages.reserve(lists, now, 3, 8)
        new = pages.fork(lists, rows.tolist())
        pages.free(lists)
        lists = new
        assert (granted.tolist(), src.tolist(), dst.tolist()) == want
        _same(refs, pages, table, lists)
    # Tables with rows apart, on another stream.
    wide = torch.full((3, 9), -1, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fa.reserve_pages(refs, wide[:, :4], _ints([9, 1, 17]), 20, 8, counts=_ints([9, 1, 17]))
    side.synchronize()
    want = [[-1] * 4 for _ in range(3)]
    pages.reserve(want, [9, 1, 17], 20, 8, [9, 1, 17])
    assert wide[:, :4].tolist() == want and (wide[:, 4:] == -1).all() and refs.tolist() == pages.refs


def test_refused():
    refs, table, rows = _ints([0, 0]), _ints([[0, 1]]), _ints([0])
    for bad, match in ((lambda: fa.fork_pages(refs.long(), table, rows), "refs"), (lambda: fa.fork_pages(refs, table[0], rows), "page_table"),
                       (lambda: fa.fork_pages(refs, table.mT, rows.expand(2)), "contiguous rows|rows must be"), (lambda: fa.free_pages(refs, table, _ints([0, 1])), "keep"),
                       (lambda: fa.reserve_pages(refs, table, rows.long(), 1, 8), "lengths"), (lambda: fa.reserve_pages(refs, table, rows, 1, 8, counts=_ints([1, 2])), "counts")):
        with pytest.raises(RuntimeError, match=match):
            bad()
    for bad, match in ((lambda: fa.reserve_pages(refs, table, rows, 1, 12), "power of two"), (lambda: fa.reserve_pages(refs, table, rows, -1, 8), "tokens"),
                       (lambda: fa.reserve_pages(refs, table, rows, 2**40, 8), "32-bit"), (lambda: fa.free_pages(refs, table.expand(3, 2)), "a row apart")):
        with pytest.raises(ValueError, match=match):
            bad()
    cache = fa.PagedKVCache.empty(2, 8, 1, 64)
    for bad, match in ((lambda: fa.copy_pages(cache, rows, rows.long()), "src and dst"), (lambda: fa.copy_pages(cache, rows, refs), "src and dst"),
                       (lambda: fa.keep_tokens(cache, table, rows, rows, 1), "kept"), (lambda: fa.keep_tokens(cache, table, rows, _ints([[0], [1]]), 1), "kept")):
        with pytest.raises(RuntimeError, match=match):
            bad()
    with pytest.raises(ValueError, match="256"):
        fa.keep_tokens(cache, table, rows, _ints([[0]]), 300)
