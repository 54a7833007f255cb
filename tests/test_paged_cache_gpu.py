"""mcCacheReserve and mcCacheRelease against bookkeeping in Python lists."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def A(gpu_mode):
    from minicaffe import attention
    return attention


def ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def plain_reserve(block, width, max_tokens, cached, new, table, free):
    """Request by request; the pool is used up for all once one cannot be served from it."""
    table, free = [list(t) for t in table], list(free)
    contexts, starts, slots, positions, denied, asked, pool = [], [0], [], [], 0, 0, len(free)
    for r, (c, n) in enumerate(zip(cached, new)):
        have, need = -(-c // block), -(-(c + n) // block)
        ok = need <= width
        if ok:
            asked += need - have
            ok = need == have or asked <= pool
        if ok:
            for j in range(have, need):
                table[r][j] = free.pop()
        denied += not ok
        contexts.append(c + n if ok else c)
        starts.append(starts[-1] + n)
        for p in range(c, c + n):
            slots.append(table[r][p // block] * block + p % block if ok else -1)
            positions.append(p)
    slots, positions = slots[:max_tokens], positions[:max_tokens]
    pad = max_tokens - len(slots)
    return table, contexts, starts, slots + [-1] * pad, positions + [0] * pad, len(free), denied


def reserve(A, block, width, max_tokens, cached, new, table, free, spare=3):
    n = len(cached)
    d = dict(cached=ints(cached), new=ints(new), table=ints(table).reshape(n, width), contexts=ints([-7] * n),
             starts=ints([-7] * (n + 1)), slots=ints([-7] * max_tokens), positions=ints([-7] * max_tokens),
             free=ints(list(free) + [-5] * spare), count=ints([len(free)]), left=ints([-7]), denied=ints([-7]))
    A.cache_reserve(n, block, width, max_tokens, len(free) + spare, *[d[k].data_ptr() for k in (
        "cached", "new", "free", "count", "table", "contexts", "starts", "slots", "positions", "left", "denied")])
    torch.cuda.synchronize()
    assert d["free"].tolist() == list(free) + [-5] * spare and d["count"].item() == len(free)
    return (d["table"].tolist(), d["contexts"].tolist(), d["starts"].tolist(), d["slots"].tolist(), d["positions"].tolist(),
            d["left"].item(), d["denied"].item())


def random_case(seed, requests, block, longest_new, longest_cached, slack):
    r = np.random.default_rng(seed)
    cached = r.integers(0, longest_cached + 1, requests)
    new = r.integers(0, longest_new + 1, requests)
    have, need = -(-cached // block), -(-(cached + new) // block)
    width = max(1, int(need.max()))
    blocks = r.permutation(int(need.sum()) + 50)
    table = np.full((requests, width), -1)
    at = 0
    for i, n in enumerate(have):
        table[i, :n] = blocks[at:at + n]
        at += n
    free = blocks[at:at + max(0, int((need - have).sum()) + slack)]
    return width, cached.tolist(), new.tolist(), table.tolist(), free.tolist()


@pytest.mark.parametrize("requests", [1, 2, 63, 64, 65, 256, 257, 1000, 4096])
@pytest.mark.parametrize("block", [1, 16, 24])
@pytest.mark.parametrize("kind", ["step", "prompts", "chunks", "short of blocks"])
def test_against_lists(A, requests, block, kind):
    new, cached = {"step": (1, 200), "prompts": (40, 0), "chunks": (9, 60), "short of blocks": (20, 30)}[kind]
    for seed in (1, 2):
        width, c, n, table, free = random_case(seed, requests, block, new, cached, -5 if kind == "short of blocks" else 7)
        for max_tokens in (sum(n), sum(n) + 300, sum(n) // 2):
            want = plain_reserve(block, width, max_tokens, c, n, table, free)
            assert reserve(A, block, width, max_tokens, c, n, table, free) == want


def test_a_table_that_is_not_wide_enough(A):
    c, n, table, free = [30, 3, 0], [3, 2, 40], [[5, 6], [7, -1], [-1, -1]], [10, 11, 12]
    want = plain_reserve(16, 2, 50, c, n, table, free)
    assert want[-1] == 2
    assert reserve(A, 16, 2, 50, c, n, table, free) == want


def test_lengths_that_cannot_be(A):
    """Negative lengths count as none; enormous ones are denied, and the others served or denied by the rule."""
    got = reserve(A, 16, 2, 20, [-5, 3, 0, 7], [4, -2, 2 ** 31 - 1, 5], [[-1, -1], [1, -1], [-1, -1], [2, -1]], [8, 9])
    table, contexts, starts, slots, positions, left, denied = got
    assert contexts == [4, 3, 0, 12] and denied == 1 and left == 1 and table[0] == [9, -1]
    assert slots[:4] == [144, 145, 146, 147] and slots[4:] == [-1] * 16 and starts[:3] == [0, 4, 4]


def test_no_requests(A):
    assert reserve(A, 16, 1, 5, [], [], [], [3, 4]) == ([], [], [0], [-1] * 5, [0] * 5, 2, 0)


def test_release_and_reserve_again(A):
    block, width = 16, 4
    contexts, table = ints([40, 17, 0, 64]), ints([[1, 2, 3, -1], [4, 5, -1, -1], [-1] * 4, [6, 7, 8, 9]])
    free, count, left = ints([20, 21] + [-5] * 10), ints([2]), ints([0])
    ended = ints([1, 0, 1, 1])
    A.cache_release(4, block, width, 12, ended.data_ptr(), table.data_ptr(), contexts.data_ptr(), free.data_ptr(),
                    count.data_ptr(), left.data_ptr())
    torch.cuda.synchronize()
    assert left.item() == 9 and contexts.tolist() == [0, 17, 0, 0]
    assert free.tolist() == [20, 21, 1, 2, 3, 6, 7, 8, 9, -5, -5, -5]
    # in place, and with less room than comes back
    contexts, ended, table = ints([64]), ints([1]), ints([[11, 12, 13, 14]])
    A.cache_release(1, block, width, 11, ended.data_ptr(), table.data_ptr(), contexts.data_ptr(), free.data_ptr(), left.data_ptr(),
                    left.data_ptr())
    torch.cuda.synchronize()
    assert left.item() == 11 and free.tolist()[9:] == [11, 12, -5]


@pytest.mark.parametrize("requests", [255, 256, 257, 700])
def test_release_many(A, requests):
    r = np.random.default_rng(3)
    contexts = r.integers(0, 100, requests)
    finished = r.integers(0, 2, requests)
    table = r.permutation(requests * 7).reshape(requests, 7)
    free, count, c = ints([0] * (requests * 7 + 3)), ints([3]), ints(contexts)
    ended, blocks = ints(finished), ints(table)
    A.cache_release(requests, 16, 7, len(free), ended.data_ptr(), blocks.data_ptr(), c.data_ptr(), free.data_ptr(), count.data_ptr(),
                    count.data_ptr())
    torch.cuda.synchronize()
    want = [0] * 3 + [b for i in range(requests) if finished[i] for b in table[i, :-(-contexts[i] // 16)]]
    assert count.item() == len(want) and free.tolist()[:len(want)] == want
    assert c.tolist() == np.where(finished, 0, contexts).tolist()


def test_captured_steps_replay(A):
    """Steps of text in a graph: two calls a replay, the pool's count handed from one to the other and back."""
    n, block, width = 3, 4, 10
    new, table, free = ints([1] * n), ints(np.full((n, width), -1)), ints(range(30, 0, -1))
    lens = [ints([0] * n), ints([0] * n)]
    counts = [ints([30]), ints([0])]
    starts, slots, positions, denied = ints([0] * (n + 1)), ints([0] * n), ints([0] * n), ints([0])

    def step(i, stream):
        A.cache_reserve(n, block, width, n, 30, lens[i].data_ptr(), new.data_ptr(), free.data_ptr(), counts[i].data_ptr(), table.data_ptr(),
                        lens[1 - i].data_ptr(), starts.data_ptr(), slots.data_ptr(), positions.data_ptr(), counts[1 - i].data_ptr(),
                        denied.data_ptr(), stream=stream)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(0, s.cuda_stream)
            step(1, s.cuda_stream)
    seen = set()
    for i in range(15):
        graph.replay()
        torch.cuda.synchronize()
        assert lens[0].tolist() == [2 * (i + 1)] * n and counts[0].item() == 30 - n * -(-2 * (i + 1) // block) and denied.item() == 0
        assert positions.tolist() == [2 * i + 1] * n
        assert not seen & set(slots.tolist())
        seen |= set(slots.tolist())


def test_refusals(A):
    from minicaffe import MiniCaffeError
    here, there = ints([0] * 64), ints([0] * 64)
    x, y = here.data_ptr(), there.data_ptr()

    def call(n=2, block=16, width=4, tokens=8, capacity=8, cached=x, contexts=y, count=x, left=y, slots=y):
        A.cache_reserve(n, block, width, tokens, capacity, cached, x, x, count, y, contexts, y, slots, y, left, y)

    for kw, word in ((dict(n=-1), "requests"), (dict(n=4097), "requests"), (dict(block=0), "block"), (dict(width=0), "width"),
                     (dict(tokens=-1), "possible"), (dict(tokens=2 ** 23), "possible"), (dict(capacity=2 ** 23), "possible"),
                     (dict(cached=None), "null"), (dict(count=None), "null"), (dict(slots=None), "null"), (dict(left=x), "free_left"),
                     (dict(contexts=x), "cached_lens")):
        with pytest.raises(MiniCaffeError, match=word):
            call(**kw)
    for kw in (dict(n=-1), dict(block=0), dict(capacity=-1)):
        a = dict(n=2, block=16, width=4, capacity=8)
        a.update(kw)
        with pytest.raises(MiniCaffeError, match="extents"):
            A.cache_release(a["n"], a["block"], a["width"], a["capacity"], x, x, y, y, x, y)
    with pytest.raises(MiniCaffeError, match="null"):
        A.cache_release(2, 16, 4, 8, None, x, y, y, x, y)
