"""mcAttentionPacked and mcAttentionPaged against attention in 64 bits (attention_ref.py)."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from attention_ref import TYPES, check, rows64  # noqa: E402


@pytest.fixture(scope="module")
def A(gpu_mode):
    from minicaffe import attention
    return attention


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def starts_of(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def randn(g, *shape, kind="f32"):
    return torch.randn(shape, generator=g, device="cuda").to(TYPES[kind])


def packed(A, q, k, v, q_lens, k_lens, causal, scale=None, out=None):
    scale = scale or 1 / math.sqrt(q.shape[2])
    kind = [n for n, t in TYPES.items() if t == q.dtype][0]
    geom = A.AttentionGeom(A.TYPES[kind], q.shape[1], k.shape[1], q.shape[2], int(causal), scale)
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda") if out is None else out
    lse = torch.full((q.shape[1], q.shape[0]), float("nan"), device="cuda")
    qs, ks = ints(starts_of(q_lens)), ints(starts_of(k_lens))
    A.attention_packed(geom, A.heads_of(q), A.heads_of(k), A.heads_of(v), qs.data_ptr(), ks.data_ptr(), len(q_lens), len(q),
                       len(k), A.heads_of(out), lse=lse.data_ptr())
    torch.cuda.synchronize()
    return out, lse


def check_packed(q, k, v, q_lens, k_lens, causal, out, lse, scale=None):
    scale = scale or 1 / math.sqrt(q.shape[2])
    kind = [n for n, t in TYPES.items() if t == q.dtype][0]
    qs, ks = starts_of(q_lens), starts_of(k_lens)
    group = q.shape[1] // k.shape[1]
    for i, (nq, nk) in enumerate(zip(q_lens, k_lens)):
        if nq == 0:
            continue
        seen = [max(0, min(nk, nk - nq + r + 1)) if causal else nk for r in range(nq)]
        kv = slice(ks[i], ks[i + 1])
        for h in range(q.shape[1]):
            rows = slice(qs[i], qs[i + 1])
            want = rows64(q[rows, h], k[kv, h // group], v[kv, h // group], scale, seen)
            check(kind, q.shape[2], nk, out[rows, h], lse[h, rows], want, float(v.abs().max()) if v.numel() else 0.0)


# lengths around the tiles' edges, empty sequences among them
LENGTHS = [[1], [2, 1, 3], [31, 0, 33], [64], [65, 1, 127], [0, 128, 0], [129, 17], [257]]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_packed_lengths(A, kind, causal, lengths):
    g = torch.Generator(device="cuda").manual_seed(1)
    n = sum(lengths)
    q, k, v = (randn(g, n, h, 64, kind=kind) for h in (2, 1, 1))
    out, lse = packed(A, q, k, v, lengths, lengths, causal)
    check_packed(q, k, v, lengths, lengths, causal, out, lse)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 80, 96, 104, 128, 136, 160, 192, 200, 248, 256])
def test_packed_head_sizes(A, kind, dim):
    g = torch.Generator(device="cuda").manual_seed(2)
    lengths = [37, 100]
    q, k, v = (randn(g, 137, h, dim, kind=kind) for h in (3, 1, 1))
    out, lse = packed(A, q, k, v, lengths, lengths, True)
    check_packed(q, k, v, lengths, lengths, True, out, lse)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (6, 2), (7, 1), (16, 1), (24, 8)])
def test_packed_head_groups(A, kind, heads):
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (randn(g, 70, h, 64, kind=kind) for h in (heads[0], heads[1], heads[1]))
    out, lse = packed(A, q, k, v, [70], [70], True)
    check_packed(q, k, v, [70], [70], True, out, lse)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_lens,k_lens", [([5, 3], [0, 9]), ([70, 40], [3, 130]), ([1, 1, 1], [300, 1, 64]), ([200], [64]),
                                           ([33, 0, 2], [31, 50, 1])])
def test_packed_more_or_fewer_keys_than_queries(A, kind, causal, q_lens, k_lens):
    """Rows that see nothing among them: zeros, and -inf."""
    g = torch.Generator(device="cuda").manual_seed(4)
    q = randn(g, sum(q_lens), 2, 64, kind=kind)
    k, v = (randn(g, sum(k_lens), 1, 64, kind=kind) for _ in range(2))
    out, lse = packed(A, q, k, v, q_lens, k_lens, causal)
    check_packed(q, k, v, q_lens, k_lens, causal, out, lse)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["fused", "transposed", "padded", "broadcast"])
def test_packed_strides(A, kind, layout):
    """Slices of a fused projection, heads before tokens, rows with room behind, one key head for all by stride 0."""
    g = torch.Generator(device="cuda").manual_seed(5)
    n, h, hk, d = 150, 4, 2, 80
    if layout == "fused":
        x = randn(g, n, h + 2 * hk, d, kind=kind)
        q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
        out = torch.full((n, h + 1, d), float("nan"), dtype=TYPES[kind], device="cuda")
        out, rest = out[:, :h], out[:, h:]
    elif layout == "transposed":
        q, k, v = (randn(g, m, n, d, kind=kind).transpose(0, 1) for m in (h, hk, hk))
        out = torch.full((h, n, d), float("nan"), dtype=TYPES[kind], device="cuda").transpose(0, 1)
        rest = None
    elif layout == "padded":
        q, k, v = (randn(g, n, m, d + 16, kind=kind)[..., 8:8 + d] for m in (h, hk, hk))
        out = torch.full((n, h, d + 8), float("nan"), dtype=TYPES[kind], device="cuda")
        out, rest = out[..., :d], out[..., d:]
    else:
        q = randn(g, n, h, d, kind=kind)
        k, v = (randn(g, n, 1, d, kind=kind).expand(n, hk, d) for _ in range(2))
        out, rest = None, None
    out, lse = packed(A, q, k, v, [100, 50], [100, 50], True, out=out)
    check_packed(q, k, v, [100, 50], [100, 50], True, out, lse)
    assert rest is None or torch.isnan(rest).all()              # nothing beside the rows is written


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_packed_what_a_row_does_not_see_does_not_reach_it(A, kind, poison):
    """The other sequence, and later keys and values of the own one, hold NaN, infinities or the type's lowest value."""
    g = torch.Generator(device="cuda").manual_seed(6)
    lengths, d = [90, 75], 64
    q, k, v = (randn(g, 165, h, d, kind=kind) for h in (2, 1, 1))
    value = torch.finfo(TYPES[kind]).min if poison == "lowest" else poison
    clean = packed(A, q, k, v, lengths, lengths, True)
    for at in (slice(90, 165), slice(0, 90), slice(50, 90), slice(130, 165), slice(33, 34)):
        for which in ("k", "v"):
            k2, v2 = k.clone(), v.clone()
            (k2 if which == "k" else v2)[at] = value
            out, lse = packed(A, q, k2, v2, lengths, lengths, True)
            end = 90 if at.start < 90 else 165
            rows = [r for r in range(165) if not at.start <= r < end]        # (rows of the sequence from the first poisoned key on see it)
            assert torch.equal(out[rows], clean[0][rows]) and torch.equal(lse[:, rows], clean[1][:, rows])
            if which == "v" and poison != "lowest":                          # and those that see it show it
                seen = out[at.start:end]
                assert torch.isnan(seen).all() if math.isnan(value) else (torch.isnan(seen) | (seen == value)).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_packed_sharp_and_flat_weights(A, kind):
    """Scores of hundreds, and scores that are all the same; a scale of its own."""
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = (randn(g, 300, 1, 64, kind=kind) for _ in range(3))
    for scale in (20.0, 1e-6):
        out, lse = packed(A, q, k, v, [300], [300], True, scale=scale)
        check_packed(q, k, v, [300], [300], True, out, lse, scale=scale)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_packed_order_of_growing_scores(A, kind):
    """The running maximum rises with every key, or falls."""
    d = 64
    for sign in (1, -1):
        q = torch.ones((200, 1, d), device="cuda", dtype=TYPES[kind])
        k = (sign * torch.arange(200, device="cuda").float() / 8)[:, None, None].expand(200, 1, d).to(TYPES[kind]).contiguous()
        g = torch.Generator(device="cuda").manual_seed(8)
        v = randn(g, 200, 1, d, kind=kind)
        out, lse = packed(A, q, k, v, [200], [200], True)
        check_packed(q, k, v, [200], [200], True, out, lse)


def test_packed_long_sequence(A):
    """Some rows of 5000 keys, in every type and by both masks."""
    g = torch.Generator(device="cuda").manual_seed(9)
    for kind in TYPES:
        n = 5000
        q, k, v = (randn(g, n, 1, 128, kind=kind) for _ in range(3))
        for causal in (False, True):
            out, lse = packed(A, q, k, v, [n], [n], causal)
            rows = [0, 1, 63, 64, 1000, 2047, 2048, 4998, 4999]
            want = rows64(q[rows, 0], k[:, 0], v[:, 0], 1 / math.sqrt(128), [r + 1 if causal else n for r in rows])
            check(kind, 128, n, out[rows, 0], lse[0, rows], want, float(v.abs().max()))


def test_packed_rows_of_no_sequence_are_left_alone(A):
    g = torch.Generator(device="cuda").manual_seed(10)
    q, k, v = (randn(g, 100, 1, 64) for _ in range(3))
    out, lse = packed(A, q, k, v, [40, 30], [40, 30], True)
    assert torch.isnan(out[70:]).all() and not torch.isnan(out[:70]).any()


# ---- over a paged cache ---------------------------------------------------------------

def make_cache(g, contexts, block, hk, d, kind, order="blocks", spare=3, fill=float("nan")):
    """Keys and values of requests scattered over a cache whose other slots hold `fill`."""
    need = [-(-n // block) for n in contexts]
    total = sum(need) + spare
    shape = (total, block, hk, d) if order == "blocks" else (total, hk, block, d)
    keys, values = (torch.full(shape, fill, dtype=TYPES[kind], device="cuda") for _ in range(2))
    if order != "blocks":
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(3)).tolist()
    width = max(need + [1]) + 1
    table = torch.full((len(contexts), width), 2 ** 30, dtype=torch.int32, device="cuda")     # entries behind a request's end are rubbish
    ks, vs, at = [], [], 0
    for r, n in enumerate(contexts):
        mine = perm[at:at + need[r]]
        at += need[r]
        table[r, :need[r]] = ints(mine)
        k, v = randn(g, n, hk, d, kind=kind), randn(g, n, hk, d, kind=kind)
        for j, b in enumerate(mine):
            part = slice(j * block, min(n, (j + 1) * block))
            keys[b, :part.stop - part.start], values[b, :part.stop - part.start] = k[part], v[part]
        ks.append(k)
        vs.append(v)
    return keys, values, table, ks, vs


def paged(A, q, keys, values, table, q_lens, contexts, causal=True, max_q=None, max_context=None):
    kind = [n for n, t in TYPES.items() if t == q.dtype][0]
    geom = A.AttentionGeom(A.TYPES[kind], q.shape[1], keys.shape[2], q.shape[2], int(causal), 1 / math.sqrt(q.shape[2]))
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    lse = torch.full((q.shape[1], q.shape[0]), float("nan"), device="cuda")
    starts, lens = ints(starts_of(q_lens)), ints(contexts)
    A.attention_paged(geom, A.heads_of(q), A.PagedCache.of(keys, values), table.data_ptr(), table.shape[1], starts.data_ptr(),
                      lens.data_ptr(), len(q_lens), len(q), max(q_lens) if max_q is None else max_q,
                      max(contexts) if max_context is None else max_context, A.heads_of(out), lse=lse.data_ptr())
    torch.cuda.synchronize()
    return out, lse


def check_paged(q, ks, vs, q_lens, contexts, out, lse, causal=True):
    kind = [n for n, t in TYPES.items() if t == q.dtype][0]
    starts = starts_of(q_lens)
    group = q.shape[1] // (ks[0].shape[1])
    for r, (nq, n) in enumerate(zip(q_lens, contexts)):
        if nq == 0:
            continue
        rows = slice(starts[r], starts[r + 1])
        seen = [max(0, n - nq + i + 1) if causal else n for i in range(nq)]
        for h in range(q.shape[1]):
            want = rows64(q[rows, h], ks[r][:, h // group], vs[r][:, h // group], 1 / math.sqrt(q.shape[2]), seen)
            check(kind, q.shape[2], n, out[rows, h], lse[h, rows], want, max([float(v.abs().max()) for v in vs if v.numel()] + [0.0]))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block", [1, 7, 16, 64, 100])
@pytest.mark.parametrize("contexts", [[1], [2, 40], [63, 64, 65], [0, 130, 5], [500, 17]])
def test_paged_single_tokens(A, kind, block, contexts):
    g = torch.Generator(device="cuda").manual_seed(11)
    keys, values, table, ks, vs = make_cache(g, contexts, block, 2, 64, kind)
    q = randn(g, len(contexts), 4, 64, kind=kind)
    q_lens = [1] * len(contexts)
    out, lse = paged(A, q, keys, values, table, q_lens, contexts)
    check_paged(q, ks, vs, q_lens, contexts, out, lse)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,contexts", [([5, 1], [5, 90]), ([33], [200]), ([64, 0, 3], [64, 10, 300]), ([7, 9], [3, 9]),
                                             ([130], [131]), ([16], [700])])
@pytest.mark.parametrize("causal", [False, True])
def test_paged_chunks(A, kind, q_lens, contexts, causal):
    """Chunks beside what the cache holds; one that is longer than its context has rows that see nothing."""
    g = torch.Generator(device="cuda").manual_seed(12)
    keys, values, table, ks, vs = make_cache(g, contexts, 16, 2, 64, kind)
    q = randn(g, sum(q_lens), 6, 64, kind=kind)
    out, lse = paged(A, q, keys, values, table, q_lens, contexts, causal)
    check_paged(q, ks, vs, q_lens, contexts, out, lse, causal)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [8, 40, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("q_len", [1, 20])
def test_paged_head_sizes(A, kind, dim, q_len):
    g = torch.Generator(device="cuda").manual_seed(13)
    contexts = [150, 33]
    keys, values, table, ks, vs = make_cache(g, contexts, 16, 1, dim, kind)
    q = randn(g, 2 * q_len, 4, dim, kind=kind)
    out, lse = paged(A, q, keys, values, table, [q_len] * 2, contexts)
    check_paged(q, ks, vs, [q_len] * 2, contexts, out, lse)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(1, 1), (12, 12), (14, 2), (16, 1), (40, 1), (96, 2)])
@pytest.mark.parametrize("q_len", [1, 3])
def test_paged_head_groups(A, kind, heads, q_len):
    g = torch.Generator(device="cuda").manual_seed(14)
    keys, values, table, ks, vs = make_cache(g, [77], 16, heads[1], 64, kind)
    q = randn(g, q_len, heads[0], 64, kind=kind)
    out, lse = paged(A, q, keys, values, table, [q_len], [77])
    check_paged(q, ks, vs, [q_len], [77], out, lse)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_paged_heads_before_slots(A, kind):
    g = torch.Generator(device="cuda").manual_seed(15)
    keys, values, table, ks, vs = make_cache(g, [100, 9], 16, 4, 64, kind, order="heads")
    q = randn(g, 2, 8, 64, kind=kind)
    out, lse = paged(A, q, keys, values, table, [1, 1], [100, 9])
    check_paged(q, ks, vs, [1, 1], [100, 9], out, lse)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("contexts,q_lens", [([20000], [1]), ([9000, 50, 12000], [1, 1, 1]), ([12000], [5]), ([6000], [70])])
def test_paged_long_contexts_in_pieces(A, kind, contexts, q_lens):
    """Long contexts with few rows; the call is repeated: scratch and counters are as the first found them, and so are the bits."""
    g = torch.Generator(device="cuda").manual_seed(16)
    keys, values, table, ks, vs = make_cache(g, contexts, 16, 1, 64, kind)
    q = randn(g, sum(q_lens), 2, 64, kind=kind)
    first = paged(A, q, keys, values, table, q_lens, contexts)
    check_paged(q, ks, vs, q_lens, contexts, *first)
    again = paged(A, q, keys, values, table, q_lens, contexts)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_paged_bounds_that_are_larger_than_the_lengths(A):
    """max_q and max_context are bounds: larger ones give the same answer within the same error."""
    g = torch.Generator(device="cuda").manual_seed(17)
    contexts, q_lens = [300, 41, 7], [1, 2, 1]
    keys, values, table, ks, vs = make_cache(g, contexts, 16, 2, 64, "bf16")
    q = randn(g, 4, 4, 64, kind="bf16")
    for max_q, max_context in ((2, 300), (50, 5000), (200, 100000)):
        out, lse = paged(A, q, keys, values, table, q_lens, contexts, max_q=max_q, max_context=max_context)
        check_paged(q, ks, vs, q_lens, contexts, out, lse)


@pytest.mark.parametrize("q_len", [1, 40])
def test_paged_block_numbers_outside_the_cache_are_left_out(A, q_len):
    g = torch.Generator(device="cuda").manual_seed(18)
    keys, values, table, ks, vs = make_cache(g, [200], 16, 1, 64, "f32", fill=0.0)
    q = randn(g, q_len, 2, 64)
    for bad in (-1, len(keys), 2 ** 31 - 1, -2 ** 31):
        table[0, 3] = bad
        out, lse = paged(A, q, keys, values, table, [q_len], [200])
        for h in range(2):
            for i in range(q_len):
                seen = [j for j in range(200 - q_len + i + 1) if j // 16 != 3]
                want = rows64(q[i:i + 1, h], ks[0][seen, 0], vs[0][seen, 0], 1 / 8, [len(seen)])
                check("f32", 64, 200, out[i:i + 1, h], lse[h, i:i + 1], want, 10.0)
    table[0] = -1                                              # no key at all
    out, lse = paged(A, q, keys, values, table, [q_len], [200])
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_paged_offsets_beyond_32_bits(A):
    """A cache of more than 2^32 bytes in each of its halves: its first and last blocks."""
    g = torch.Generator(device="cuda").manual_seed(19)
    block, hk, d = 64, 8, 256
    blocks = 2 ** 32 // (block * hk * d) + 8                   # more than 2^32 elements of bf16
    keys = torch.empty((blocks, block, hk, d), dtype=torch.bfloat16, device="cuda")
    values = torch.empty_like(keys)
    where = [blocks - 1, 0, blocks - 2]
    k, v = randn(g, 180, hk, d, kind="bf16"), randn(g, 180, hk, d, kind="bf16")
    for i, b in enumerate(where):
        n = min(64, 180 - 64 * i)
        keys[b, :n], values[b, :n] = k[64 * i:64 * i + n], v[64 * i:64 * i + n]
    table = ints(where)[None].contiguous()
    for q_len in (1, 40):
        q = randn(g, q_len, hk, d, kind="bf16")
        out, lse = paged(A, q, keys, values, table, [q_len], [180])
        check_paged(q, [k], [v], [q_len], [180], out, lse)


@pytest.mark.parametrize("which", ["packed", "paged"])
def test_on_a_stream_of_its_own(A, which):
    g = torch.Generator(device="cuda").manual_seed(20)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    if which == "packed":
        q, k, v = (randn(g, 300, 2, 64, kind="bf16") for _ in range(3))
        want, _ = packed(A, q, k, v, [300], [300], True)
        geom = A.AttentionGeom(A.BF16, 2, 2, 64, 1, 1 / 8)
        st, out = ints([0, 300]), torch.empty_like(q)
        torch.cuda.synchronize()
        A.attention_packed(geom, A.heads_of(q), A.heads_of(k), A.heads_of(v), st.data_ptr(), st.data_ptr(), 1, 300, 300,
                           A.heads_of(out), stream=s.cuda_stream)
    else:
        keys, values, table, _, _ = make_cache(g, [9000], 16, 1, 64, "bf16")
        q = randn(g, 1, 4, 64, kind="bf16")
        want, _ = paged(A, q, keys, values, table, [1], [9000])
        geom = A.AttentionGeom(A.BF16, 4, 1, 64, 1, 1 / 8)
        st, lens, out = ints([0, 1]), ints([9000]), torch.empty_like(q)
        torch.cuda.synchronize()
        A.attention_paged(geom, A.heads_of(q), A.PagedCache.of(keys, values), table.data_ptr(), table.shape[1], st.data_ptr(),
                          lens.data_ptr(), 1, 1, 1, 9000, A.heads_of(out), stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, want)


def test_captured_calls_replay(A):
    """Both attentions in one graph, replayed on new values with eager work between."""
    g = torch.Generator(device="cuda").manual_seed(21)
    contexts = [5000, 70]
    keys, values, table, _, _ = make_cache(g, contexts, 16, 2, 64, "bf16", fill=0.0)
    q = randn(g, 2, 4, 64, kind="bf16")
    pq, pk, pv = (randn(g, 90, 2, 64, kind="bf16") for _ in range(3))
    starts, lens, one = ints([0, 90]), ints(contexts), ints([0, 1, 2])
    out, pout = torch.empty_like(q), torch.empty_like(pq)
    geom = A.AttentionGeom(A.BF16, 4, 2, 64, 1, 1 / 8)
    pgeom = A.AttentionGeom(A.BF16, 2, 2, 64, 1, 1 / 8)

    def calls(stream):
        A.attention_packed(pgeom, A.heads_of(pq), A.heads_of(pk), A.heads_of(pv), starts.data_ptr(), starts.data_ptr(), 1, 90, 90,
                           A.heads_of(pout), stream=stream)
        A.attention_paged(geom, A.heads_of(q), A.PagedCache.of(keys, values), table.data_ptr(), table.shape[1], one.data_ptr(),
                          lens.data_ptr(), 2, 2, 1, 5000, A.heads_of(out), stream=stream)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        calls(s.cuda_stream)                      # scratch of this stream is there before the capture
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            calls(s.cuda_stream)
    for i in range(4):
        q.copy_(randn(g, 2, 4, 64, kind="bf16"))
        pq.copy_(randn(g, 90, 2, 64, kind="bf16"))
        keys.mul_(-1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), pout.clone()
        calls(0)
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], pout)


# ---- refusals ---------------------------------------------------------------------------

def test_refusals(A):
    from minicaffe import MiniCaffeError
    x = torch.zeros((32, 2, 64), device="cuda")
    st = ints([0, 32])

    def call(geom=(0, 2, 2, 64, 1, 0.125), q=None, k=None, out=None, starts=st.data_ptr(), num=1, total=32):
        h = A.heads_of(x)
        A.attention_packed(A.AttentionGeom(*geom), q or h, k or h, h, starts, starts, num, total, total, out or h)

    for geom, word in (((3, 2, 2, 64, 1, 0.125), "type"), ((0, 3, 2, 64, 1, 0.125), "share"), ((0, 0, 0, 64, 1, 0.125), "share"),
                       ((0, 2, 2, 60, 1, 0.125), "head_dim"), ((0, 2, 2, 264, 1, 0.125), "head_dim"),
                       ((0, 2, 2, 0, 1, 0.125), "head_dim"), ((0, 2, 2, 64, 1, 0.0), "scale"),
                       ((0, 2, 2, 64, 1, float("nan")), "scale"), ((0, 2, 2, 64, 1, float("inf")), "scale")):
        with pytest.raises(MiniCaffeError, match=word):
            call(geom=geom)
    with pytest.raises(MiniCaffeError, match="q is null"):
        call(q=A.Heads(0, 128, 64))
    with pytest.raises(MiniCaffeError, match="k: .*16 bytes"):
        call(k=A.Heads(x.data_ptr() + 4, 128, 64))
    with pytest.raises(MiniCaffeError, match="out: .*16 bytes"):
        call(out=A.Heads(x.data_ptr(), 127, 64))
    with pytest.raises(MiniCaffeError, match="null"):
        call(starts=None)
    with pytest.raises(MiniCaffeError, match="extents"):
        call(num=-1)
    call(num=0)
    call(total=0)                                              # nothing to do
    with pytest.raises(ValueError):
        A.heads_of(x.transpose(1, 2))
    with pytest.raises(ValueError):
        A.heads_of(x[0])


def test_refusals_paged(A):
    from minicaffe import MiniCaffeError
    c = torch.zeros((4, 16, 2, 64), device="cuda")
    q = torch.zeros((1, 2, 64), device="cuda")
    st, lens, table = ints([0, 1]), ints([5]), ints([[0, 1]][0])

    def call(cache=None, width=2, tab=table.data_ptr(), max_q=1, max_context=5):
        h = A.heads_of(q)
        A.attention_paged(A.AttentionGeom(0, 2, 2, 64, 1, 0.125), h, cache or A.PagedCache.of(c, c), tab, width, st.data_ptr(),
                          lens.data_ptr(), 1, 1, max_q, max_context, h)

    good = (c.data_ptr(), c.data_ptr(), 4, 16) + c.stride()[:3]
    for at, value, word in ((0, 0, "null"), (1, 0, "null"), (2, 0, "blocks"), (3, 0, "blocks"), (2, 2 ** 30, "slots"),
                            (4, 2047, "16 bytes"), (6, 63, "16 bytes"), (0, c.data_ptr() + 8, "16 bytes")):
        bad = list(good)
        bad[at] = value
        with pytest.raises(MiniCaffeError, match=word):
            call(cache=A.PagedCache(*bad))
    for kw in (dict(width=0), dict(max_q=-1), dict(max_context=-1)):
        with pytest.raises(MiniCaffeError, match="extents"):
            call(**kw)
    with pytest.raises(MiniCaffeError, match="null"):
        call(tab=None)
    call(max_q=0)
    with pytest.raises(ValueError):
        A.PagedCache.of(c, c[:2])


# ---- many sequences, and values at the ends of the range ---------------------------------

@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("count", [64, 65, 200, 4200])
def test_packed_many_sequences(A, kind, count):
    """Finding a row tile's sequence among more than a wavefront's lanes; empty sequences among them."""
    g = torch.Generator(device="cuda").manual_seed(22)
    lengths = [(7 * i) % 4 if count > 1000 else (13 * i) % 37 for i in range(count)]
    n = sum(lengths)
    q, k, v = (randn(g, n, h, 64, kind=kind) for h in (2, 1, 1))
    out, lse = packed(A, q, k, v, lengths, lengths, True)
    check_packed(q, k, v, lengths, lengths, True, out, lse)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("count,longest", [(70, 3), (130, 40)])
def test_paged_many_requests(A, kind, count, longest):
    """Chunks of many requests, some empty, over contexts long enough to be cut into pieces."""
    g = torch.Generator(device="cuda").manual_seed(23)
    q_lens = [(11 * i) % (longest + 1) for i in range(count)]
    contexts = [n + (29 * i) % 60 + (900 if i == 3 else 0) for i, n in enumerate(q_lens)]
    keys, values, table, ks, vs = make_cache(g, contexts, 16, 1, 64, kind)
    q = randn(g, sum(q_lens), 2, 64, kind=kind)
    out, lse = paged(A, q, keys, values, table, q_lens, contexts)
    check_paged(q, ks, vs, q_lens, contexts, out, lse)


@pytest.mark.parametrize("dim", [64, 128, 200])
@pytest.mark.parametrize("sizes", [(1e18, 1e-18, 1.0), (1e-18, 1e18, 1.0), (1.0, 1.0, 1e37), (1.0, 1.0, 1e-30), (1e-20, 1e-10, 1.0)])
def test_packed_fp32_over_its_range(A, dim, sizes):
    """Values far from one, whose terms in fewer bits have to reach as far as fp32 does."""
    g = torch.Generator(device="cuda").manual_seed(24)
    q, k, v = (randn(g, 150, 1, dim) * s for s in sizes)
    out, lse = packed(A, q, k, v, [150], [150], True)
    check_packed(q, k, v, [150], [150], True, out, lse)


def test_packed_fp32_largest_values(A):
    """Finite values that round to infinity in bf16 stay finite."""
    g = torch.Generator(device="cuda").manual_seed(25)
    q, k, v = (randn(g, 100, 1, 64) for _ in range(3))
    v[::2] = torch.finfo(torch.float32).max
    v[1::2] = -torch.finfo(torch.float32).max
    v /= 4
    v[5] = torch.finfo(torch.float32).max
    q[:, :, 0], k[:, :, 0] = 3.4e38, 0.0
    out, lse = packed(A, q, k, v, [100], [100], True)
    # the sum of weights times values stays within 1.25 / 4 of the largest but in row 5 and those that weigh it
    assert torch.isfinite(lse).all()
    rows = [r for r in range(5)]
    check_packed(q[rows], k[rows], v[rows], [5], [5], True, out[rows], lse[:, rows])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("where", ["packed", "single", "chunk"])
def test_infinite_keys(A, kind, where):
    """A key of infinity gives scores of plus and minus infinity: rows with the first are NaN, the others ignore it."""
    g = torch.Generator(device="cuda").manual_seed(26)
    n, d, at = 60, 64, 20
    q_len = {"packed": n, "single": 1, "chunk": 40}[where]
    q, k, v = randn(g, q_len, 1, d, kind=kind), randn(g, n, 1, d, kind=kind), randn(g, n, 1, d, kind=kind)
    k[at] = 0
    k[at, 0, 7] = float("inf")
    if where == "packed":
        out, _ = packed(A, q, k, v, [n], [n], True)
    else:
        keys, values = (torch.zeros((4, 16, 1, d), dtype=TYPES[kind], device="cuda") for _ in range(2))
        keys.view(-1, 1, d)[:n], values.view(-1, 1, d)[:n] = k, v
        out, _ = paged(A, q, keys, values, ints([0, 1, 2, 3])[None].contiguous(), [q_len], [n])
    for r in range(q_len):
        sees = n - q_len + r + 1
        if sees > at and q[r, 0, 7] > 0:
            assert torch.isnan(out[r]).all()
        else:
            kept = [j for j in range(sees) if j != at]
            want = rows64(q[r:r + 1, 0], k[kept, 0], v[kept, 0], 1 / 8, [len(kept)])
            lse = torch.log(torch.exp(torch.zeros(1))) + want[1]
            check(kind, d, n, out[r:r + 1, 0], lse, want, 5.0)


# ---- strides that a tile's 32-bit offsets could not hold ------------------------------------

@pytest.mark.parametrize("kind,size", [("f32", 4), ("bf16", 2)])
@pytest.mark.parametrize("which", ["k", "v", "cache"])
def test_refused_key_strides(A, kind, size, which):
    from minicaffe import MiniCaffeError
    code = {"f32": 0, "bf16": 2}[kind]
    dtype = torch.float32 if kind == "f32" else torch.bfloat16
    x = torch.zeros((16, 2, 64), device="cuda", dtype=dtype)
    c = torch.zeros((1, 16, 2, 64), device="cuda", dtype=dtype)
    st, lens, table = ints([0, 16]), ints([16]), ints([0])
    h = A.heads_of(x)
    geom = A.AttentionGeom(code, 2, 2, 64, 1, 0.125)
    for stride in (-128, 2 ** 25 // size + 16 // size, 2 ** 62):
        with pytest.raises(MiniCaffeError, match="token_stride"):
            if which == "cache":
                bad = A.PagedCache(c.data_ptr(), c.data_ptr(), 1, 16, c.stride(0), stride, c.stride(2))
                A.attention_paged(geom, h, bad, table.data_ptr(), 1, st.data_ptr(), lens.data_ptr(), 1, 16, 16, 16, h)
            else:
                bad = A.Heads(x.data_ptr(), stride, 64)
                A.attention_packed(geom, h, bad if which == "k" else h, bad if which == "v" else h, st.data_ptr(), st.data_ptr(),
                                   1, 16, 16, h)


# ---- enough workgroups for three to a CU, and rows of 192 values ------------------------------

def check_heads(q, k, v, lengths, causal, out, lse, heads):
    """As check_packed, as many key heads as query heads, `heads` of them."""
    check_packed(q[:, heads], k[:, heads], v[:, heads], lengths, lengths, causal, out[:, heads], lse[heads])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_many_workgroups(A, kind, dim, causal):
    """Short sequences with many key heads: 2048 workgroups and more; an empty sequence, one token, and ragged ends."""
    g = torch.Generator(device="cuda").manual_seed(31)
    lengths = [(11 * i) % 43 for i in range(66)] + [131, 65, 64, 33, 1]
    n = sum(lengths)
    q, k, v = (randn(g, n, 32, dim, kind=kind) for _ in range(3))
    out, lse = packed(A, q, k, v, lengths, lengths, causal)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    check_heads(q, k, v, lengths, causal, out, lse, [0, 13, 31])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_packed_workgroups_at_once(A, kind, dim):
    """Between 512 and 768 workgroups of equal length, not causal; an infinity and a NaN in two sequences' values."""
    g = torch.Generator(device="cuda").manual_seed(32)
    lengths = [200] * 12
    q, k, v = (randn(g, 2400, 20, dim, kind=kind) for _ in range(3))
    clean, clean_lse = packed(A, q, k, v, lengths, lengths, False)
    check_heads(q, k, v, lengths, False, clean, clean_lse, [0, 3, 19])
    poisoned = v.clone()
    poisoned[250, 3, 5] = float("inf")
    poisoned[1999, 0, 0] = float("nan")
    out, lse = packed(A, q, k, poisoned, lengths, lengths, False)
    assert torch.isposinf(out[200:400, 3, 5]).all() and torch.isnan(out[1800:2000, 0, 0]).all()
    out[200:400, 3, 5] = clean[200:400, 3, 5]
    out[1800:2000, 0, 0] = clean[1800:2000, 0, 0]
    check_heads(q, k, v, lengths, False, out, lse, [0, 3, 19])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [136, 192])
@pytest.mark.parametrize("lengths", [[1], [33, 0, 128, 257], [700]])
def test_packed_192(A, kind, dim, lengths):
    g = torch.Generator(device="cuda").manual_seed(33)
    n = sum(lengths)
    q, k, v = (randn(g, n, h, dim, kind=kind) for h in (4, 2, 2))
    out, lse = packed(A, q, k, v, lengths, lengths, True)
    check_packed(q, k, v, lengths, lengths, True, out, lse)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [136, 192, 200, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_wide_rows_and_many(A, kind, dim, causal):
    """Rows of more than 128 values and enough of them for eight wavefronts: 512 queries a sequence, 512 workgroups of 128;
    an infinity in one sequence's values."""
    g = torch.Generator(device="cuda").manual_seed(34)
    lengths = [530, 700, 0, 812, 601]
    n = sum(lengths)
    q, k, v = (randn(g, n, 24, dim, kind=kind) for _ in range(3))
    out, lse = packed(A, q, k, v, lengths, lengths, causal)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    check_heads(q, k, v, lengths, causal, out, lse, [0, 23])
    poisoned = v.clone()
    poisoned[530, 7, dim - 1] = float("inf")             # the second sequence's first key: all of its rows see it
    again, _ = packed(A, q, k, poisoned, lengths, lengths, causal)
    rows = slice(530, 530 + 700)
    assert torch.isposinf(again[rows, 7, dim - 1]).all()
    again[rows, 7, dim - 1] = out[rows, 7, dim - 1]
    check_heads(q, k, v, lengths, causal, again, lse, [7])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [192, 256])
@pytest.mark.parametrize("block", [16, 24, 7])
def test_paged_wide_chunks(A, kind, dim, block):
    """Chunks over a paged cache, rows of more than 128 values: four wavefronts, and eight where there are 1024 rows."""
    g = torch.Generator(device="cuda").manual_seed(35)
    for q_lens, contexts in (([40, 0, 3, 129], [300, 50, 3, 700]), ([300], [1500])):
        keys, values, table, ks, vs = make_cache(g, contexts, block, 1, dim, kind)
        q = randn(g, sum(q_lens), 4, dim, kind=kind)
        out, lse = paged(A, q, keys, values, table, q_lens, contexts)
        check_paged(q, ks, vs, q_lens, contexts, out, lse)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("block", [16, 5])
def test_paged_many_chunks(A, kind, dim, block):
    """Chunks of many requests, 1280 workgroups and more; a block that does not exist in one of them."""
    g = torch.Generator(device="cuda").manual_seed(36)
    q_lens = [(13 * i) % 47 for i in range(47)]
    contexts = [n + (29 * i) % 90 for i, n in enumerate(q_lens)]
    keys, values, table, ks, vs = make_cache(g, contexts, block, 28, dim, kind, fill=0.0)
    q = randn(g, sum(q_lens), 28, dim, kind=kind)
    out, lse = paged(A, q, keys, values, table, q_lens, contexts)
    some = [0, 27]
    check_paged(q[:, some], [k[:, some] for k in ks], [v[:, some] for v in vs], q_lens, contexts, out[:, some], lse[some])
    at = 40                                              # its first block: those keys are left out
    assert contexts[at] > 2 * block and q_lens[at] > 0
    table[at, 0] = -1
    again, again_lse = paged(A, q, keys, values, table, q_lens, contexts)
    starts = starts_of(q_lens)
    mine = slice(starts[at], starts[at + 1])
    rest = [n - block for n in contexts[at:at + 1]]
    check_paged(q[mine][:, some], [ks[at][block:, some]], [vs[at][block:, some]], [q_lens[at]], rest, again[mine][:, some],
                again_lse[some, mine])
    keep = torch.ones(len(q), dtype=torch.bool, device="cuda")
    keep[mine] = False
    assert torch.equal(again[keep], out[keep]) and torch.equal(again_lse[:, keep], lse[:, keep])


@pytest.mark.parametrize("kind,dim", [("f32", 64), ("bf16", 128), ("f16", 80), ("bf16", 256)])
@pytest.mark.parametrize("requests,longest", [(1, 384), (1, 640), (5, 3000), (40, 700)])
def test_paged_single_tokens_in_more_or_fewer_pieces(A, kind, dim, requests, longest):
    """One piece, two, as many as there are steps; lengths far below the longest among them."""
    g = torch.Generator(device="cuda").manual_seed(37)
    contexts = [longest] + [1 + (97 * i) % longest for i in range(1, requests)]
    keys, values, table, ks, vs = make_cache(g, contexts, 16, 2, dim, kind)
    q = randn(g, requests, 6, dim, kind=kind)
    first = paged(A, q, keys, values, table, [1] * requests, contexts)
    check_paged(q, ks, vs, [1] * requests, contexts, *first)
    again = paged(A, q, keys, values, table, [1] * requests, contexts)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
