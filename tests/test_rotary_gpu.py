"""mcRotary against turns of complex numbers in 64 bits."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from attention_ref import TYPES, UNIT  # noqa: E402


@pytest.fixture(scope="module")
def A(gpu_mode):
    from minicaffe import attention
    return attention


def axis_of(sections, cycled):
    left, order = list(sections), []
    while sum(left):
        for a in range(len(left)):
            take = min(left[a], 1) if cycled else left[a]
            order += [a] * take
            left[a] -= take
    return torch.tensor(order)


def turned64(x, positions, frequencies, sections, cycled, adjacent):
    """What the definition says: the angle is the product in 32 bits."""
    pairs = sum(sections)
    angle = (positions.cpu()[axis_of(sections, cycled)].t().float() * frequencies.cpu()).double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    x = x.double().cpu()
    y = x.clone()
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if adjacent else (slice(0, pairs), slice(pairs, 2 * pairs))
    z = torch.complex(x[..., a], x[..., b]) * turn
    y[..., a], y[..., b] = z.real, z.imag
    size = x.abs().clone()                              # |a| + |b| of the pair
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def check(kind, got, want):
    y, size = want
    # cosine, sine (an ulp or two each), two products and a sum in 32 bits, one rounding to the type
    bound = UNIT[kind] * y.abs() + 6 * 2.0 ** -24 * size + (2.0 ** -25 if kind == "f16" else 0.0)
    off = (got.double().cpu() - y).abs()
    assert (off <= bound).all(), (off - bound).max()


def inputs(kind, tokens, heads, kv, dim, axes, seed=1, far=3000):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((tokens, heads + 2 * kv, dim), generator=g, device="cuda").to(TYPES[kind])
    pos = torch.randint(0, far, (axes, tokens), generator=g, device="cuda", dtype=torch.int32)
    return x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], pos


def frequencies(pairs):
    return (1e4 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().cuda()


CASES = [
    # heads, kv, dim, sections, cycled, adjacent
    (4, 2, 64, [32], False, False), (4, 2, 64, [32], False, True), (3, 1, 128, [16, 24, 24], False, False),
    (3, 1, 128, [16, 24, 24], True, False), (2, 2, 80, [10, 30], False, True), (2, 2, 80, [20], False, False),
    (5, 5, 96, [8, 8, 8], True, True), (1, 1, 256, [32, 32, 32, 32], False, False), (7, 1, 8, [1], False, False),
    (7, 1, 8, [1, 0], True, True), (2, 1, 40, [9], False, False), (2, 1, 40, [4, 3, 3], True, False), (2, 1, 24, [0, 6], False, True),
    (32, 8, 128, [64], False, False),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("tokens", [1, 13])
def test_against_64_bits(A, kind, case, tokens):
    heads, kv, dim, sections, cycled, adjacent = case
    q, k, v, pos = inputs(kind, tokens, heads, kv, dim, len(sections))
    f = frequencies(sum(sections))
    block = 5
    keys, values = (torch.full((6, block, kv, dim), 7.0, dtype=TYPES[kind], device="cuda") for _ in range(2))
    slots = torch.randperm(30, generator=torch.Generator().manual_seed(2))[:tokens].int().cuda()
    q_out, k_out = torch.empty_like(q).contiguous(), torch.empty_like(k).contiguous()
    geom = A.rotary_geom(A.TYPES[kind], heads, kv, dim, 2 * sum(sections), sections, adjacent=adjacent, cycled=cycled)
    A.rotary(geom, f.data_ptr(), pos.data_ptr(), pos.stride(0), tokens, A.heads_of(q), A.heads_of(q_out), k=A.heads_of(k),
             k_out=A.heads_of(k_out), v=A.heads_of(v), cache=A.PagedCache.of(keys, values), slots=slots.data_ptr())
    torch.cuda.synchronize()
    check(kind, q_out, turned64(q, pos, f, sections, cycled, adjacent))
    check(kind, k_out, turned64(k, pos, f, sections, cycled, adjacent))
    at = slots.long()
    flat_k, flat_v = keys.view(30, kv, dim), values.view(30, kv, dim)
    assert torch.equal(flat_k[at], k_out) and torch.equal(flat_v[at], v)
    rest = torch.ones(30, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert (flat_k[rest] == 7).all() and (flat_v[rest] == 7).all()
    # the values behind rotary_dim are copied bit by bit
    assert torch.equal(q_out[..., 2 * sum(sections):], q[..., 2 * sum(sections):])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_in_place_and_queries_alone(A, kind):
    q, k, v, pos = inputs(kind, 9, 3, 2, 64, 2)
    f, sections = frequencies(32), [12, 20]
    want_q, want_k = turned64(q, pos, f, sections, False, False), turned64(k, pos, f, sections, False, False)
    q1, k1 = q.clone(), k.clone()
    A.rotary(A.rotary_geom(A.TYPES[kind], 3, 0, 64, 64, sections), f.data_ptr(), pos.data_ptr(), pos.stride(0), 9, A.heads_of(q1),
             A.heads_of(q1))
    q2 = q.clone()
    A.rotary(A.rotary_geom(A.TYPES[kind], 3, 2, 64, 64, sections), f.data_ptr(), pos.data_ptr(), pos.stride(0), 9, A.heads_of(q2),
             A.heads_of(q2), k=A.heads_of(k1), k_out=A.heads_of(k1))
    torch.cuda.synchronize()
    check(kind, q1, want_q)
    check(kind, k1, want_k)
    assert torch.equal(q1, q2)


def test_far_positions(A):
    """The cosine of an angle of a million is as exact as that of a small one."""
    q, _, _, pos = inputs("f32", 500, 1, 0, 64, 1, far=2 ** 20)
    f = frequencies(32)
    out = torch.empty_like(q)
    pos[0, :4] = torch.tensor([0, -1, -2 ** 20, 2 ** 31 - 1], dtype=torch.int32)
    A.rotary(A.rotary_geom(A.F32, 1, 0, 64, 64, [32]), f.data_ptr(), pos.data_ptr(), pos.stride(0), 500, A.heads_of(q), A.heads_of(out))
    torch.cuda.synchronize()
    check("f32", out, turned64(q, pos, f, [32], False, False))


def test_slots_outside_the_cache_are_not_stored(A):
    q, k, v, pos = inputs("bf16", 6, 1, 2, 64, 1)
    f = frequencies(32)
    keys, values = (torch.full((3, 4, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.tensor([-1, 12, 2 ** 31 - 1, -2 ** 31, 11, 0], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    A.rotary(A.rotary_geom(A.BF16, 1, 2, 64, 64, [32]), f.data_ptr(), pos.data_ptr(), pos.stride(0), 6, A.heads_of(q), A.heads_of(out),
             k=A.heads_of(k), v=A.heads_of(v), cache=A.PagedCache.of(keys, values), slots=slots.data_ptr())
    torch.cuda.synchronize()
    flat = values.view(12, 2, 64)
    assert torch.equal(flat[11], v[4]) and torch.equal(flat[0], v[5]) and (flat[1:11] == 7).all()
    assert (keys.view(12, 2, 64)[1:11] == 7).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_many_tokens_and_heads_before_slots(A, kind):
    tokens, kv, dim = 1037, 3, 64
    q, k, v, pos = inputs(kind, tokens, 6, kv, dim, 3)
    f, sections = frequencies(32), [8, 12, 12]
    keys, values = (torch.zeros((70, kv, 16, dim), dtype=TYPES[kind], device="cuda").transpose(1, 2) for _ in range(2))
    slots = torch.randperm(70 * 16, generator=torch.Generator().manual_seed(2))[:tokens].int().cuda()
    out = torch.empty_like(q).contiguous()
    A.rotary(A.rotary_geom(A.TYPES[kind], 6, kv, dim, dim, sections, cycled=True), f.data_ptr(), pos.data_ptr(), pos.stride(0), tokens,
             A.heads_of(q), A.heads_of(out), k=A.heads_of(k), v=A.heads_of(v), cache=A.PagedCache.of(keys, values),
             slots=slots.data_ptr())
    torch.cuda.synchronize()
    check(kind, out, turned64(q, pos, f, sections, True, False))
    at = slots.long()
    check(kind, keys[at // 16, at % 16], turned64(k, pos, f, sections, True, False))
    assert torch.equal(values[at // 16, at % 16], v)


def test_refusals(A):
    from minicaffe import MiniCaffeError
    x, f = torch.zeros((4, 2, 64), device="cuda"), torch.zeros(32, device="cuda")
    pos = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    cache = A.PagedCache.of(torch.zeros((1, 4, 2, 64), device="cuda"), torch.zeros((1, 4, 2, 64), device="cuda"))

    def call(type=0, heads=2, kv=2, dim=64, rot=64, sections=(16, 16), tokens=4, freq=f.data_ptr(), q=None, **kw):
        h = A.heads_of(x)
        A.rotary(A.rotary_geom(type, heads, kv, dim, rot, list(sections)), freq, pos.data_ptr(), 4, tokens, q or h, h, **kw)

    h = A.heads_of(x)
    for kw, word in ((dict(type=5), "type"), (dict(heads=0), "heads"), (dict(dim=60), "head_dim"), (dict(rot=63), "rotary_dim"),
                     (dict(rot=66), "rotary_dim"), (dict(rot=0), "rotary_dim"), (dict(sections=(16, 15)), "sections"),
                     (dict(sections=(33, -1)), "section"), (dict(tokens=-1), "tokens"), (dict(freq=None), "null"),
                     (dict(q=A.Heads(x.data_ptr() + 4, 128, 64)), "16 bytes"), (dict(k=h), "neither"), (dict(k_out=h), "without k"),
                     (dict(v=h), "without a cache"), (dict(kv=0, k=h, k_out=h), "heads_kv"), (dict(k=h, cache=cache), "slots")):
        with pytest.raises(MiniCaffeError, match=word):
            call(**kw)
    call(tokens=0)
    with pytest.raises(ValueError):
        call(sections=())


def test_refused_axis_stride(A):
    from minicaffe import MiniCaffeError
    x, f = torch.zeros((4, 2, 64), device="cuda"), torch.zeros(32, device="cuda")
    pos = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    h = A.heads_of(x)
    with pytest.raises(MiniCaffeError, match="axis_stride"):
        A.rotary(A.rotary_geom(0, 2, 0, 64, 64, [16, 16]), f.data_ptr(), pos.data_ptr(), -4, 4, h, h)
