"""Sampling and shared-prefix attention kernels against plain forms in 64 bits, over the sizes, masks, layouts and ways of
calling where they can go wrong."""
import math

import pytest
import torch

from faster_yoco_b200 import ops
from faster_yoco_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(autouse=True)
def _native():
    ops.set_backend("native")
    yield
    assert int(ops._C().status()[0].item()) == 0


def cuda(*s, seed=0, dtype=torch.float32):
    return torch.randn(*s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


# ----------------------------------------------------------------------------------------------------------------------
# sampling


def rows_of(v, N, dtype):
    return torch.as_tensor(v, device="cuda").to(dtype).expand(N).contiguous()


def check_sample(x, u, t=1.0, k=0, p=1.0, mp=0.0):
    """Tokens equal to the 64-bit plain form's; log-probabilities within the rounding of two fp32 results (half a step
    each) and of the fixed-point sums (half of 2^-44 for each of at most 2^17 weights, against a sum of 1 or more)."""
    N = x.shape[0]
    tok, lp = ops.sample(x, u, t, k, p, mp, return_logprob=True)
    want, wlp = ref.sample(x, u, rows_of(t, N, torch.float32), rows_of(k, N, torch.int64),
                           rows_of(p, N, torch.float32), rows_of(mp, N, torch.float32))
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32
    assert torch.equal(tok, want)
    fine = torch.isfinite(wlp)
    assert torch.equal(lp[~fine], wlp[~fine])
    tol = 2.0 ** -23 * wlp[fine].abs() + 2.0 ** -28
    assert bool(((lp[fine].double() - wlp[fine].double()).abs() <= tol).all())
    assert torch.equal(ops.sample(x, u, t, k, p, mp), tok)
    return tok


def logits_like(N, V, dtype, seed, peaked=True):
    x = (2.0 if peaked else 0.5) * cuda(N, V, seed=seed)
    if peaked:
        m = min(40, V)
        at = cuda(N, V, seed=seed + 100).topk(m, dim=1).indices
        x.scatter_add_(1, at, 14.0 - 0.3 * torch.arange(m, device="cuda").float() + cuda(N, m, seed=seed + 200))
    return x.to(dtype)


SETTINGS = {"plain": dict(), "hot": dict(t=1.7), "cold": dict(t=0.05), "greedy": dict(t=0.0), "top_k": dict(t=0.8, k=50),
            "top_1": dict(k=1), "top_p": dict(t=0.8, p=0.95), "small_p": dict(p=0.01), "no_p": dict(p=0.0),
            "min_p": dict(mp=0.05), "all": dict(t=0.9, k=40, p=0.9, mp=0.02), "wide_k": dict(k=3000, p=0.99),
            "most": dict(t=1.2, p=0.9999)}


@pytest.mark.parametrize("mode", SETTINGS)
@pytest.mark.parametrize("V,dtype", [(1, torch.float32), (2, torch.bfloat16), (31, torch.float16), (33, torch.float32),
                                     (1024, torch.bfloat16), (5001, torch.float32), (8192, torch.float16),
                                     (50001, torch.bfloat16), (100288, torch.bfloat16), (131071, torch.float32)])
@pytest.mark.parametrize("peaked", [True, False])
def test_sample(mode, V, dtype, peaked):
    N = 3 if V > 10000 else 9
    x = logits_like(N, V, dtype, seed=V % 97, peaked=peaked)
    u = torch.rand(N, generator=torch.Generator(device="cuda").manual_seed(V), device="cuda")
    check_sample(x, u, **SETTINGS[mode])


@pytest.mark.parametrize("N", [1, 2, 5, 17, 40, 75, 147, 149, 300, 700])
def test_sample_batches(N):
    """Every way of dividing rows over the machine gives the same tokens."""
    x = logits_like(N, 20011, torch.bfloat16, seed=N)
    u = torch.rand(N, generator=torch.Generator(device="cuda").manual_seed(N), device="cuda")
    for kw in (dict(t=0.8, p=0.95), dict(k=50, p=0.9), dict(mp=0.01), dict(t=1.5)):
        tok = check_sample(x, u, **kw)
        assert torch.equal(tok[:1], ops.sample(x[:1], u[:1], kw.get("t", 1.0), kw.get("k", 0), kw.get("p", 1.0),
                                               kw.get("mp", 0.0)))


@pytest.mark.parametrize("V", [7, 1000, 40000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sample_edges(V, dtype):
    x = torch.zeros(12, V, device="cuda", dtype=dtype)
    x[0] = -INF
    x[1] = float("nan")
    x[2, V - 1] = INF                          # one certain token
    x[3, 1::2] = INF                           # several: equal shares
    x[4] = -INF
    x[4, V // 2] = -80.0                       # a single candidate
    x[5, ::2] = -0.0                           # equal to +0
    x[6] = torch.finfo(dtype).min              # the type's lowest value everywhere: a flat distribution
    x[7, 1:] = torch.finfo(dtype).min
    x[8, ::3] = float("nan")
    x[9, : V - 2] = -INF
    x[10] = torch.linspace(-60, 30, V, device="cuda").to(dtype)
    x[11] = torch.linspace(3e38, -3e38, V, device="cuda").to(dtype)
    for u0 in (0.0, 0.3, 1.0 - 2.0 ** -24):
        u = torch.full((12,), u0, device="cuda")
        for kw in (dict(), dict(k=3), dict(p=0.6), dict(mp=0.5), dict(t=0.0), dict(k=V - 1, p=0.7), dict(t=1e-30),
                   dict(t=INF), dict(k=V + 5), dict(mp=1.0), dict(k=2, p=0.3, mp=0.9)):
            tok = check_sample(x, u, **kw)
            assert tok[:2].tolist() == [-1, -1] and int(tok[2]) == V - 1 and int(tok[4]) == V // 2


@pytest.mark.parametrize("N,V", [(24, 40), (12, 700), (1, 50001), (200, 9001)])
def test_sample_neighbours_at_low_temperatures(N, V):
    """Logits a few steps of fp32 below the largest, at temperatures where such a step is anything from nothing to
    thousands in the exponent: every weight is the definition's, or zero."""
    g = torch.Generator(device="cuda").manual_seed(V)
    r = torch.arange(N, device="cuda")
    top = 120 * torch.rand(N, 1, generator=g, device="cuda") - 60
    x = top - 0.5 - 5 * torch.rand(N, V, generator=g, device="cuda")
    at = torch.rand(N, V, generator=g, device="cuda").topk(20, dim=1).indices
    steps = torch.randint(1, 65, (N, 20), generator=g, device="cuda", dtype=torch.int32)
    steps[:, 0] = 0
    # one step down: the next smaller integer image of a positive float, the next larger one of a negative
    x.scatter_(1, at, (top.view(torch.int32) - steps * top.sign().int()).view(torch.float32))
    t = torch.tensor([1e-6, 1e-7, 3e-8, 1e-8, 5e-9, 1e-9, 1e-10, 1e-12, 1e-30, 1e-40], device="cuda")[r % 10]
    for u0 in (0.0, 0.4, 0.8, 1.0 - 2.0 ** -24):
        u = torch.full((N,), u0, device="cuda")
        for kw in (dict(), dict(k=10), dict(p=0.7), dict(mp=0.3), dict(k=600, p=0.9)):
            check_sample(x, u, t, **kw)


def check_sample_on_borders(x, u, t=1.0, k=0, p=1.0, mp=0.0):
    """check_sample for rows where u may fall ON a border between two tokens (a pattern that repeats, halved by u = 0.5:
    the first half of 900 logits of weights 1, w, w, 1, w, w, ... is exactly half of them, so the rounding of the sums says
    which side of it a token lies). Sums of at most 2^17 weights, each within 2^-48, in 64 bits are within 2^17 2^-53 +
    2^-48 < 2^-34 of their value: the token is the definition's at u (1 - 2^-34) or at u (1 + 2^-34)."""
    N = x.shape[0]
    tok, lp = ops.sample(x, u, t, k, p, mp, return_logprob=True)
    pars = (rows_of(t, N, torch.float32), rows_of(k, N, torch.int64), rows_of(p, N, torch.float32),
            rows_of(mp, N, torch.float32))
    good = torch.zeros(N, dtype=torch.bool, device="cuda")
    for side in (1 - 2.0 ** -34, 1 + 2.0 ** -34):
        want, wlp = ref.sample(x, u.double() * side, *pars)
        tol = 2.0 ** -23 * wlp.abs() + 2.0 ** -28
        good |= (tok == want) & ((lp.double() - wlp.double()).abs() <= tol)
    assert bool(good.all())


@pytest.mark.parametrize("V", [8, 900, 40000])
def test_sample_largest_far_below_zero(V):
    low = torch.finfo(torch.float32).min
    x = torch.full((6, V), low, device="cuda")
    x[0, V // 2] = -1e38
    x[1, ::3] = -2e38
    x[2, 1::2] = -3e38
    x[3] = torch.linspace(-1e37, -3.4e38, V, device="cuda")
    x[4] = -10 - torch.arange(V, device="cuda") / V
    x[5, 2:5] = 3e38
    for u0 in (0.0, 0.5, 1.0 - 2.0 ** -24):
        u = torch.full((6,), u0, device="cuda")
        for t in (1.0, 1e-36, 1e38, 3e38):
            for kw in (dict(), dict(k=4), dict(p=0.6), dict(mp=0.5), dict(k=700, p=0.9)):
                check_sample_on_borders(x, u, t, **kw)


@pytest.mark.parametrize("kw", [dict(p=1 - 2.0 ** -22), dict(k=(1 << 22) - 3, p=1 - 2.0 ** -22)])
def test_sample_tail_of_many_small_weights(kw):
    """2^22 logits: the last one weighs 1, the others about 2^-42 each, 2^-20 together, of which top-p leaves three quarters.
    Tokens of the tail come before the heavy one, so u well below their share picks one of them, at an index that the
    rounding of 64-bit sums (2^22 2^-53 of their value) moves by less than a thousandth."""
    V = 1 << 22
    x = torch.full((3, V), -42 * math.log(2), device="cuda")
    x[:, -1] = 0.0
    u = torch.tensor([2.0 ** -22, 1.7e-7, 0.9], device="cuda")
    tok = check_sample(x, u, **kw)
    assert int(tok[0]) < V // 2 and int(tok[2]) == V - 1


def test_sample_row_parameters():
    N, V = 60, 30011
    x = logits_like(N, V, torch.bfloat16, seed=3)
    x[:, :2] = -INF
    u = torch.rand(N, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    r = torch.arange(N, device="cuda")
    t = torch.tensor([0.0, 0.6, 1.0, 1.3, float("nan")], device="cuda")[r % 5]
    k = torch.tensor([0, 50, 20, -1, 200, 1, V], device="cuda")[r % 7]
    p = torch.tensor([1.0, 0.95, 0.9, 2.0], device="cuda")[r % 4]
    mp = torch.tensor([0.0, 0.0, 0.02], device="cuda")[r % 3]
    a = check_sample(x, u, t, k, p, mp)
    assert torch.equal(a, ops.sample(x, u, t, k.int(), p, mp))
    assert torch.equal(a[7:8], ops.sample(x[7:8], u[7:8], float(t[7]), int(k[7]), float(p[7]), float(mp[7])))


def test_sample_layouts():
    """Odd row strides and bases, a broadcast row, more leading dimensions, strided parameters."""
    big = logits_like(8, 6001, torch.bfloat16, seed=5)
    u = torch.rand(16, device="cuda")[::2]
    want = ops.sample(big[:, 3:4500].contiguous(), u.contiguous(), 0.8, 0, 0.9)
    assert torch.equal(ops.sample(big[:, 3:4500], u, 0.8, 0, 0.9), want)
    assert torch.equal(ops.sample(big[:, 3:4500].t().contiguous().t(), u, 0.8, 0, 0.9), want)
    one = ops.sample(big[2:3].expand(8, -1), u, 0.8, 0, 0.9)
    assert torch.equal(one, ops.sample(big[2:3].repeat(8, 1), u, 0.8, 0, 0.9))
    assert torch.equal(ops.sample(big[:, 3:4500].view(2, 4, -1), u.reshape(2, 4), 0.8, 0, 0.9).flatten(), want)
    assert ops.sample(big[:0], u[:0]).shape == (0,)
    assert ops.sample(big[0], u[0]).shape == ()


def test_sample_frequencies():
    """2^17 even draws hit each of 16 tokens as often as its weight says (inverse transform on an even grid: within
    one draw of the expected count at either end of the token's interval)."""
    w = torch.arange(1, 17, device="cuda", dtype=torch.float32)
    n = 1 << 17
    u = (torch.arange(n, device="cuda", dtype=torch.float64) / n).float()
    tok = ops.sample(w.log().expand(n, 16), u)
    count = torch.bincount(tok, minlength=16).double()
    assert bool(((count - n * (w / w.sum()).double()).abs() <= 2).all())


# ----------------------------------------------------------------------------------------------------------------------
# shared-prefix attention


def oracle(q, pk, pv, k, v, lengths, pre, scale):
    """(o, tolerance) in 64 bits. The tolerance counts: the rounding of each softmax weight to the inputs' type for the
    product with v (half a step u of each, so u sum p|v|), the rounding of the result (u |o|), scores summed in fp32 over D
    products (each weight off by at most twice D 2^-24 sum |q k| scale), and 2^-19 for fp32 exponentials, sums and the
    joining of partial results."""
    B, Lq, Hq, D = q.shape
    G, P, Hk = pk.shape[:3]
    S, u = k.shape[1], torch.finfo(q.dtype).eps / 2
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64,
                                                                                     device="cuda")
    for b in range(B):
        g = b // (B // G)
        n0, n1 = min(max(int(pre[g]), 0), P), min(max(int(lengths[b]), 0), S)
        keys = torch.cat([pk[g, :n0], k[b, :n1]]).double().repeat_interleave(Hq // Hk, 1)
        vals = torch.cat([pv[g, :n0], v[b, :n1]]).double().repeat_interleave(Hq // Hk, 1)
        if n0 + n1 == 0:
            continue
        s = torch.einsum("ihd,jhd->hij", q[b].double(), keys) * scale
        sa = torch.einsum("ihd,jhd->hij", q[b].double().abs(), keys.abs()) * scale
        hide = torch.arange(n0 + n1, device="cuda")[None] > (torch.arange(Lq, device="cuda") + n0 + n1 - Lq)[:, None]
        hide &= torch.arange(n0 + n1, device="cuda")[None] >= n0
        s = s.masked_fill(hide, -INF)
        p = torch.softmax(s, -1).nan_to_num()
        o = torch.einsum("hij,jhd->ihd", p, vals)
        a = torch.einsum("hij,jhd->ihd", p, vals.abs())
        d = 2 * D * 2.0 ** -24 * sa.masked_fill(hide, 0).amax(-1).t()[..., None] + 2.0 ** -19
        out[b], tol[b] = o, u * (a + o.abs()) + 2 * d * a
    # values below the type's normal range round by half a step of its smallest
    return out, tol * 1.01 + torch.finfo(q.dtype).tiny


def make(G, n, Lq, Hq, Hk, D, P, S, dtype, ragged, seed=0):
    B = G * n
    x = dict(q=2 * cuda(B, Lq, Hq, D, seed=seed), pk=cuda(G, P, Hk, D, seed=seed + 1), pv=cuda(G, P, Hk, D, seed=seed + 2),
             k=cuda(B, S, Hk, D, seed=seed + 3), v=cuda(B, S, Hk, D, seed=seed + 4))
    x = {a: t.to(dtype) for a, t in x.items()}
    lengths = torch.full((B,), S, dtype=torch.int32, device="cuda")
    pre = torch.full((G,), P, dtype=torch.int32, device="cuda")
    if ragged:
        lengths -= (torch.arange(B, device="cuda") * 37 % (S + 1)).int()
        pre -= (torch.arange(G, device="cuda") * 53 % (P + 1)).int()
        for t, m, c in ((x["v"], lengths, S), (x["k"], lengths, S), (x["pv"], pre, P), (x["pk"], pre, P)):
            t.masked_fill_((torch.arange(c, device="cuda") >= m[:, None])[:, :, None, None], float("nan"))
    return x, lengths, pre


def check_attention(x, lengths, pre, scale=None, args=None):
    got = ops.shared_prefix_attention(*(args or x.values()), lengths=lengths, prefix_lengths=pre, scale=scale)
    want, tol = oracle(x["q"], x["pk"], x["pv"], x["k"], x["v"], lengths, pre, scale or x["q"].shape[-1] ** -0.5)
    assert got.dtype == x["q"].dtype and got.is_contiguous() and bool(torch.isfinite(got).all())
    worst = ((got.double() - want).abs() - tol).max().item() if got.numel() else 0.0
    assert worst <= 0, worst
    return got


# G, n, Lq, Hq, Hk, D, P, S
SHAPES = [(1, 1, 1, 1, 1, 64, 1, 1), (1, 2, 1, 4, 4, 64, 37, 5), (1, 3, 1, 6, 2, 128, 128, 128),
          (1, 8, 1, 6, 2, 128, 1000, 33), (1, 5, 1, 24, 8, 128, 129, 257), (2, 3, 1, 24, 8, 128, 4099, 130),
          (1, 43, 1, 6, 2, 128, 700, 17), (1, 90, 1, 6, 2, 128, 1500, 40), (3, 50, 1, 6, 2, 64, 300, 9),
          (1, 130, 1, 3, 1, 128, 5000, 1), (1, 4, 24, 24, 8, 128, 333, 24), (1, 3, 50, 6, 2, 128, 260, 170),
          (2, 2, 7, 8, 1, 64, 90, 300), (1, 2, 129, 4, 4, 64, 50, 129), (4, 1, 1, 24, 8, 128, 2100, 1),
          (1, 6, 1, 40, 1, 128, 512, 64), (1, 3, 1, 128, 1, 128, 200, 20), (1, 2, 3, 256, 2, 64, 140, 70),
          (1, 1, 1, 2, 2, 128, 40000, 3), (5, 2, 2, 6, 2, 128, 127, 2500), (1, 300, 1, 2, 2, 64, 640, 300)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ragged", [False, True])
def test_shared_prefix(shape, dtype, ragged):
    x, lengths, pre = make(*shape, dtype, ragged, seed=sum(shape))
    check_attention(x, lengths, pre)


# hundreds of groups of one row each (nothing shared), as many with prefixes of a few keys, a whole prompt of queries, the
# fewest and the most heads a key / value head may have
MORE_SHAPES = [(300, 1, 1, 6, 2, 128, 50, 20), (700, 1, 1, 4, 4, 64, 3, 1), (64, 1, 1, 24, 8, 128, 700, 130),
               (1, 1, 1000, 6, 2, 128, 0, 1000), (2, 1, 300, 6, 2, 64, 200, 300), (40, 4, 2, 3, 3, 128, 129, 33),
               (2, 1, 1, 640, 1, 64, 300, 40)]


@pytest.mark.parametrize("shape", MORE_SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ragged", [False, True])
def test_shared_prefix_more_shapes(shape, dtype, ragged):
    x, lengths, pre = make(*shape, dtype, ragged, seed=sum(shape))
    check_attention(x, lengths, pre)


@pytest.mark.parametrize("P,S", [(0, 0), (0, 5), (70, 0), (0, 300), (1, 0)])
@pytest.mark.parametrize("n", [1, 60])
def test_shared_prefix_empty_sides(P, S, n):
    x, _, _ = make(2, n, 1, 6, 2, 128, P, S, torch.bfloat16, False)
    none = torch.zeros(2 * n, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    full = none[0] + S, none[1] + P
    check_attention(x, *full)
    got = check_attention(x, *none)
    assert not got.any()
    some = full[0].clone()
    some[::2] = 0
    check_attention(x, some, full[1])
    half = full[1].clone()
    half[0] = 0
    check_attention(x, some, half)


def test_shared_prefix_lengths_are_clamped():
    x, _, _ = make(2, 2, 1, 6, 2, 128, 140, 70, torch.bfloat16, False)
    lengths = torch.tensor([-5, 1 << 40, 70, 3], device="cuda")
    pre = torch.tensor([-1, 1 << 40], device="cuda")
    check_attention(x, lengths, pre)


def test_shared_prefix_queries_before_the_first_own_key():
    """More queries than own keys: the first ones see the prefix only (or nothing: zeros)."""
    x, _, _ = make(2, 3, 9, 6, 2, 128, 150, 12, torch.float16, False)
    lengths = torch.tensor([0, 1, 5, 8, 9, 12], dtype=torch.int32, device="cuda")
    check_attention(x, lengths, torch.tensor([150, 0], device="cuda"))


def test_shared_prefix_layouts():
    """Cache slices, a fused projection's columns, heads-first storage, odd alignment, broadcast prefixes."""
    x, lengths, pre = make(2, 4, 1, 6, 2, 128, 200, 50, torch.bfloat16, True)
    want = check_attention(x, lengths, pre)

    def slot(t, extra):                                   # a slice of a larger cache
        big = torch.full((t.shape[0] + 1, t.shape[1] + extra, *t.shape[2:]), float("nan"), device="cuda", dtype=t.dtype)
        big[:t.shape[0], :t.shape[1]] = t
        return big[:t.shape[0], :t.shape[1]]

    def heads_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def columns(t):                                       # [.., heads * D] columns of a wider projection
        big = torch.randn(*t.shape[:2], (t.shape[2] + 3) * t.shape[3], device="cuda").to(t.dtype)
        big = big.view(*t.shape[:2], t.shape[2] + 3, t.shape[3])
        big[:, :, 2:-1] = t
        return big[:, :, 2:-1]

    def odd(t):                                           # a base off the 16-byte grid
        flat = torch.empty(t.numel() + 3, device="cuda", dtype=t.dtype)
        flat[3:] = t.flatten()
        return flat[3:].view(t.shape)

    for f in (lambda t: slot(t, 7), heads_first, columns, odd):
        got = ops.shared_prefix_attention(*(f(t) for t in x.values()), lengths=lengths, prefix_lengths=pre)
        assert torch.equal(got, want)
    one = [x["q"], x["pk"][:1].expand(2, -1, -1, -1), x["pv"][:1].expand(2, -1, -1, -1), x["k"], x["v"]]
    same = dict(x, pk=one[1].contiguous(), pv=one[2].contiguous())
    check_attention(same, lengths, pre[:1].expand(2), args=one)
    assert torch.equal(ops.shared_prefix_attention(*x.values(), lengths=lengths.long().repeat_interleave(2)[::2],
                                                   prefix_lengths=pre.long()), want)
    assert ops.shared_prefix_attention(x["q"][:, :0], *list(x.values())[1:]).shape == (8, 0, 6, 128)
    assert ops.shared_prefix_attention(x["q"][:0], x["pk"], x["pv"], x["k"][:0], x["v"][:0]).shape == (0, 1, 6, 128)


def test_shared_prefix_scores_far_apart():
    """Maxima that grow by hundreds along the keys, weights that vanish in fp32, and the largest key at either end."""
    for seed, (pos, big) in enumerate([(0, 40.0), (999, 40.0), (500, -40.0)]):
        x, lengths, pre = make(1, 4, 1, 6, 2, 128, 1000, 60, torch.bfloat16, False, seed=seed)
        x["pk"] *= torch.linspace(0.1, 4.0, 1000, device="cuda")[None, :, None, None].to(torch.bfloat16)
        x["pk"][:, pos] = big * x["q"][0, 0, :2].sign()
        check_attention(x, lengths, pre, scale=0.3)


@pytest.mark.parametrize("G,n,Lq,P,S", [(2, 3, 1, 40, 9), (2, 20, 1, 3000, 300), (2, 70, 1, 900, 140), (2, 4, 5, 2000, 200)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shared_prefix_nan_reaches_the_result(G, n, Lq, P, S, dtype):
    """One NaN in a query, in a prefix key or in an own key makes the results that see it NaN, wherever the keys are cut
    into pieces, and leaves the bits of all others as they are. The PyTorch form says the same."""
    x, lengths, pre = make(G, n, Lq, 6, 2, 128, P, S, dtype, False)
    want = ops.shared_prefix_attention(*x.values(), lengths=lengths, prefix_lengths=pre)
    spots = {"q": (1, 0, 2, 7), "pk": (1, P - 5, 1, 3), "k": (0, S - Lq, 0, 127)}
    seen = {"q": (1, 0, 2), "pk": (slice(n, None), slice(None), slice(3, None)), "k": (0, slice(None), slice(0, 3))}
    for name, at in spots.items():
        for value in ((float("nan"), INF) if name == "q" else (float("nan"),)):
            y = {a: t.clone() for a, t in x.items()}
            y[name][at] = value
            bad = torch.zeros(want.shape[:3], dtype=torch.bool, device="cuda")
            bad[seen[name]] = True
            for backend in ("native", "torch"):
                ops.set_backend(backend)
                got = ops.shared_prefix_attention(*y.values(), lengths=lengths, prefix_lengths=pre)
                ops.set_backend("native")
                assert torch.equal(torch.isnan(got).all(-1), bad) and torch.equal(torch.isnan(got).any(-1), bad)
                if backend == "native":
                    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("P,S", [(3, 1), (1, 3), (40, 7), (700, 20)])
@pytest.mark.parametrize("sign", [1, -1])
def test_shared_prefix_largest_fp16_values(P, S, sign):
    """A mean of values at the end of fp16's range is there too, whatever the rounding of its weights: random ones, and one
    of 1 among many of 0.5 + 2^-12 + 2^-14, which fp16 rounds up by 0.75 2^-12, 1.5 half steps of the result."""
    x, lengths, pre = make(1, 40, 1, 6, 2, 128, P, S, torch.float16, False)
    for name in ("pv", "v"):
        x[name].fill_(sign * torch.finfo(torch.float16).max)
    check_attention(x, lengths, pre)
    s = math.log(0.5 + 2.0 ** -12 + 2.0 ** -14)
    coarse = float(torch.tensor(s).half())
    x["q"].zero_()
    x["q"][..., 0], x["q"][..., 1] = 1.0, 2.0 ** -6
    for name in ("pk", "k"):
        x[name].zero_()
        x[name][..., 0], x[name][..., 1] = coarse, 64 * (s - coarse)
    x["pk"][:, 0] = 0.0
    check_attention(x, lengths, pre, scale=1.0)


def test_shared_prefix_other_types():
    """fp32 and other head dims take the PyTorch expression."""
    for dtype, D in ((torch.float32, 128), (torch.float16, 32)):
        x, lengths, pre = make(2, 2, 2, 4, 2, D, 30, 9, dtype, True)
        check_attention(x, lengths, pre)


def test_shared_prefix_is_deterministic_and_row_independent():
    x, lengths, pre = make(1, 20, 1, 24, 8, 128, 3000, 90, torch.bfloat16, True)
    a = ops.shared_prefix_attention(*x.values(), lengths=lengths, prefix_lengths=pre)
    for _ in range(5):
        assert torch.equal(a, ops.shared_prefix_attention(*x.values(), lengths=lengths, prefix_lengths=pre))


def test_offsets_beyond_32_bits():
    """Rows, groups and positions 2^31 elements and more apart, in one buffer of 13 GB."""
    far = (1 << 31) + 1024
    buf = torch.zeros(3 * far, device="cuda", dtype=torch.bfloat16)
    x, lengths, pre = make(3, 1, 2, 6, 2, 128, 300, 70, torch.bfloat16, True)

    def spread(t, base, dim):                 # the steps along dim are `far`, everything else is dense
        shape = list(t.shape)
        shape[dim] = 1
        strides = [shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1]
        strides[dim] = far
        y = buf[base:].as_strided(t.shape, strides)
        return y.copy_(t)

    base, got = 0, []
    for name, t in x.items():
        got.append(spread(t, base, 0))
        base += 1 << 18
    check_attention(x, lengths, pre, args=got)
    one = dict(x, pk=x["pk"][:, :3], pv=x["pv"][:, :3], k=x["k"][:, :3], v=x["v"][:, :3])
    got = [spread(t, i << 18, 1) for i, t in enumerate(one.values())]
    check_attention(one, torch.tensor([3, 1, 2], device="cuda"), torch.tensor([2, 3, 1], device="cuda"), args=got)
    logits = logits_like(3, 30011, torch.bfloat16, seed=8)
    u = torch.rand(3, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")
    y = buf[5:].as_strided(logits.shape, (far + 3, 1))
    y.copy_(logits)
    for kw in (dict(t=0.8, p=0.95), dict(k=50), dict(mp=0.01), dict(t=0.0)):
        assert torch.equal(check_sample(y, u, **kw), check_sample(logits, u, **kw))


@pytest.mark.parametrize("n,Lq,P,S", [(20, 1, 3000, 90), (3, 24, 700, 150), (90, 1, 500, 30)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shared_prefix_rows_do_not_touch_one_another(n, Lq, P, S, dtype):
    """Other queries, own keys, values and lengths in all rows but one leave that row's bits as they are; so does another
    prefix in the other group."""
    x, lengths, pre = make(2, n, Lq, 6, 2, 128, P, S, dtype, True)
    want = ops.shared_prefix_attention(*x.values(), lengths=lengths, prefix_lengths=pre)
    for row in (0, n // 2, n, 2 * n - 1):
        g = row // n
        y, l2, p2 = make(2, n, Lq, 6, 2, 128, P, S, dtype, True, seed=50)
        l2, p2 = l2.flip(0).contiguous(), p2.clone()
        for name in ("k", "v"):
            y[name] = y[name].nan_to_num()
        for name in ("q", "k", "v"):
            y[name][row] = x[name][row]
        for name in ("pk", "pv"):
            y[name][g] = x[name][g]
        l2[row], p2[g] = lengths[row], pre[g]
        got = ops.shared_prefix_attention(*y.values(), lengths=l2, prefix_lengths=p2)
        assert torch.equal(got[row], want[row])
        assert not torch.equal(got, want)


# ----------------------------------------------------------------------------------------------------------------------
# ways of calling


def both_ops(x, lengths, pre, logits, u):
    o = ops.shared_prefix_attention(*x.values(), lengths=lengths, prefix_lengths=pre)
    return o, ops.sample(logits, u, 0.8, 0, 0.95)


def test_streams_and_concurrent_calls():
    cases = []
    for i in range(3):
        x, lengths, pre = make(1, 30, 1, 24, 8, 128, 2000 + 300 * i, 100, torch.bfloat16, True, seed=10 * i)
        cases.append((x, lengths, pre, logits_like(20, 30011, torch.bfloat16, seed=i), torch.rand(20, device="cuda")))
    want = [both_ops(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(10):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(both_ops(*c))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_captured_and_replayed():
    """One graph of a decode step's operators: lengths, logits and uniforms change between replays."""
    x, lengths, pre = make(1, 16, 1, 24, 8, 128, 1500, 64, torch.bfloat16, False)
    logits, u = logits_like(16, 20011, torch.bfloat16, seed=1), torch.rand(16, device="cuda")
    both_ops(x, lengths, pre, logits, u)
    graphs = []
    for _ in range(2):                                    # two graphs alive at once, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both_ops(x, lengths, pre, logits, u)
        graphs.append((g, out))
    for step in range(6):
        lengths.fill_(1 + 11 * step)
        pre.fill_(1500 - 200 * step)
        x["q"].copy_(cuda(*x["q"].shape, seed=step).to(torch.bfloat16))
        logits.copy_(logits_like(16, 20011, torch.bfloat16, seed=50 + step))
        u.copy_(torch.rand(16, device="cuda"))
        g, out = graphs[step % 2]
        g.replay()
        torch.cuda.synchronize()
        want = both_ops(x, lengths, pre, logits, u)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_native_refusals():
    C = ops._C()
    x, lengths, pre = make(1, 4, 1, 6, 2, 128, 20, 5, torch.bfloat16, False)
    q, pk, pv, k, v = x.values()
    for args in ((q.float(), pk, pv, k, v), (q, pk.half(), pv, k, v), (q, pk[:, :10], pv, k, v), (q, pk, pv, k[:2], v[:2]),
                 (q[..., :32], pk[..., :32], pv[..., :32], k[..., :32], v[..., :32]), (q.cpu(), pk, pv, k, v)):
        with pytest.raises(RuntimeError):
            C.shared_prefix_attention(*args, None, None, 0.1)
    with pytest.raises(RuntimeError):
        C.shared_prefix_attention(q, pk, pv, k, v, lengths[:2], None, 0.1)
    logits, u = cuda(4, 100), torch.rand(4, device="cuda")
    for a in ((logits.double(), u), (logits, u[:2]), (logits.cpu(), u), (logits.t(), u)):
        with pytest.raises(RuntimeError):
            C.sample(*a, None, 1.0, None, 0, None, 1.0, None, 0.0, False)
    with pytest.raises(ValueError):
        ops.sample(logits, u.cpu())
    with pytest.raises(ValueError):
        ops.shared_prefix_attention(q, pk, pv, k, v, lengths=lengths.cpu())


@pytest.mark.parametrize("scale", [1e-46, 1e-39, 1e39, 1e300])
def test_shared_prefix_refuses_scales_outside_fp32(scale):
    """Zero or infinite as an fp32 factor: hidden keys' -inf would become NaN."""
    x, lengths, pre = make(1, 4, 1, 6, 2, 128, 20, 5, torch.bfloat16, True)
    with pytest.raises(RuntimeError):
        ops._C().shared_prefix_attention(*x.values(), lengths, pre, scale)
    with pytest.raises(ValueError):
        ops.shared_prefix_attention(*x.values(), lengths=lengths, prefix_lengths=pre, scale=scale)


def test_shared_prefix_refuses_pieces_of_seconds():
    """2^27 keys (overlapping rows of one buffer) against two blocks of queries an SM: each SM's share of one block would take
    longer than the kernel's waits may. Refused before anything is launched."""
    n = torch.cuda.get_device_properties(0).multi_processor_count * 256
    pk = torch.zeros((1 << 27) * 8 + 128, device="cuda", dtype=torch.bfloat16).as_strided((1, 1 << 27, 1, 128), (8, 8, 8, 1))
    q, own = (torch.zeros(n, s, 1, 128, device="cuda", dtype=torch.bfloat16) for s in (1, 0))
    with pytest.raises(RuntimeError, match="too many keys"):
        ops.shared_prefix_attention(q, pk, pk, own, own)


@pytest.mark.parametrize("scale", [2.0 ** -126, 1e-30, 1e-3])
def test_shared_prefix_small_scales(scale):
    x, lengths, pre = make(2, 4, 1, 6, 2, 128, 200, 50, torch.bfloat16, True)
    check_attention(x, lengths, pre, scale=scale)


# ----------------------------------------------------------------------------------------------------------------------
# the run of them that generation makes


def test_sampled_generation_native():
    """Forked decoding of one prompt: each step's hidden states agree with those of the repeated prompt, and every token
    is the one drawn from its logits."""
    from faster_yoco_b200.config import build_args
    from faster_yoco_b200.models.yoco import YOCO
    torch.manual_seed(0)
    with torch.device("cuda"):
        m = YOCO(build_args("yoco_small", vocab_size=264, max_seq_len=1024, max_batch_size=1, init_std=0.02))
    m = m.to(torch.bfloat16).eval()
    prompt = torch.randint(3, 264, (2, 300), device="cuda")
    n = 5
    with torch.no_grad():
        one, many = {}, {}
        m(prompt[:, :-1], incremental_state=one, start_pos=0, is_prefilling=True, skip_cross_decoder=True)
        wide = prompt.repeat_interleave(n, 0)
        m(wide[:, :-1], incremental_state=many, start_pos=0, is_prefilling=True, skip_cross_decoder=True)
        forked = m.fork_state(one, 2, n)
        cur = wide[:, -1:]
        for step in range(6):
            pos = prompt.shape[1] - 1 + step
            a, _ = m(cur, incremental_state=forked, start_pos=pos, is_prefilling=False)
            b, _ = m(cur, incremental_state=many, start_pos=pos, is_prefilling=False)
            err = (a.float() - b.float()).abs().max() / b.float().abs().max()
            assert err < 3e-2
            cur = ops.sample(a[:, -1], torch.rand(2 * n, device="cuda"), 1.0, 50, 0.95)[:, None]
    assert forked["prefix_key"].data_ptr() == one["prev_key"].data_ptr()
    assert forked["prev_key"].shape[1] < one["prev_key"].shape[1]


def test_a_forked_state_outlives_what_its_parent_does_native():
    """The kernels update the retention states and the K / V cache in place: what the parent does after a fork, behind the
    prompt, inside it and over all of it, leaves the bits of the forked rows' logits as they are."""
    from faster_yoco_b200.config import build_args
    from faster_yoco_b200.models.yoco import YOCO
    torch.manual_seed(0)
    with torch.device("cuda"):
        m = YOCO(build_args("yoco_small", vocab_size=264, max_seq_len=1024, max_batch_size=1))
    m = m.to(torch.bfloat16).eval()
    prompt, other = (torch.randint(3, 264, (2, 300), device="cuda") for _ in range(2))
    for copies in (1, 3):
        step = torch.randint(3, 264, (2 * copies, 1), device="cuda")

        def decode(forked):
            return torch.cat([m(step, incremental_state=forked, start_pos=300 + i, is_prefilling=False)[0] for i in range(3)])

        with torch.no_grad():
            state = {}
            m(prompt, incremental_state=state, start_pos=0, is_prefilling=True, skip_cross_decoder=True)
            want = decode(m.fork_state(state, 2, copies))
            first, second, third = (m.fork_state(state, 2, copies) for _ in range(3))
            m(prompt[:, :1], incremental_state=state, start_pos=300, is_prefilling=False)
            assert torch.equal(decode(first), want)
            m(prompt[:, :1], incremental_state=state, start_pos=200, is_prefilling=False)
            assert torch.equal(decode(second), want)
            m(other, incremental_state=state, start_pos=0, is_prefilling=True, skip_cross_decoder=True)
            assert torch.equal(decode(third), want)


def test_generate_samples_native():
    from faster_yoco_b200.config import build_args
    from faster_yoco_b200.data.tokenizers import ByteTokenizer
    from faster_yoco_b200.eval.generate import generate
    from faster_yoco_b200.models.yoco import YOCO
    torch.manual_seed(0)
    with torch.device("cuda"):
        m = YOCO(build_args("yoco_small", vocab_size=264, max_seq_len=512, max_batch_size=1))
    m = m.to(torch.bfloat16).eval()
    tok = ByteTokenizer()
    prompt = torch.tensor([tok.encode("x" * 300, bos=True)], device="cuda")
    gen = lambda: torch.Generator(device="cuda").manual_seed(3)
    kw = dict(generate_tokens=6, chunk_length=128, num_samples=8, temperature=0.9, top_p=0.95)
    out = generate(m, prompt, tok, generator=gen(), **kw)
    assert out.shape == (8, prompt.shape[1] + 6) and bool((out[:, :prompt.shape[1]] == prompt).all())
    assert torch.equal(out, generate(m, prompt, tok, generator=gen(), **kw))
    assert bool((out[:, prompt.shape[1]] >= 0).all())


@pytest.mark.parametrize("kw", [dict(top_p=0.95), dict(top_k=20, temperature=1.3), dict(min_p=0.02, top_k=40, top_p=0.9)])
def test_generate_draws_the_definitions_tokens(kw, monkeypatch):
    """Every token of a generation on the kernels is the 64-bit form's, for the logits that the model gave at that step, the
    generator's next uniform numbers and the settings that were asked for."""
    from faster_yoco_b200.config import build_args
    from faster_yoco_b200.data.tokenizers import ByteTokenizer
    from faster_yoco_b200.eval.generate import generate
    from faster_yoco_b200.models.yoco import YOCO
    torch.manual_seed(0)
    with torch.device("cuda"):
        m = YOCO(build_args("yoco_small", vocab_size=264, max_seq_len=512, max_batch_size=1))
    m = m.to(torch.bfloat16).eval()
    tok, n, steps = ByteTokenizer(), 8, 6
    prompts = torch.tensor([tok.encode("x" * 300, bos=True), tok.encode("y" * 300, bos=True)], device="cuda")
    P = prompts.shape[1]
    kw = dict(dict(temperature=0.9), **kw)
    given, plain = [], YOCO.forward

    def forward(self, *a, **k):
        out = plain(self, *a, **k)
        if not k["is_prefilling"]:
            given.append((a[0].clone(), out[0][:, -1].float()))
        return out

    monkeypatch.setattr(YOCO, "forward", forward)
    out = generate(m, prompts, tok, generate_tokens=steps, chunk_length=128, num_samples=n,
                   generator=torch.Generator(device="cuda").manual_seed(5), **kw)
    gen = torch.Generator(device="cuda").manual_seed(5)
    N = 2 * n
    pars = (rows_of(kw["temperature"], N, torch.float32), rows_of(kw.get("top_k", 0), N, torch.int64),
            rows_of(kw.get("top_p", 1.0), N, torch.float32), rows_of(kw.get("min_p", 0.0), N, torch.float32))
    ended = torch.zeros(N, dtype=torch.bool, device="cuda")
    assert len(given) == steps or bool((out[:, P:] == tok.eos_id).any(1).all())
    for i, (fed, logits) in enumerate(given):
        assert torch.equal(fed[:, 0], out[:, P + i - 1])
        logits[:, tok.bos_id] = logits[:, tok.pad_id] = -INF
        want, _ = ref.sample(logits, torch.rand(N, generator=gen, device="cuda"), *pars)
        want = torch.where(ended, torch.full_like(want, tok.pad_id), want)
        assert torch.equal(out[:, P + i], want)
        ended |= want == tok.eos_id
    assert len({tuple(r.tolist()) for r in out[:n, P:]}) > 1
