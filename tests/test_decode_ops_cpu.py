"""Sampling and shared-prefix attention on the CPU: the PyTorch forms against brute-force definitions in 64 bits, the
refusals, and generation of several sampled continuations of one prompt."""
import math

import numpy as np
import pytest
import torch

from faster_yoco_b200 import ops
from faster_yoco_b200.config import build_args
from faster_yoco_b200.data.tokenizers import ByteTokenizer

INF = float("inf")


# ----------------------------------------------------------------------------------------------------------------------
# sampling


def brute_sample(x, u, t, k, p, mp):
    """One row by the definition, on Python lists."""
    x = [float(v) for v in x]
    order = sorted((i for i, v in enumerate(x) if v > -INF), key=lambda i: (-x[i], i))     # NaN > -inf is false
    if not order:
        return -1, -INF
    if not t > 0:
        return order[0], 0.0
    top = x[order[0]]
    w = {i: 1.0 if x[i] == top else (0.0 if top == INF else math.exp(max((x[i] - top) / t, -1e4))) for i in order}
    if k > 0:
        order = order[:k]
    if p < 1:
        total, run, n = math.fsum(w[i] for i in order), 0.0, 0
        while n == 0 or (n < len(order) and run < p * total):
            run += w[order[n]]
            n += 1
        order = order[:n]
    kept = sorted([order[0]] + [i for i in order[1:] if w[i] >= mp])
    total, run = math.fsum(w[i] for i in kept), 0.0
    for i in kept:
        run += w[i]
        if run > u * total:
            break
    return i, math.log(w[i] / total)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (0.8, 0, 0.9, 0.0), (1.3, 20, 0.8, 0.0), (1.0, 0, 1.0, 0.2),
            (0.9, 12, 0.95, 0.05), (0.0, 3, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0)]


@pytest.mark.parametrize("t,k,p,mp", SETTINGS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_matches_definition(t, k, p, mp, dtype):
    g = torch.Generator().manual_seed(3)
    x = (2 * torch.randn(40, 37, generator=g)).to(dtype)           # bf16: many ties
    x[::5, ::3] = -INF
    x[1::7, 4] = float("nan")
    u = torch.rand(40, generator=g)
    tok, lp = ops.sample(x, u, t, k, p, mp, return_logprob=True)
    t32, p32, mp32 = (float(np.float32(v)) for v in (t, p, mp))
    for r in range(40):
        want, wlp = brute_sample(x[r].tolist(), float(u[r]), t32, k, p32, mp32)
        assert int(tok[r]) == want
        # both sides round one 64-bit value to fp32
        assert abs(float(lp[r]) - wlp) <= 2 ** -23 * abs(wlp) + 1e-12


def test_sample_edges_cpu():
    x = torch.tensor([[-INF, -INF, -INF], [float("nan")] * 3, [0.0, INF, INF], [1.0, 1.0, 1.0], [-0.0, 0.0, -1.0]])
    u = torch.tensor([0.5, 0.5, 0.75, 0.0, 0.0])
    tok, lp = ops.sample(x, u, return_logprob=True)
    assert tok.tolist() == [-1, -1, 2, 0, 0]
    assert lp[0] == -INF and lp[1] == -INF and abs(float(lp[2]) - math.log(0.5)) < 1e-6
    assert ops.sample(x, u, 0.0).tolist() == [-1, -1, 1, 0, 0]
    assert ops.sample(x[3:], torch.tensor([0.999, 0.0]), top_k=1).tolist() == [0, 0]       # ties: lowest index
    assert ops.sample(x[0], torch.tensor(0.5)).shape == ()
    assert ops.sample(x.view(5, 1, 3), u.view(5, 1)).shape == (5, 1)
    assert ops.sample(x[:0], u[:0]).shape == (0,)


def test_sample_row_parameters_cpu():
    g = torch.Generator().manual_seed(5)
    x, u = torch.randn(10, 50, generator=g), torch.rand(10, generator=g)
    t = torch.tensor([s[0] for s in SETTINGS])
    k = torch.tensor([s[1] for s in SETTINGS])
    p = torch.tensor([s[2] for s in SETTINGS])
    mp = torch.tensor([s[3] for s in SETTINGS])
    got = ops.sample(x, u, t, k, p, mp)
    for r, s in enumerate(SETTINGS):
        assert int(got[r]) == int(ops.sample(x[r:r + 1], u[r:r + 1], *s))


def test_sample_refusals():
    x, u = torch.randn(2, 4), torch.rand(2)
    bad = [(x.double(), u, {}), (x, u.double(), {}), (x, u[:1], {}), (x[:, :0], u, {}), (x, u, {"temperature": -1.0}),
           (x, u, {"temperature": float("nan")}), (x, u, {"top_p": -0.1}), (x, u, {"min_p": 1.5}),
           (x, u, {"top_k": torch.ones(2)}), (x, u, {"top_p": torch.ones(3)}), (x, u, {"min_p": torch.ones(2).double()})]
    for xx, uu, kw in bad:
        with pytest.raises(ValueError):
            ops.sample(xx, uu, **kw)
    with pytest.raises(RuntimeError):
        ops.sample(x.requires_grad_(), u)
    with torch.no_grad():
        ops.sample(x, u)


@pytest.mark.parametrize("top_k", [0.5, 2.7, -0.1, INF, -INF, float("nan")])
def test_sample_refuses_a_top_k_that_is_no_whole_number(top_k):
    """0.5 is not the 0 that keeps everything."""
    x, u = torch.randn(2, 4), torch.rand(2)
    with pytest.raises(ValueError, match="top_k"):
        ops.sample(x, u, top_k=top_k)
    assert torch.equal(ops.sample(x, u, top_k=2.0), ops.sample(x, u, top_k=2))
    assert torch.equal(ops.sample(x, u, top_k=-(1 << 50)), ops.sample(x, u))
    assert torch.equal(ops.sample(x, u, top_k=1 << 50), ops.sample(x, u))


# ----------------------------------------------------------------------------------------------------------------------
# shared-prefix attention


def brute_attention(q, pk, pv, k, v, lengths, prefix_lengths):
    B, Lq, Hq, D = q.shape
    G, Hk = pk.shape[0], pk.shape[2]
    out = torch.zeros(B, Lq, Hq, D, dtype=torch.float64)
    for b in range(B):
        g = b // (B // G)
        for i in range(Lq):
            n = max(0, min(int(lengths[b]), int(lengths[b]) - Lq + i + 1))
            for h in range(Hq):
                hk = h // (Hq // Hk)
                keys = torch.cat([pk[g, :prefix_lengths[g], hk], k[b, :n, hk]]).double()
                vals = torch.cat([pv[g, :prefix_lengths[g], hk], v[b, :n, hk]]).double()
                if len(keys):
                    w = torch.softmax(keys @ q[b, i, h].double() / math.sqrt(D), 0)
                    out[b, i, h] = w @ vals
    return out


@pytest.mark.parametrize("G,n,Lq,Hq,Hk,P,S", [(1, 3, 1, 4, 4, 9, 5), (2, 2, 3, 6, 2, 7, 6), (3, 1, 1, 2, 1, 0, 4),
                                              (1, 2, 2, 2, 2, 5, 0), (1, 1, 1, 2, 2, 0, 0)])
def test_shared_prefix_matches_definition(G, n, Lq, Hq, Hk, P, S):
    gen = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=gen)
    B, D = G * n, 16
    q, pk, pv, k, v = r(B, Lq, Hq, D), r(G, P, Hk, D), r(G, P, Hk, D), r(B, S, Hk, D), r(B, S, Hk, D)
    lengths = torch.tensor([(S - b) % (S + 1) for b in range(B)])
    pre = torch.tensor([max(0, P - 2 * g) for g in range(G)], dtype=torch.int32)
    v.masked_fill_((torch.arange(S) >= lengths[:, None])[:, :, None, None], float("nan"))
    got = ops.shared_prefix_attention(q, pk, pv, k, v, lengths, pre)
    assert torch.isfinite(got).all()
    torch.testing.assert_close(got.double(), brute_attention(q, pk, pv, k, v, lengths, pre), rtol=1e-5, atol=1e-5)
    full = ops.shared_prefix_attention(q, pk, pv, k.nan_to_num(), v.nan_to_num())
    want = brute_attention(q, pk, pv, k.nan_to_num(), v.nan_to_num(), [S] * B, [P] * G)
    torch.testing.assert_close(full.double(), want, rtol=1e-5, atol=1e-5)


def test_shared_prefix_equals_attention():
    """With one row a group and nothing masked it is the causal attention over the concatenated keys."""
    gen = torch.Generator().manual_seed(8)
    r = lambda *s: torch.randn(*s, generator=gen)
    q, pk, pv, k, v = r(2, 3, 4, 16), r(2, 9, 2, 16), r(2, 9, 2, 16), r(2, 3, 2, 16), r(2, 3, 2, 16)
    got = ops.shared_prefix_attention(q, pk, pv, k, v)
    want = ops.ref.attention(q, torch.cat([pk, k], 1), torch.cat([pv, v], 1), q_offset=9)
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)


def test_shared_prefix_nan_reaches_the_result():
    """A NaN query, and a NaN or +inf score among those that a query sees, give NaN; all other results stay as they are."""
    gen = torch.Generator().manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=gen)
    q, pk, pv, k, v = r(4, 3, 4, 16), r(2, 9, 2, 16), r(2, 9, 2, 16), r(4, 5, 2, 16), r(4, 5, 2, 16)
    want = ops.shared_prefix_attention(q, pk, pv, k, v)
    bad = torch.zeros(4, 3, 4, dtype=torch.bool)
    q[0, 1, 2, 5] = float("nan")
    bad[0, 1, 2] = True
    pk[1, 4, 1, 0] = float("nan")              # rows 2 and 3, the second key / value head's query heads
    bad[2:, :, 2:] = True
    k[1, 3, 0, 7] = float("nan")               # own key 3 of 5: of three queries the last two see it
    bad[1, 1:, :2] = True
    k[3, 0, 0] = INF * q[3, 0, 0].sign()       # a score of +inf for one query, of mixed signs (NaN) for the others
    bad[3, :, 1] = torch.isnan(q[3, :, 1] @ k[3, 0, 0]) | ((q[3, :, 1] @ k[3, 0, 0]) == INF)
    bad[3, :, 0] = True
    got = ops.shared_prefix_attention(q, pk, pv, k, v)
    assert torch.equal(torch.isnan(got).all(-1), bad) and torch.equal(torch.isnan(got).any(-1), bad)
    torch.testing.assert_close(got[~bad], want[~bad], rtol=1e-6, atol=1e-6)


def test_shared_prefix_refusals():
    r = torch.randn
    q, pk, k = r(4, 1, 4, 16), r(2, 5, 2, 16), r(4, 3, 2, 16)
    ok = (q, pk, pk, k, k)
    ops.shared_prefix_attention(*ok)
    bad = [((q, r(3, 5, 2, 16), r(3, 5, 2, 16), k, k), {}), ((q, pk, r(2, 4, 2, 16), k, k), {}),
           ((q, pk, pk, r(3, 3, 2, 16), r(3, 3, 2, 16)), {}), ((r(4, 1, 3, 16), pk, pk, k, k), {}),
           ((q.half(), pk, pk, k, k), {}), ((q[0], pk, pk, k, k), {}), ((r(4, 1, 4, 8), pk, pk, k, k), {}),
           (ok, {"lengths": torch.zeros(3, dtype=torch.int32)}), (ok, {"lengths": torch.zeros(4)}),
           (ok, {"prefix_lengths": torch.zeros(4, dtype=torch.int32)})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(*args, **kw)
    with pytest.raises(RuntimeError):
        ops.shared_prefix_attention(q.clone().requires_grad_(), pk, pk, k, k)


# ----------------------------------------------------------------------------------------------------------------------
# generation


def _tiny(**kw):
    from faster_yoco_b200.models.yoco import YOCO
    torch.manual_seed(0)
    return YOCO(build_args("yoco_tiny", vocab_size=264, n_layers=2, max_seq_len=512, max_batch_size=2, **kw)).eval()


@pytest.mark.parametrize("window", [None, 16])
@pytest.mark.parametrize("text", ["the magic number of the city is", "two\x00", ""])
def test_forked_greedy_matches_repeated_prompt(text, window):
    from faster_yoco_b200.eval.generate import generate
    ops.set_backend("torch")
    m, tok = _tiny(sliding_window=window), ByteTokenizer()
    ids = tok.encode(text, bos=True)
    prompt = torch.tensor([ids, ids[::-1]])
    out = generate(m, prompt, tok, generate_tokens=5, chunk_length=8, num_samples=3)
    want = generate(m, prompt.repeat_interleave(3, 0), tok, generate_tokens=5, chunk_length=8)
    assert torch.equal(out, want)


def test_sampled_generation():
    """Every drawn token is the one the definition gives for the logits of the whole sequence so far."""
    from faster_yoco_b200.eval.generate import generate
    ops.set_backend("torch")
    m, tok = _tiny(), ByteTokenizer()
    prompt = torch.tensor([tok.encode("a long shared prompt", bos=True)])
    gen = torch.Generator().manual_seed(11)
    out = generate(m, prompt, tok, generate_tokens=6, chunk_length=8, num_samples=4, temperature=0.9, top_k=40,
                   top_p=0.95, generator=gen)
    assert out.shape == (4, prompt.shape[1] + 6)
    gen = torch.Generator().manual_seed(11)
    for step in range(prompt.shape[1], out.shape[1]):
        with torch.no_grad():
            lg = m(out[:, :step])[0][:, -1].float()
        lg[:, tok.bos_id] = lg[:, tok.pad_id] = -INF
        nxt = ops.sample(lg, torch.rand(4, generator=gen), 0.9, 40, 0.95)
        done = (out[:, prompt.shape[1]:step] == tok.eos_id).any(1)
        assert torch.equal(out[~done, step], nxt[~done])
        if bool((out[:, prompt.shape[1]:step + 1] == tok.eos_id).any(1).all()):
            break
    assert len({tuple(r.tolist()) for r in out}) > 1


def test_sampled_generation_of_other_models():
    from faster_yoco_b200.eval.generate import generate
    from faster_yoco_b200.models.transformer import LLaMA, Transformer, llama_args_from_cfg
    ops.set_backend("torch")
    torch.manual_seed(0)
    m = LLaMA(Transformer(llama_args_from_cfg(64, 2, 2, 1, 264, batch_size=4, tokens_per_sample=64))).eval()
    tok = ByteTokenizer()
    prompt = torch.tensor([tok.encode("abc", bos=True)])
    out = generate(m, prompt, tok, generate_tokens=3, chunk_length=8, yoco=False, num_samples=3, temperature=1.0,
                   generator=torch.Generator().manual_seed(1))
    assert out.shape == (3, prompt.shape[1] + 3)


@pytest.mark.parametrize("window", [None, 16])
@pytest.mark.parametrize("copies", [1, 3])
def test_a_forked_state_outlives_what_its_parent_does(window, copies):
    """The parent goes on behind the prompt, starts again inside it and is overwritten from its first position; states
    that were forked before each of these decode as if it had rested."""
    ops.set_backend("torch")
    m = _tiny(sliding_window=window)
    gen = torch.Generator().manual_seed(2)
    prompt, other = (torch.randint(3, 264, (2, 40), generator=gen) for _ in range(2))
    step = torch.randint(3, 264, (2 * copies, 1), generator=gen)

    def fill(state, ids, at):
        m(ids, incremental_state=state, start_pos=at, is_prefilling=True, skip_cross_decoder=True)

    def decode(forked):
        return torch.cat([m(step, incremental_state=forked, start_pos=40 + i, is_prefilling=False)[0] for i in range(2)], 1)

    with torch.no_grad():
        state = {}
        fill(state, prompt, 0)
        want = decode(m.fork_state(state, 2, copies))
        first, second = m.fork_state(state, 2, copies), m.fork_state(state, 2, copies)
        cache = state["prev_key"]
        m(prompt[:, :1], incremental_state=state, start_pos=40, is_prefilling=False)
        assert state["prev_key"] is cache                  # behind the prompt nothing has to move
        assert torch.equal(decode(first), want)
        m(prompt[:, :1], incremental_state=state, start_pos=20, is_prefilling=False)
        fill(state, other, 0)
        assert torch.equal(decode(second), want)
        assert state["prev_key"] is not cache and "lent" not in state
    long = {}
    with torch.no_grad():                                  # a cache that grows leaves the lent one behind
        fill(long, prompt, 0)
        forked = m.fork_state(long, 2, copies)
        fill(long, torch.randint(3, 264, (2, 600), generator=gen), 0)
        assert "lent" not in long and torch.equal(decode(forked), want)


class _Scripted(torch.nn.Module):
    """A model whose logits at a position are given: [rows, vocabulary] by position."""

    def __init__(self, logits):
        super().__init__()
        self.logits = logits

    def forward(self, x, incremental_state=None, start_pos=0, is_prefilling=True, **_):
        return (None if is_prefilling else self.logits[start_pos][:, None].clone()), None


@pytest.mark.parametrize("nothing", [float("nan"), -INF])
def test_sampled_generation_of_a_row_without_candidates(nothing):
    """Logits that leave nothing to draw end generation with an error, unless the row has ended before."""
    from faster_yoco_b200.eval.generate import generate
    ops.set_backend("torch")
    tok = ByteTokenizer()
    prompt = torch.tensor([tok.encode("ab", bos=True)] * 3)
    P = prompt.shape[1]
    gen = torch.Generator().manual_seed(0)
    logits = {P - 1 + i: torch.randn(3, 264, generator=gen) for i in range(4)}
    logits[P - 1][1] = -INF                    # row 1 ends with its first token
    logits[P - 1][1, tok.eos_id] = 0.0
    logits[P - 1][::2, tok.eos_id] = -INF
    logits[P][1] = nothing
    logits[P][::2, tok.eos_id] = -INF
    m = _Scripted(logits)
    out = generate(m, prompt, tok, generate_tokens=2, temperature=1.0, yoco=False)
    assert bool((out >= 0).all()) and int(out[1, P]) == tok.eos_id and int(out[1, P + 1]) == tok.pad_id
    logits[P + 1][2] = nothing
    with pytest.raises(RuntimeError, match=r"rows \[2\]"):
        generate(m, prompt, tok, generate_tokens=3, temperature=1.0, yoco=False)


def test_fork_state_refuses_misuse():
    from faster_yoco_b200.eval.generate import generate
    ops.set_backend("torch")
    m, tok = _tiny(), ByteTokenizer()
    with pytest.raises(ValueError):
        generate(m, torch.tensor([[1, 2]]), tok, num_samples=0)
    with pytest.raises(ValueError):
        generate(m, torch.tensor([[1, 2]]), tok, temperature=-0.5)
    state = {}
    with torch.no_grad():
        m(torch.tensor([[5, 6, 7]]), incremental_state=state, start_pos=0, is_prefilling=True, skip_cross_decoder=True)
        forked = m.fork_state(state, 1, 2)
        with pytest.raises(ValueError):
            m.fork_state(forked, 2, 2)
        with pytest.raises(ValueError):
            m(torch.tensor([[5], [6]]), incremental_state=forked, start_pos=2, is_prefilling=False)


def _tp_generation_worker(rank, world, full_sd, prompt, want):
    from faster_yoco_b200.eval.generate import generate
    from faster_yoco_b200.models.yoco import YOCO, shard_state_dict
    from faster_yoco_b200.parallel import tp
    ops.set_backend("torch")
    tp.init_model_parallel(world)
    m = YOCO(build_args("yoco_tiny", vocab_size=264, n_layers=2, max_seq_len=512, max_batch_size=2,
                        model_parallel_size=world)).eval()
    m.load_state_dict(shard_state_dict(full_sd, world, rank), strict=True)
    out = generate(m, prompt, ByteTokenizer(), generate_tokens=8, chunk_length=8, num_samples=3, temperature=1.0, top_p=0.9,
                   generator=torch.Generator().manual_seed(20 + rank))
    assert torch.equal(out, want)
    tp.destroy_model_parallel()


def test_sampled_generation_of_tensor_parallel_ranks():
    """Two ranks whose generators differ go on with the same tokens: those of one rank with the first one's generator."""
    from faster_yoco_b200.eval.generate import generate
    from faster_yoco_b200.utils.launch import run_ranks
    ops.set_backend("torch")
    m, tok = _tiny(), ByteTokenizer()
    prompt = torch.tensor([tok.encode("two ranks", bos=True)])
    want = generate(m, prompt, tok, generate_tokens=8, chunk_length=8, num_samples=3, temperature=1.0, top_p=0.9,
                    generator=torch.Generator().manual_seed(20))
    run_ranks(_tp_generation_worker, 2, {k: v.detach().clone() for k, v in m.state_dict().items()}, prompt, want)
