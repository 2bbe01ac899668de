"""The next token of every row of logits, against 64 bits on the CPU."""
import math

import numpy as np
import pytest
import torch

import paged_oracle as po
from kmll_b200 import ops

pytestmark = pytest.mark.gpu


def dev(v, dtype):
    return torch.tensor(np.asarray(v), dtype=dtype, device="cuda")


def check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, borders=0):
    """The operator's weights are within 2^-45 of the largest one each: a border that is 2^-44 * vocab of the whole from u or p may fall on either
    side (float64 sums differ by less), so such rows, `borders` of them by construction, are not compared here; the log-probability is off by that over the token's weight, and by its rounding."""
    rows, vocab = logits.shape
    settings = [None if x is None else dev(x, d) for x, d in ((temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32), (min_p, torch.float32))]
    tokens, logprobs = ops.sample_rows(logits, dev(u, torch.float64), *settings)
    x = logits.double().cpu().numpy()
    close = 0
    for r in range(rows):
        t, lp, gap = po.sample(x[r], float(u[r]), *(d if s is None else float(s[r]) if s.is_floating_point() else int(s[r])
                                                    for s, d in zip(settings, (1.0, 0, 1.0, 0.0))))
        if gap < 2.0 ** -44 * vocab:
            close += 1
            continue
        assert tokens[r].item() == t, (r, tokens[r].item(), t, gap)
        if math.isinf(lp):
            assert logprobs[r].item() == lp
        else:
            assert abs(logprobs[r].item() - lp) <= 2.0 ** -24 * abs(lp) + vocab * 2.0 ** -44 * math.exp(-max(lp, -40.0)) + 1e-12
    assert close <= max(1, rows // 20, borders)
    return tokens, logprobs


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 2), (5, 31), (20, 1000), (40, 4099), (80, 32000), (7, 151936), (33, 50257)])
def test_all_settings(cuda, dtype, rows, vocab):
    rng = np.random.default_rng(rows + vocab)
    logits = torch.tensor(rng.normal(0, 1, (rows, vocab)) * rng.uniform(0.2, 6, (rows, 1)), device="cuda").to(dtype)
    check(logits, rng.random(rows), rng.uniform(0.3, 2.0, rows), rng.choice([0, 1, 2, 20, 400, vocab, 10 ** 9], rows), rng.choice([1.0, 0.0, 0.3, 0.9, 0.999], rows),
          rng.choice([0.0, 0.01, 0.3, 1.0], rows))


@pytest.mark.parametrize("name", ["none", "temperature", "top_k", "top_p", "min_p"])
def test_one_setting_alone(cuda, name):
    rng = np.random.default_rng(7)
    logits = torch.tensor(rng.normal(0, 2, (24, 5000)), device="cuda", dtype=torch.float32)
    value = dict(none={}, temperature=dict(temperature=np.linspace(0.1, 3, 24)), top_k=dict(top_k=np.arange(1, 25)), top_p=dict(top_p=np.linspace(0.02, 1.0, 24)),
                 min_p=dict(min_p=np.linspace(0.0, 1.0, 24)))[name]
    check(logits, np.linspace(0.0, 0.99999, 24), **value)


def test_equal_logits_go_by_index(cuda):
    """Flat rows: every token weighs the same, so token = floor(u * n); more than can be ranked at once."""
    vocab = 100003
    u = (np.arange(20) + 0.5) / 20
    tokens, logprobs = ops.sample_rows(torch.zeros(20, vocab, device="cuda"), dev(u, torch.float64))
    assert tokens.tolist() == [int(x * vocab) for x in u] and torch.allclose(logprobs, torch.full((20,), -math.log(vocab), device="cuda"), rtol=1e-6, atol=0)
    k = [1 + 5000 * i for i in range(20)]
    tokens, _ = ops.sample_rows(torch.zeros(20, vocab, device="cuda"), dev(u, torch.float64), top_k=dev(k, torch.int32))
    assert tokens.tolist() == [int(x * n) for x, n in zip(u, k)]
    tokens, _ = ops.sample_rows(torch.zeros(20, vocab, device="cuda", dtype=torch.bfloat16), dev(u, torch.float64), top_p=dev([0.25] * 20, torch.float32))
    assert tokens.tolist() == [int(x * math.ceil(0.25 * vocab)) for x in u]
    minus = torch.zeros(2, 64, device="cuda")
    minus[:, ::2] = -0.0  # equal to 0
    assert ops.sample_rows(minus, dev([0.0, 0.51], torch.float64))[0].tolist() == [0, 32]


def test_two_levels_with_many_equals(cuda):
    """A few values, thousands of tokens each: bins that have to be split down to the index."""
    rng = np.random.default_rng(2)
    x = rng.choice(np.array([0.0, -0.001, -0.002, -3.0, 1e-30], np.float32), (12, 60000))
    check(torch.tensor(x, device="cuda"), rng.random(12), top_p=[0.9, 0.5, 1.0] * 4, top_k=[0, 30000, 7] * 4)


def test_logits_that_are_not_finite(cuda):
    inf, nan = math.inf, math.nan
    x = torch.full((8, 3000), -inf, device="cuda")
    x[1] = nan
    x[2, 77] = 0.5
    x[3, 5], x[3, 9] = inf, inf
    x[4] = torch.linspace(-5, 5, 3000, device="cuda")
    x[4, ::3] = nan
    x[5, 10:20] = torch.finfo(torch.float32).min  # masked by the lowest value, beside -infinity
    x[6] = torch.finfo(torch.float32).min
    x[6, 2999] = 1.0
    x[7, 0], x[7, 1] = torch.finfo(torch.float32).max, -1.0
    # (rows 3 and 5 have 2 and 10 equal weights, so half of them is a border: sums of ones are exact, and the token is the one behind it)
    tokens, logprobs = check(x, [0.5] * 8, borders=2)
    assert tokens.tolist()[:4] == [-1, -1, 77, 9] and tokens.tolist()[5:] == [15, 2999, 0]
    assert logprobs.tolist()[:2] == [-inf, -inf] and logprobs[2] == 0
    tokens, _ = ops.sample_rows(x, dev([0.3] * 8, torch.float64), temperature=dev([0.0] * 8, torch.float32))
    assert tokens.tolist()[:4] == [-1, -1, 77, 5]
    tokens, _ = ops.sample_rows(x, dev([0.3] * 8, torch.float64), temperature=dev([inf] * 8, torch.float32))
    assert tokens.tolist()[2:4] == [77, 5] and tokens[5].item() in (12, 13)


def test_settings_at_their_ends(cuda):
    x = torch.tensor(np.random.default_rng(4).normal(0, 1, (1, 999)), device="cuda", dtype=torch.float32).repeat(9, 1)
    best, order = int(x[0].argmax()), torch.sort(x[0].double(), descending=True, stable=True).indices.tolist()
    u = [0.0, 1.0, -3.0, 7.0, math.nan, 0.999999, 0.5, 0.5, 0.5]
    tokens, logprobs = ops.sample_rows(x, dev(u, torch.float64), dev([1, 1, 1, 1, 1, 1, math.nan, 1e-8, -1], torch.float32), dev([0, 0, 0, 0, 0, 1, 0, 0, 0], torch.int32))
    assert tokens.tolist() == [best, order[-1], best, order[-1], best, best, best, best, best] and logprobs.tolist()[5:] == [0.0] * 4
    tokens, _ = ops.sample_rows(x, dev([0.999] * 9, torch.float64), top_p=dev([0, -1, 1e-9] + [1] * 6, torch.float32), min_p=dev([0, 0, 0, 1, 5, 0, 0, 0, 0], torch.float32),
                                top_k=dev([0] * 5 + [-4, 10 ** 9, 2, 3], torch.int32))
    assert tokens.tolist()[:5] == [best] * 5 and tokens.tolist()[7:] == order[1:3]


def test_rows_at_a_pitch_and_one_row_among_others(cuda):
    rng = np.random.default_rng(5)
    wide = torch.tensor(rng.normal(0, 2, (6, 1111)), device="cuda", dtype=torch.float32)
    u = rng.random(6)
    a, la = check(wide[:, 3:1003], u, [0.9] * 6)
    b, lb = ops.sample_rows(wide[:, 3:1003].contiguous(), dev(u, torch.float64), dev([0.9] * 6, torch.float32))
    assert torch.equal(a, b) and torch.equal(la, lb)
    for r in range(6):  # however many rows share a call
        t, lp = ops.sample_rows(wide[r:r + 1, 3:1003], dev(u[r:r + 1], torch.float64), dev([0.9], torch.float32))
        assert t[0] == a[r] and lp[0] == la[r]


def test_captured_and_replayed(cuda):
    x = torch.randn(4, 4000, generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    u, p = dev([0.1, 0.4, 0.7, 0.95], torch.float64), dev([0.9] * 4, torch.float32)
    tokens, logprobs = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    ops.sample_rows(x, u, top_p=p, tokens=tokens, logprobs=logprobs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_rows(x, u, top_p=p, tokens=tokens, logprobs=logprobs)
    for seed in range(3):
        x.normal_(generator=torch.Generator("cuda").manual_seed(seed)).mul_(3)
        graph.replay()
        again, lp = ops.sample_rows(x, u, top_p=p)
        assert torch.equal(again, tokens) and torch.equal(lp, logprobs)


def test_shares_follow_the_weights(cuda):
    """A grid of u over one row: each token comes up as often as its share says, to one grid step at either end."""
    x = torch.tensor([[1.0, 3.0, -1.0, 2.0, 3.0]], device="cuda")
    n = 4096
    tokens, _ = ops.sample_rows(x.repeat(n, 1), (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5) / n)
    share = torch.softmax(x[0].double(), 0).tolist()
    for t, s in enumerate(share):
        assert abs(int((tokens == t).sum()) - s * n) <= 2


def test_session_samples_on_the_device(cuda):
    """With top-k alone the device takes the tokens of the host sampler (same walk, same random numbers); temperature 0 is arg-max decoding; top-p and
    min-p runs repeat themselves."""
    from kmll_b200 import runtime as rt
    from kmll_b200.session import SamplingOptions, Session
    cfg = rt.DecoderConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, hidden_dim=512, vocab_size=640, max_seq_len=96, rope_theta=1e6, norm_eps=1e-5,
                           format=rt.FORMAT_W4G128)
    dec = rt.Decoder(cfg)
    dec.init_random(5, 0.05, False)
    s, prompt = Session(dec), np.random.default_rng(2).integers(0, 640, 9)

    def run(f):
        s.prefill(prompt)
        return [st.token_id for st in f()]

    hot = SamplingOptions(temperature=1.2, seed=11)
    assert run(lambda: s.generate_sampled_until(14, None, hot, top_k=12)) == run(lambda: s.generate_sampled_top_k_until(14, 12, None, hot))
    assert run(lambda: s.generate_sampled_until(10, None, SamplingOptions(temperature=0.0))) == run(lambda: s.generate_greedy_until(10))
    a, b = (run(lambda: s.generate_sampled_until(14, None, hot, top_p=0.8, min_p=0.01)) for _ in range(2))
    assert a == b and s.tokens()[9:] == b
    stop = a[5]
    assert run(lambda: s.generate_sampled_until(14, stop, hot, top_p=0.8, min_p=0.01)) == a[:a.index(stop) + 1]
    for bad in (dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.1), dict(top_k=-1)):
        with pytest.raises(ValueError):
            s.generate_sampled_until(1, None, hot, **bad)
    dec.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab, spread", [(300, 0.01), (20000, 0.05), (20000, 0.4), (100000, 1.0), (100000, 3.0), (100000, 12.0)])
def test_both_borders_near_and_far(cuda, dtype, vocab, spread):
    """Top-p's border and the choice in one bin, in neighbouring ones and far apart, with few and with many tokens in them; min-p on either side of
    top-p's border.  The six rows of the last u and the four of the last p below 1 have their borders where 1e-7 and 1e-6 of the weight lie behind, on
    up to 1e5 tokens: these weigh down to 1e-12 of the whole, less than the distance (1e-8) within which borders are not compared."""
    rng = np.random.default_rng(vocab + int(100 * spread))
    rows = 24
    logits = torch.tensor(rng.normal(0, spread, (rows, vocab)), device="cuda").to(dtype)
    p, u = np.tile([0.02, 0.5, 0.9, 0.999, 0.999999, 0.0], 4), np.repeat([0.0, 0.3, 0.97, 0.9999999], 6)
    check(logits, u, top_p=p, borders=10)
    check(logits, u, top_p=p, min_p=np.tile([0.9, 0.3, 0.02, 1e-4], 6), borders=10)


@pytest.mark.parametrize("rows", [1, 15, 30, 60, 140])
def test_many_launches_one_behind_the_other(cuda, rows):
    """Rows enough for clusters of every size; every launch's blocks meet before they write to each other's shared memory, however late some of them start."""
    x = torch.randn(rows, 40000, generator=torch.Generator("cuda").manual_seed(rows), device="cuda")
    best = x.argmax(1).to(torch.int32)
    u, cold = dev([0.5] * rows, torch.float64), dev([0.0] * rows, torch.float32)
    k = dev([30] * rows, torch.int32)
    first = ops.sample_rows(x, u, top_k=k)
    outs = [(ops.sample_rows(x, u, temperature=cold)[0], ops.sample_rows(x, u, top_k=k)) for _ in range(60)]
    for greedy, (tokens, logprobs) in outs:
        assert torch.equal(greedy, best) and torch.equal(tokens, first[0]) and torch.equal(logprobs, first[1])


def test_rows_too_far_apart_are_refused(cuda):
    from kmll_b200.lib import KmllError
    far = torch.empty(2 ** 32 + 256, dtype=torch.bfloat16, device="cuda").as_strided((2, 64), (2 ** 32 + 64, 1))
    with pytest.raises(KmllError, match="32 bits"):
        ops.sample_rows(far, dev([0.5, 0.5], torch.float64))
