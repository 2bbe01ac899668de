"""Requests of unequal length, without a GPU: refusals, the rules of the oracle, the layouts."""
import ctypes as C

import numpy as np
import pytest

import paged_oracle as po
from kmll_b200 import lib


@pytest.fixture(scope="module")
def handle():
    return lib.load()


def plan_args(**over):
    a = dict(stream=None, lengths=16, new_tokens=16, requests=2, block=16, block_table=16, table_width=4, free_blocks=16, free_capacity=8, free_count=16, token_capacity=8,
             context=16, query_start=16, positions=16, slots=16, free_count_out=16, status=16)
    assert set(over) <= set(a)
    return list((a | over).values())


@pytest.mark.parametrize("over, code, word", [
    (dict(requests=-1), -2, b"negative"), (dict(requests=8193), -5, b"8193"), (dict(block=24), -2, b"24"), (dict(block=256), -2, b"256"),
    (dict(table_width=1 << 28, block=16), -2, b"32 bits"), (dict(lengths=None), -1, b"lengths"), (dict(new_tokens=None), -1, b"new_tokens"),
    (dict(free_count=None), -1, b"free_count"), (dict(free_blocks=None), -1, b"free_blocks"), (dict(block_table=None), -1, b"block_table"),
    (dict(slots=None), -1, b"slots"), (dict(positions=None), -1, b"positions"), (dict(status=None), -1, b"status"), (dict(context=None), -1, b"context"),
    (dict(query_start=None), -1, b"query_start"), (dict(free_count_out=None), -1, b"free_count_out"), (dict(token_capacity=-1), -2, b"negative")])
def test_plan_refusals(handle, over, code, word):
    assert handle.kmll_paged_plan(*plan_args(**over)) == code and word in handle.kmll_last_error()


def test_release_refusals(handle):
    good = [None, 16, 16, 2, 16, 16, 4, 16, 8, 16, 16, 16, 16]
    for at, value, code in ((1, None, -1), (2, None, -1), (3, -1, -2), (3, 9000, -5), (4, 48, -2), (5, None, -1), (7, None, -1), (9, None, -1), (10, None, -1), (12, None, -1)):
        bad = list(good)
        bad[at] = value
        assert handle.kmll_paged_release(*bad) == code, at


def prepare_args(**over):
    a = dict(stream=None, query=16, ld_query=256, key=16, ld_key=128, value=16, ld_value=128, is_f32=1, freqs=16, n_freqs=32, positions=16, slots=16, tokens=3, heads=4,
             kv_heads=2, head_dim=64, query_rot=32, k_codes=16, k_scales=16, v_codes=16, v_scales=16, pages=4, block=16)
    assert set(over) <= set(a)
    return list((a | over).values())


@pytest.mark.parametrize("over, code, word", [
    (dict(tokens=-1), -2, b"negative"), (dict(block=8), -2, b"8"), (dict(head_dim=72), -2, b"72"), (dict(head_dim=272), -2, b"272"), (dict(pages=0), -2, b"pages"),
    (dict(pages=1 << 28), -2, b"32 bits"), (dict(n_freqs=33), -2, b"33"), (dict(ld_query=255), -2, b"overlap"), (dict(ld_key=64), -2, b"overlap"),
    (dict(ld_value=64), -2, b"overlap"), (dict(k_codes=None), -1, b"cache"), (dict(v_scales=None), -1, b"cache"), (dict(k_codes=24), -2, b"aligned"),
    (dict(key=None), -1, b"key"), (dict(query=None), -1, b"query"), (dict(slots=None), -1, b"slots"), (dict(positions=None), -1, b"positions"),
    (dict(freqs=None), -1, b"freqs"), (dict(query_rot=None), -1, b"query_rot"), (dict(query=32, ld_query=300), -2, b"in place"), (dict(kv_heads=0), -2, b"kv heads")])
def test_prepare_refusals(handle, over, code, word):
    assert handle.kmll_prepare_paged_attention(*prepare_args(**over)) == code and word in handle.kmll_last_error()


def attention_args(**over):
    a = dict(stream=None, query=16, is_f32=1, query_start=16, context=16, block_table=16, table_width=4, requests=2, tokens=2, max_query=1, max_context=64, heads=4, k_codes=16,
             k_scales=16, v_codes=16, v_scales=16, pages=8, block=16, kv_heads=2, head_dim=64, scale=0.125, window=0, workspace=16, out=16)
    assert set(over) <= set(a)
    return list((a | over).values())


@pytest.mark.parametrize("over, code, word", [
    (dict(heads=5), -2, b"5 query heads"), (dict(heads=0), -2, b"0 query heads"), (dict(scale=0.0), -2, b"scale"), (dict(scale=-1.0), -2, b"scale"),
    (dict(scale=float("nan")), -2, b"scale"), (dict(scale=float("inf")), -2, b"scale"), (dict(window=-1), -2, b"window"), (dict(requests=-1), -2, b"negative"),
    (dict(max_context=-1), -2, b"negative"), (dict(table_width=1 << 28), -2, b"32 bits"), (dict(query=None), -1, b"query"), (dict(out=None), -1, b"out"),
    (dict(context=None), -1, b"context"), (dict(block_table=None), -1, b"block_table"), (dict(query_start=None), -1, b"query_start"), (dict(v_codes=None), -1, b"cache"),
    (dict(head_dim=100), -2, b"100")])
def test_attention_refusals(handle, over, code, word):
    assert handle.kmll_paged_attention(*attention_args(**over)) == code and word in handle.kmll_last_error()


def test_attention_calls_that_do_not_fit_are_refused_before_any_launch(handle):
    capacity = handle.kmll_paged_attention(*attention_args(requests=40000, heads=4, kv_heads=2))
    assert capacity < -2 and b"40000 requests" in handle.kmll_last_error()
    assert handle.kmll_paged_attention(*attention_args(tokens=1 << 24, max_query=1 << 24, heads=4, kv_heads=2)) == capacity and b"tokens" in handle.kmll_last_error()
    # positions: a tile's end behind the last one still fits into 32 bits
    assert handle.kmll_paged_attention(*attention_args(table_width=(1 << 31) // 16 - 1)) == -2 and b"32 bits" in handle.kmll_last_error()


@pytest.mark.parametrize("at, value, code", [(1, None, -1), (3, 31, -2), (4, -1, -2), (5, 0, -2), (5, (1 << 19) + 1, -2), (6, None, -1), (11, None, -1)])
def test_sample_refusals(handle, at, value, code):
    args = [None, 16, 1, (1 << 20) if at != 3 else 32, 2, 32, 16, None, None, None, None, 16, None]
    args[at] = value
    assert handle.kmll_sample_rows(*args) == code


def test_nothing_to_do_is_no_error(handle):
    assert handle.kmll_prepare_paged_attention(*prepare_args(tokens=0, key=None, query=None, slots=None)) == 0
    assert handle.kmll_paged_attention(*attention_args(requests=0, query=None)) == 0
    assert handle.kmll_paged_attention(*attention_args(tokens=0, out=None)) == 0
    assert handle.kmll_paged_cache_rows(None, 16, 16, 16, 16, 4, 16, 2, 64, None, 0, None, None) == 0
    assert handle.kmll_sample_rows(None, None, 1, 32, 0, 32, None, None, None, None, None, None, None) == 0


def test_python_refusals_need_no_gpu():
    import torch

    from kmll_b200 import ops
    for bad in (dict(block=8), dict(head_dim=40), dict(pages=0), dict(kv_heads=0), dict(head_dim=512)):
        with pytest.raises(lib.KmllError):
            ops.DevicePagedI8Cache.create(**(dict(pages=2, block=16, kv_heads=1, head_dim=64, device="cpu") | bad))
    c = ops.DevicePagedI8Cache.create(2, 16, 1, 64, device="cpu")
    assert c.nbytes == 2 * 2 * 16 * 64 + 2 * 2 * 4
    with pytest.raises(lib.KmllError):
        ops.DevicePagedI8Cache.from_parts(c.k_codes, c.v_codes[:, :, :, :32], c.k_scales, c.v_scales)
    with pytest.raises(lib.KmllError):
        ops.DevicePagedI8Cache.from_parts(c.k_codes, c.v_codes, c.k_scales.double(), c.v_scales)
    with pytest.raises(lib.KmllError):  # no CPU path
        ops.paged_cache_rows(c, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(lib.KmllError):
        ops.sample_rows(torch.zeros(2, 8), torch.zeros(2, dtype=torch.float64))
    with pytest.raises(lib.KmllError):
        ops.sample_rows(torch.zeros(2, 8, dtype=torch.float16), torch.zeros(2, dtype=torch.float64))


def test_store_keeps_every_value_within_its_bound():
    """A value that was coded once is within half a step, one that was coded again g times within (g + 1) / 2 steps of the last scale."""
    rng = np.random.default_rng(0)
    s = po.Store(1, 16, 1, 32)
    x = rng.normal(0, 1, (16, 1, 32)) * np.linspace(0.5, 3, 16)[:, None, None]
    for t in range(16):
        s.append(x[t:t + 1], [t])
    got = s.codes[0] * s.scales[0].astype(np.float64)[:, None]
    assert np.abs(got - x).max() <= s.scales[0, 0] * (16 + 1) / 2
    assert abs(float(s.scales[0, 0]) - np.abs(x).max() / 127) <= np.abs(x).max() / 127 * 2 ** -24
    one = po.Store(1, 16, 1, 32)
    one.append(x, list(range(16)))
    assert np.abs(one.codes[0] * float(one.scales[0, 0]) - x).max() <= float(one.scales[0, 0]) * (0.5 + 1e-5)


def test_layouts_hold_every_code_once():
    codes = np.arange(2 * 32 * 2 * 48).reshape(2, 32, 2, 48) % 251 - 125
    k, v = po.key_layout(codes), po.value_layout(codes)
    assert k.shape == (2, 2, 3, 32, 16) and v.shape == (2, 2, 2, 48, 16)
    assert k[1, 1, 2, 31, 5] == codes[1, 31, 1, 37] and v[1, 0, 1, 47, 3] == codes[1, 19, 0, 47]


def test_oracle_sampler_agrees_with_the_host_sampler():
    """The host sampler of the session walks the k best logits best first, as the operator does."""
    from kmll_b200.session import SamplingOptions, sample_from_top_logits

    class Fixed:
        def __init__(self, u):
            self.u = u

        def next_unit_f64(self):
            return self.u

    rng = np.random.default_rng(3)
    logits = rng.normal(0, 2, 500).astype(np.float32)
    order = np.argsort(-logits, kind="stable")[:20]
    for u in np.linspace(0.01, 0.99, 41):
        token, _, gap = po.sample(logits.astype(np.float64), u, 0.75, 20)
        if gap > 1e-5:  # (the host's weights are f32)
            assert sample_from_top_logits([(int(i), float(logits[i])) for i in order], SamplingOptions(temperature=0.75), Fixed(float(u)))[0] == token


def test_pointer_types_of_the_new_entry_points():
    protos = lib.parse_prototypes(lib.HEADERS[0])
    assert len(protos["kmll_paged_attention"][1]) == 24 and protos["kmll_paged_attention_workspace_bytes"][0] is C.c_size_t
    assert len(protos["kmll_prepare_paged_attention"][1]) == 23 and len(protos["kmll_paged_plan"][1]) == 17 and len(protos["kmll_sample_rows"][1]) == 13


def test_pitches_beyond_32_bits_are_refused():
    """A pitch of 2^32 + 64 must not become one of 64 (tensors without memory: only their strides are looked at)."""
    import torch

    from kmll_b200 import ops
    rows = torch.empty_strided((3, 1, 64), (2 ** 32 + 64, 64, 1), dtype=torch.bfloat16, device="meta")
    with pytest.raises(lib.KmllError, match="32 bits"):
        ops._head_rows(rows, 3, 1, 64, torch.bfloat16, "key", rows.get_device())
    assert ops._head_rows(rows[:1], 1, 1, 64, torch.bfloat16, "key", rows.get_device())[1] == 64  # (one row has no pitch)
    near = torch.empty_strided((2, 64), (2 ** 31 - 1, 1), dtype=torch.float32, device="meta")
    assert ops._row_pitch(near, "logits") == 2 ** 31 - 1
