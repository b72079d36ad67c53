"""Attention over packed sequences against its definition in 64 bits."""
import math
import random

import pytest
import torch

from encoder_util import attention_bound, attention_reference, close, starts

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def make(rows, heads, dim, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, heads, dim, generator=g, device="cuda") * scale).to(dtype)


def check(of, q, k, v, q_len, k_len, window=(-1, -1), scale=None, q_used=None, k_used=None, max_q=None, max_k=None, **more):
    qs, q_start = starts(q_len)
    ks, k_start = starts(k_len)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if "out" not in more else more.pop("out")
    dev = lambda n: None if n is None else torch.tensor(n, dtype=torch.int32, device="cuda")  # noqa: E731
    longest = lambda used, n: max([min(a, max(b, 0)) for a, b in zip(n, used)] if used else n, default=0)  # noqa: E731
    got = of.attention(q, k, v, q_start, k_start, longest(q_used, q_len) if max_q is None else max_q, longest(k_used, k_len) if max_k is None else max_k,
                       dev(q_used), dev(k_used), window=window, scale=scale, out=out, **more)
    assert got is out
    ref = attention_reference(q, k, v, qs, ks, q_used, k_used, window, scale)
    bound = attention_bound(ref, q.dtype, max(k_len, default=0))
    there = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for s, n in enumerate(q_len):
        there[qs[s] : qs[s] + (n if q_used is None else min(n, max(q_used[s], 0)))] = True
    assert (got[~there] == 7.0).all()  # rows behind a sequence's last query are left as they were
    far = (got.double() - ref[0]).abs() - bound
    assert close(got[there], ref[0][there], bound[there]), "over the bound by %g" % far[there].nan_to_num(0).max()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 24, 32, 40, 64, 72, 80, 96, 120, 128])
def test_head_sizes(native_lib, dtype, dim):
    lens = [1, 2, 130, 67]
    q, k, v = (make(200, 2, dim, dtype, n) for n in (1, 2, 3))
    check(native_lib, q, k, v, lens, lens)
    check(native_lib, q, k, v, lens, lens, (-1, 0))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (2, 1), (3, 1), (4, 2), (5, 5), (10, 2), (8, 1), (12, 3), (16, 1), (21, 3), (40, 1), (200, 1)])
def test_groups_of_heads(native_lib, Hq, Hkv):
    lens = [70, 1, 129, 33]
    q, k, v = make(233, Hq, 64, torch.float16, 1), make(233, Hkv, 64, torch.float16, 2), make(233, Hkv, 64, torch.float16, 3)
    for window in ((-1, -1), (-1, 0), (20, 5)):
        check(native_lib, q, k, v, lens, lens, window)


LENGTHS = [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 383, 384, 385, 511, 513, 640, 1000, 1666]


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (0, 0), (0, -1), (128, 128), (1, 3), (200, 0), (100, 500), (2000, 2000)])
def test_lengths_and_windows(native_lib, dim, dtype, window):
    rows = sum(LENGTHS)
    q, k, v = make(rows, 2, dim, dtype, 1), make(rows, 1, dim, dtype, 2), make(rows, 1, dim, dtype, 3)
    check(native_lib, q, k, v, LENGTHS, LENGTHS, window)


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (64, 0), (30, 40), (-1, 200), (0, 0)])
def test_more_queries_than_keys_and_fewer(native_lib, dim, dtype, window):
    # a sequence with more queries than keys has queries that see nothing under a causal mask: zeros
    pairs = [(5, 3), (3, 5), (300, 100), (100, 300), (1, 1000), (1000, 1), (7, 0), (0, 7), (0, 0), (129, 128), (128, 129), (513, 1100)]
    q_len, k_len = [p[0] for p in pairs], [p[1] for p in pairs]
    q, k, v = make(sum(q_len), 4, dim, dtype, 1), make(sum(k_len), 2, dim, dtype, 2), make(sum(k_len), 2, dim, dtype, 3)
    got = check(native_lib, q, k, v, q_len, k_len, window)
    if window == (-1, 0):
        assert (got[:2] == 0).all() and (got[8 + 0 : 8 + 200] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,Hkv,dim", [(8, 8, 64), (4, 1, 64), (8, 2, 128), (32, 8, 128), (3, 3, 80), (128, 1, 128), (40, 8, 32)])
@pytest.mark.parametrize("keys", [1, 16, 127, 129, 1000, 4097, 20011])
def test_one_token_against_many_keys(native_lib, dtype, Hq, Hkv, dim, keys):
    q, k, v = make(1, Hq, dim, dtype, 1), make(keys, Hkv, dim, dtype, 2), make(keys, Hkv, dim, dtype, 3)
    check(native_lib, q, k, v, [1], [keys], (-1, 0))
    check(native_lib, q, k, v, [1], [keys], (300, 0))


@pytest.mark.parametrize("dim,Hq,Hkv", [(64, 8, 8), (128, 8, 2)])
def test_a_step_over_a_cache_with_room(native_lib, dim, Hq, Hkv):
    room = 3000
    used = [1, 3000, 17, 128, 129, 2999, 0, -3, 5000, 1500, 64]
    S = len(used)
    dtype = torch.bfloat16
    q, k, v = make(S, Hq, dim, dtype, 1), make(S * room, Hkv, dim, dtype, 2), make(S * room, Hkv, dim, dtype, 3)
    for s, n in enumerate(used):  # what is not used yet may hold anything
        k[s * room + max(n, 0) : (s + 1) * room] = math.nan
        v[s * room + max(n, 0) : (s + 1) * room] = math.inf
    got = check(native_lib, q, k, v, [1] * S, [room] * S, (-1, 0), k_used=used)
    assert (got[6:8] == 0).all()
    # several new tokens of each
    q = make(S * 5, Hq, dim, dtype, 4)
    check(native_lib, q, k, v, [5] * S, [room] * S, (-1, 0), k_used=used)
    # tokens of which not all are there
    check(native_lib, q, k, v, [5] * S, [room] * S, (-1, 0), q_used=[5, 0, 1, 2, 3, 9, 5, 1, -1, 5, 4], k_used=used)


@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (50, 50)])
def test_padded_batches(native_lib, window):
    # a batch of equal room, sequences of different lengths; what lies behind them is no number
    room, used = 500, [500, 1, 0, 130, 257, 499]
    S = len(used)
    q, k, v = (make(S * room, 3, 64, torch.float16, n) for n in (1, 2, 3))
    for s, n in enumerate(used):
        for t in (q, k, v):
            t[s * room + n : (s + 1) * room] = math.nan
    check(native_lib, q, k, v, [room] * S, [room] * S, window, q_used=used, k_used=used)


@pytest.mark.parametrize("dim", [64, 72, 128])
def test_packed_qkv_and_other_strides(native_lib, dim):
    lens = [140, 300, 9]
    rows, H = sum(lens), 4
    for dtype in TYPES:
        qkv = make(rows, 3 * H, dim, dtype, 1)
        check(native_lib, qkv[:, :H], qkv[:, H : 2 * H], qkv[:, 2 * H :], lens, lens, (-1, 0))
        # heads outside rows, room between heads, results into rows with room between them
        t = make(3 * H, rows + 3, dim + 8, dtype, 2)
        q, k, v = (t[n * H : (n + 1) * H, :rows, :dim].transpose(0, 1) for n in range(3))
        wide = torch.full((rows, H + 1, dim + 16), 7.0, dtype=dtype, device="cuda")
        check(native_lib, q, k, v, lens, lens, (30, 30), out=wide[:, :H, 8 : 8 + dim])
        assert (wide[:, H] == 7.0).all() and (wide[:, :, :8] == 7.0).all() and (wide[:, :, 8 + dim :] == 7.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_sequences_do_not_reach_each_other(native_lib, dtype):
    # a sequence's neighbours hold no numbers: its own result is that of the sequence alone
    lens = [37, 100, 61, 128, 5]
    q, k, v = (make(sum(lens), 2, 64, dtype, n) for n in (1, 2, 3))
    clean = check(native_lib, q, k, v, lens, lens)
    for t in (k, v):
        t[37:137] = math.nan
        t[137 + 61 : 137 + 61 + 128] = -math.inf
    got = native_lib.attention(q, k, v, starts(lens)[1], starts(lens)[1], 128, 128)
    for a, b in ((0, 37), (137, 198), (326, 331)):
        assert torch.equal(got[a:b], clean[a:b])
    assert torch.isnan(got[37:137]).all()


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_keys_that_are_masked_may_hold_anything(native_lib, dim, dtype, bad):
    n = 700
    q, k, v = (make(n, 2, dim, dtype, s) for s in (1, 2, 3))
    for at in (699, 300, 129):
        k2, v2 = k.clone(), v.clone()
        k2[at], v2[at] = bad, bad
        for window in ((-1, 0), (60, 20), (0, 0), (200, 0)):
            qs, q_start = starts([n])
            clean = check(native_lib, q, k, v, [n], [n], window)
            got = native_lib.attention(q, k2, v2, q_start, q_start, n, n, window=window)
            i = torch.arange(n, device="cuda")
            sees = (at >= i - window[0]) & (at <= i + window[1]) if window[0] >= 0 else at <= i + window[1]
            ref = attention_reference(q, k2, v2, qs, qs, window=window)
            clear = attention_reference(q, k, v, qs, qs, window=window)
            assert close(got[~sees], clear[0][~sees], attention_bound(clear, dtype, n)[~sees])
            assert torch.isfinite(got[~sees]).all() and torch.isnan(ref[0][sees]).any(-1).all()
            assert torch.isnan(got[sees]).any(-1).all()
            del clean


def test_masked_infinity_against_one_token(native_lib):
    # a window over a long cache: what lies before it is no number
    q, k, v = make(1, 4, 64, torch.float16, 1), make(5000, 2, 64, torch.float16, 2), make(5000, 2, 64, torch.float16, 3)
    k[:3990], v[:3990] = math.nan, math.inf
    check(native_lib, q, k, v, [1], [5000], (1009, 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_large_scores(native_lib, dtype, dim):
    # scores that climb along the keys (the running maximum moves in every tile) and that fall; one that outweighs all
    n = 900
    q, v = make(n, 1, dim, dtype, 1, 0.1), make(n, 1, dim, dtype, 3)
    k = make(n, 1, dim, dtype, 2, 0.1)
    q[:, :, 0] = 8.0
    for slope in (1.0, -1.0):
        k[:, 0, 0] = (torch.arange(n, device="cuda") * slope * 0.05).to(dtype)
        check(native_lib, q, k, v, [n], [n], scale=1.0)
        check(native_lib, q, k, v, [n], [n], (-1, 0), scale=1.0)
        check(native_lib, q, k, v, [n], [n], (300, 0), scale=0.25)
    k[:, 0, 0] = 0
    k[555, 0, 0] = 60.0
    check(native_lib, q, k, v, [n], [n], scale=1.0)
    # the type's lowest values as keys: scores of minus tens of thousands, alone and beside others
    k[:, 0, 0] = -60000.0 if dtype == torch.float16 else -3e38
    if dtype == torch.float16:
        check(native_lib, q, k, v, [n], [n], scale=1e-2)
    else:
        # 8 * -3e38 is no fp32 number: before the scale every score is -inf, and a row of those has no softmax, as documented
        a = starts([n])[1]
        assert torch.isnan(native_lib.attention(q, k, v, a, a, n, n, scale=1e-38)).all()
        q[:, :, 0] = 1.0
        check(native_lib, q, k, v, [n], [n], scale=1e-38)
        q[:, :, 0] = 8.0
    k[700:, 0, 0] = 0
    check(native_lib, q, k, v, [n], [n], scale=1e-2 if dtype == torch.float16 else 1e-38)


def test_a_uniform_softmax_over_many_keys(native_lib):
    # all weights equal: the mean of v, whatever the number of keys
    for n in (1, 5, 128, 1000, 30001):
        q = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
        k, v = make(n, 2, 64, torch.float16, 2), make(n, 2, 64, torch.float16, 3)
        check(native_lib, q, k, v, [3], [n])


def test_many_sequences_of_one_token(native_lib):
    # more sequences than a grid's second dimension holds
    S = 70001
    q, k, v = (make(S, 1, 8, torch.float16, n) for n in (1, 2, 3))
    start = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    assert torch.equal(native_lib.attention(q, k, v, start, start, 1, 1), v)


def test_bounds_longer_than_any_sequence(native_lib):
    lens = [100, 3, 257]
    q, k, v = (make(360, 2, 64, torch.bfloat16, n) for n in (1, 2, 3))
    want = check(native_lib, q, k, v, lens, lens, (-1, 0))
    got = native_lib.attention(q, k, v, starts(lens)[1], starts(lens)[1], 5000, 9000, causal=True)
    assert close(got, want.double(), 2.0 ** -6 * want.double().abs() + 2.0 ** -8)


def test_no_sequences_no_rows(native_lib):
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = make(4, 2, 64, torch.float16, 1)
    assert native_lib.attention(x[:0], x[:0], x[:0], none, none, 0, 0).shape == (0, 2, 64)
    two = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.ones_like(x)
    native_lib.attention(x, x, x, two, two, 4, 4, out=out)  # a sequence of nothing
    assert (out == 1).all()
    four = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    native_lib.attention(x, x[:0], x[:0], four, two, 4, 0, out=out)  # queries, but no keys anywhere
    assert (out == 0).all()


@pytest.mark.parametrize("starts_bad", [[0, 50, 40, 100], [-5, 20, 60, 100], [0, 30, 60, 1000], [90, 30, 60, 100]])
def test_starts_out_of_order_stay_inside_the_tensors(native_lib, starts_bad):
    # what they mean is not defined, where they may reach is: rows of the tensors, and no others
    base = torch.full((300, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    q, k, v = (make(100, 2, 64, torch.float16, n) for n in (1, 2, 3))
    bad = torch.tensor(starts_bad, dtype=torch.int32, device="cuda")
    native_lib.attention(q, k, v, bad, bad, 100, 100, out=base[100:200])
    native_lib.encoder_wait()
    assert (base[:100] == 7).all() and (base[200:] == 7).all()


@pytest.mark.parametrize("q_len,k_len", [([1], [9000]), ([300, 20], [300, 900]), ([1] * 40, [700] * 40)])
def test_captured_and_on_two_streams_at_once(native_lib, q_len, k_len):
    args = []
    for seed in (1, 11):
        q, k, v = make(sum(q_len), 8, 64, torch.float16, seed), make(sum(k_len), 2, 64, torch.float16, seed + 1), make(sum(k_len), 2, 64, torch.float16, seed + 2)
        args.append((q, k, v, starts(q_len)[1], starts(k_len)[1], max(q_len), max(k_len)))
    want = [native_lib.attention(*a, causal=True) for a in args]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = [[native_lib.attention(*a, causal=True, stream=s) for a, s in zip(args, side)] for _ in range(20)]
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, w) for pair in got for g, w in zip(pair, want))
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want[0])
    with torch.cuda.graph(graph):
        native_lib.attention(*args[0], causal=True, out=out)
    for a, b in zip(args[0][:3], args[1][:3]):
        a.copy_(b)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want[1])
    native_lib.encoder_wait()


def test_the_workspace_is_asked_for_and_checked(native_lib):
    q, k, v = make(1, 8, 64, torch.float16, 1), make(30000, 2, 64, torch.float16, 2), make(30000, 2, 64, torch.float16, 3)
    a, b = starts([1])[1], starts([30000])[1]
    need = native_lib.attention_workspace_bytes(q, k, v, a, b, 1, 30000)
    want = native_lib.attention(q, k, v, a, b, 1, 30000)
    if need:
        with pytest.raises(native_lib.OpenfishError):
            native_lib.attention(q, k, v, a, b, 1, 30000, workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    room = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(native_lib.attention(q, k, v, a, b, 1, 30000, workspace=room[:need] if need else room), want)
    assert (room[need:] == 255).all()


def test_the_workspace_goes_by_the_queries_that_there_can_be(native_lib):
    # one sequence of at most two queries in a tensor of many rows
    q, k, v = make(100000, 8, 64, torch.float16, 1), make(30000, 2, 64, torch.float16, 2), make(30000, 2, 64, torch.float16, 3)
    at = torch.tensor([77777, 77779], dtype=torch.int32, device="cuda")
    keys = starts([30000])[1]
    assert native_lib.attention_workspace_bytes(q, k, v, at, keys, 2, 30000, causal=True) <= 64 * 2 * 8 * 65 * 4
    out = torch.full_like(q, 7.0)
    native_lib.attention(q, k, v, at, keys, 2, 30000, causal=True, out=out)
    ref = attention_reference(q[77777:77779], k, v, [0, 2], [0, 30000], window=(-1, 0))
    assert close(out[77777:77779], ref[0], attention_bound(ref, torch.float16, 30000))
    assert (out[:77777] == 7).all() and (out[77779:] == 7).all()


def test_a_cache_beyond_32_bits_of_elements(native_lib):
    # the keys of the second sequence lie 2^32 elements in
    rows = 2 ** 32 // 128 + 4000
    cache = torch.empty(2, rows, 1, 128, dtype=torch.bfloat16, device="cuda")
    lens = [2 ** 32 // 128, 4000]
    for t, seed in zip(cache, (2, 3)):
        t[: 2 ** 32 // 128].zero_()
        t[2 ** 32 // 128 :] = make(4000, 1, 128, torch.bfloat16, seed)
    q = make(2, 4, 128, torch.bfloat16, 1)
    got = native_lib.attention(q, cache[0], cache[1], starts([1, 1])[1], starts(lens)[1], 1, lens[0])
    ref = attention_reference(q[1:], cache[0][lens[0] :], cache[1][lens[0] :], [0, 1], [0, 4000])
    assert close(got[1:], ref[0], attention_bound(ref, torch.bfloat16, 4000))
    assert (got[0] == 0).all()


def test_drawn_shapes(native_lib):
    r = random.Random(7)
    for n in range(60):
        S, Hkv, dtype = r.randint(1, 6), r.randint(1, 4), r.choice(TYPES)
        Hq, dim = Hkv * r.randint(1, 6), 8 * r.randint(1, 16)
        q_len = [r.randint(0, r.choice([3, 70, 400])) for _ in range(S)]
        k_len = [r.randint(0, r.choice([3, 70, 1500])) if r.random() < 0.5 else m for m in q_len]
        window = r.choice([(-1, -1), (-1, 0), (r.randint(0, 300), r.randint(0, 300)), (r.randint(0, 300), -1)])
        q, k, v = make(sum(q_len), Hq, dim, dtype, n), make(sum(k_len), Hkv, dim, dtype, n + 1), make(sum(k_len), Hkv, dim, dtype, n + 2)
        check(native_lib, q, k, v, q_len, k_len, window, r.choice([None, 0.3]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5])
def test_single_tokens(native_lib, dtype, dim, group):
    # lengths around what a warp and a block take at a time, in a cache with room; what is not seen is no number
    lens = [0, 1, 2, 3, 4, 5, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 1000, 7]
    S, room = len(lens), 1003
    q, k, v = make(S, 3 * group, dim, dtype, 1), make(S * room, 3, dim, dtype, 2), make(S * room, 3, dim, dtype, 3)
    for s, n in enumerate(lens):
        k[s * room + n : (s + 1) * room], v[s * room + n : (s + 1) * room] = math.nan, math.inf
    for window in ((-1, 0), (0, 0), (64, -1), (100, 3)):
        got = check(native_lib, q, k, v, [1] * S, [room] * S, window, k_used=lens)
        assert (got[0] == 0).all()
    # tokens that are not there
    check(native_lib, q, k, v, [1] * S, [room] * S, k_used=lens, q_used=[n % 3 - 1 for n in range(S)], max_q=1)


@pytest.mark.parametrize("heads,dim", [(2, 64), (1, 128)])
@pytest.mark.parametrize("keys", [50, 5000])
def test_single_tokens_with_large_scores_and_no_numbers(native_lib, heads, dim, keys):
    q, k, v = make(1, heads, dim, torch.bfloat16, 1, 0.1), make(keys, 1, dim, torch.bfloat16, 2, 0.1), make(keys, 1, dim, torch.bfloat16, 3)
    q[:, :, 0] = 8.0
    for slope in (0.05, -0.05):
        k[:, 0, 0] = (torch.arange(keys, device="cuda") * slope).to(k.dtype)
        check(native_lib, q, k, v, [1], [keys], scale=1.0)
    k[:, 0, 0] = 0
    k[keys // 2, 0, 0] = 60.0
    check(native_lib, q, k, v, [1], [keys], scale=1.0)
    at = [starts([1])[1], starts([keys])[1], 1, keys]
    for n in (0, keys // 3, keys - 1):
        # a score of no number, and of infinity: no result; of minus infinity: no part
        for bad in (math.nan, math.inf):
            k2 = k.clone()
            k2[n, 0, 0] = bad
            assert torch.isnan(native_lib.attention(q, k2, v, *at)).all()
        k2, v2 = k.clone(), v.clone()
        k2[n, 0, 0], v2[n] = -math.inf, 0
        keep = [j for j in range(keys) if j != n]
        ref = attention_reference(q, k[keep], v[keep], [0, 1], [0, keys - 1])
        assert close(native_lib.attention(q, k2, v2, *at), ref[0], attention_bound(ref, torch.bfloat16, keys))
    k[:, 0, 0] = -math.inf
    assert torch.isnan(native_lib.attention(q, k, v, *at)).all()


@pytest.mark.parametrize("S,keys", [(1, 9000), (40, 700), (300, 130)])
def test_single_tokens_captured_strided_and_on_two_streams(native_lib, S, keys):
    # heads of a packed tensor of queries, keys and values; results into rows with room between them
    args, outs = [], []
    for seed in (1, 11):
        new, cache = make(S, 12, 64, torch.float16, seed), make(S * keys, 12, 64, torch.float16, seed + 1)
        args.append((new[:, :4], cache[:, 4:8], cache[:, 8:], starts([1] * S)[1], starts([keys] * S)[1], 1, keys))
    want = [native_lib.attention(*a, causal=True) for a in args]
    for a, w in zip(args, want):
        wide = torch.full((S, 5, 72), 7.0, dtype=torch.float16, device="cuda")
        assert torch.equal(native_lib.attention(*a, causal=True, out=wide[:, :4, 8:]), w)
        assert (wide[:, 4] == 7).all() and (wide[:, :, :8] == 7).all()
        ref = attention_reference(*a[:3], list(range(S + 1)), [keys * s for s in range(S + 1)], window=(-1, 0))
        assert close(w, ref[0], attention_bound(ref, torch.float16, keys))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = [[native_lib.attention(*a, causal=True, stream=s) for a, s in zip(args, side)] for _ in range(20)]
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, w) for pair in got for g, w in zip(pair, want))
    # a step captured twice in a row: the second one's kernels follow the first one's join
    graph, out, again = torch.cuda.CUDAGraph(), torch.empty_like(want[0]), torch.empty_like(want[0])
    with torch.cuda.graph(graph):
        native_lib.attention(*args[0], causal=True, out=out)
        native_lib.attention(out, *args[0][1:], causal=True, out=again)
    for a, b in zip(args[0][:3], args[1][:3]):
        a.copy_(b)
    second = native_lib.attention(want[1], *args[1][1:], causal=True)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want[1]) and torch.equal(again, second)


def test_single_tokens_beyond_32_bits_of_elements(native_lib):
    first = 2 ** 32 // 128
    cache = torch.empty(2, first + 4000, 1, 128, dtype=torch.bfloat16, device="cuda")
    for t, seed in zip(cache, (2, 3)):
        t[:first].zero_()
        t[first:] = make(4000, 1, 128, torch.bfloat16, seed)
    q = make(2, 1, 128, torch.bfloat16, 1)
    got = native_lib.attention(q, cache[0], cache[1], starts([1, 1])[1], starts([first, 4000])[1], 1, first)
    ref = attention_reference(q[1:], cache[0][first:], cache[1][first:], [0, 1], [0, 4000])
    assert close(got[1:], ref[0], attention_bound(ref, torch.bfloat16, 4000))
    assert (got[0] == 0).all()
    # one sequence all of that long, seen from its end
    got = native_lib.attention(q[1:], cache[0], cache[1], starts([1])[1], starts([first + 4000])[1], 1, first + 4000, window=(3999, 0))
    assert close(got, ref[0], attention_bound(ref, torch.bfloat16, 4000))
