"""Attention over long key sequences in fp16, with bounds well below the results: weights below the type's smallest numbers, results
at its largest, a piece of the keys left out; and rows whose values must not show in other rows' roundings.

The bounds, from the definition (u = 2^-11, half a step of fp16; P|v| = sum p|v| over the keys a query sees):
  u |out|                        the result's own rounding
  u P|v|                         by tiles: a weight is rounded to 16 bits on its way into the matrix product
  2^-18 (1 + |z|) P|v|           a score's fp32 sum (up to 128 terms), the exponential's argument and value
  keys 2^-25 P|v|                sums over keys in fp32: by tiles keys / 16 additions into the accumulator, truncated at worst (2^-23 each), and keys / 64
                                 into the weights' sum; by lanes keys / 8 of 2^-24 into each of the two, and a scaling every fourth
  keys 2^-30 max|v|              by tiles: underflow.  A row's largest weight is held as 2^5 or more, half the smallest subnormal is 2^-25"""
import math

import pytest
import torch

from encoder_util import attention_reference, close, starts

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


def make(rows, heads, dim, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, heads, dim, generator=g, device="cuda").half()


def bound_of(ref, keys, lanes):
    out, weight, zmax, vmax = ref
    b = U * out.abs() + (2.0 ** -18 * (1 + zmax) + keys * 2.0 ** -25) * weight + 2.0 ** -25
    return b if lanes else b + U * weight * (1 + 2 * U) + keys * 2.0 ** -30 * vmax


def by_lanes(Hq, Hkv, dim, queries):
    return queries == 1 and (Hq == Hkv or (Hq == 2 * Hkv and dim <= 64))


def by_lanes(Hq, Hkv, dim, queries):
    return queries == 1 and (Hq == Hkv or (Hq == 2 * Hkv and dim <= 64))


@pytest.mark.parametrize("Hq,Hkv,dim", [(8, 8, 64), (8, 4, 32), (3, 3, 80), (2, 2, 128), (4, 1, 64), (8, 2, 128), (6, 2, 80), (40, 8, 32)])
@pytest.mark.parametrize("queries", [1, 3, 200])
@pytest.mark.parametrize("keys", [1666, 4097, 9000, 30001])
def test_many_keys_within_bounds_that_reject_a_missing_piece(native_lib, Hq, Hkv, dim, queries, keys):
    q, k, v = make(queries, Hq, dim, 1), make(keys, Hkv, dim, 2), make(keys, Hkv, dim, 3)
    ref = attention_reference(q, k, v, [0, queries], [0, keys])
    bound = bound_of(ref, keys, by_lanes(Hq, Hkv, dim, queries))
    # zeros would not do, nor a result without a 64th of the keys (a split, or a tile of the shorter ones)
    assert not close(torch.zeros_like(q), ref[0], bound)
    assert (bound < 0.25 * ref[0].abs().amax(dim=(0, 2), keepdim=True)).all()
    kept = torch.ones(keys, dtype=torch.bool, device="cuda")
    kept[keys // 2 : keys // 2 + keys // 64] = False
    some = attention_reference(q, k[kept], v[kept], [0, queries], [0, int(kept.sum())])
    assert not close(some[0].half(), ref[0], bound)
    got = native_lib.attention(q, k, v, starts([queries])[1], starts([keys])[1], queries, keys)
    assert close(got, ref[0], bound), "over the bound by %g" % ((got.double() - ref[0]).abs() - bound).max()


@pytest.mark.parametrize("Hq", [2, 8])
@pytest.mark.parametrize("keys", [1000, 30001])
def test_the_mean_of_many_values(native_lib, Hq, keys):
    # scores of zero: weights that every type holds, so nothing is rounded but sums and the result
    q = torch.zeros(3, Hq, 64, dtype=torch.float16, device="cuda")
    k, v = make(keys, 2, 64, 2), make(keys, 2, 64, 3)
    out, weight, zmax, vmax = attention_reference(q, k, v, [0, 3], [0, keys])
    bound = U * out.abs() + keys * 2.0 ** -25 * weight + 2.0 ** -25
    assert not close(torch.zeros_like(q), out, bound)
    got = native_lib.attention(q, k, v, starts([3])[1], starts([keys])[1], 3, keys)
    assert close(got, out, bound)


@pytest.mark.parametrize("dim", [64, 128])
def test_weights_below_the_smallest_numbers_of_the_type(native_lib, dim):
    # One key outweighs each of the others by 2^24.9, but not all of them together by much.  So many queries that no block's keys
    # are split (a piece without the first key would have a scale of its own).
    queries, heads, keys = 10000, 8, 131072
    q = torch.zeros(queries, heads, dim, dtype=torch.float16, device="cuda")
    q[:, :, :2] = 1.0
    k, v = torch.zeros(keys, 1, dim, dtype=torch.float16, device="cuda"), make(keys, 1, dim, 3).abs()
    k[1:, 0, 0], k[1:, 0, 1] = -24.875, -0.025
    v[0] = 0
    at = starts([queries])[1], starts([keys])[1], queries, keys
    assert native_lib.attention_workspace_bytes(q, k, v, *at, scale=math.log(2)) == 0
    got = native_lib.attention(q, k, v, *at, scale=math.log(2))
    ref = attention_reference(q[:1], k, v, [0, 1], [0, keys], scale=math.log(2))
    bound = bound_of(ref, keys, False)
    assert (bound < 0.25 * ref[0]).all()
    assert (got == got[:1, :1]).all()  # the same query all along
    assert close(got[:1], ref[0], bound), "%g for %g" % (got[0, 0, 0], ref[0][0, 0, 0])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("queries,keys,window", [(5, 1000, (-1, -1)), (300, 640, (-1, -1)), (1000, 1000, (255, 0)), (300, 20000, (-1, -1))])
@pytest.mark.parametrize("sign", [1, -1])
def test_results_at_the_largest_number_of_the_type(native_lib, dim, queries, keys, window, sign):
    # All values are the largest, so every result is; most weights (2^-3.99648 of the largest) lie just above the middle of two 16-bit
    # numbers, so that they are all rounded up and the rounded ones add up to a result half a step above.
    q = torch.zeros(queries, 4, dim, dtype=torch.float16, device="cuda")
    q[:, :, :2] = 1.0
    k = torch.zeros(keys, 2, dim, dtype=torch.float16, device="cuda")
    k[:, :, 0], k[:, :, 1] = -4.0, 0.00352
    k[::64] = 0
    v = torch.full_like(k, sign * 65504.0)
    got = native_lib.attention(q, k, v, starts([queries])[1], starts([keys])[1], queries, keys, window=window, scale=math.log(2))
    assert (got == sign * 65504.0).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_behind_the_queries_have_no_part(native_lib, dim, group, dtype):
    # what lies behind a sequence's last query (room that is not used yet) changes not a bit of the results before it
    room, used, keys = 160, [100, 33, 1, 130], 1000
    S, H = len(used), 2
    q, k, v = make(S * room, H * group, dim, 1).to(dtype), make(S * keys, H, dim, 2).to(dtype), make(S * keys, H, dim, 3).to(dtype)
    lens = torch.tensor(used, dtype=torch.int32, device="cuda")
    there = torch.cat([torch.arange(room, device="cuda") < n for n in used])
    results = []
    for behind in (0.0, math.nan, math.inf, 300.0, None):
        x = q.clone()
        if behind is not None:
            x[~there] = behind
        else:
            x[~there] *= 40
        results.append(native_lib.attention(x, k, v, starts([room] * S)[1], starts([keys] * S)[1], room, keys, q_used=lens)[there])
    for r in results[1:]:
        assert torch.equal(r, results[0])
