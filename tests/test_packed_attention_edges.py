"""Packed attention (include/cmhsa_packed.h) where single keys decide: infinite scores, marked keys at every boundary of tiles, chunks
and pages' worth of keys, weights that round the same way.  Against the float64 oracle, in every kind of launch."""
import numpy as np
import pytest
import torch

import cmhsa
from oracle import serving
from test_packed_attention import TYPES, make, offsets, op

EMPTY = [0] * 65                                                 # more sequences than a wave has lanes: tiles of 128 rows
CODES = {"float32": 0, "bfloat16": 1, "float16": 2}


def cut_workspace(cu_q, cu_k, heads, kv_heads, d, dtype):
    return cmhsa.load_library().cmhsa_packed_workspace_bytes(len(cu_q) - 1, int(cu_q[-1]), int(cu_k[-1]), heads, kv_heads, d, CODES[dtype])


def run(dev, tensors, cu_q, cu_k, heads, kv_heads):
    a, b = (torch.from_numpy(c).to(dev) for c in (cu_q, cu_k))
    return op()(*(t.to(dev) for t in tensors), a, b, heads, kv_heads).double().cpu().numpy()


# ---------------------------------------------------------------------------------------------------------- scores of -inf

# (queries, keys) of the sequences; the launches are told apart by their sizes
KINDS = {"short": ([12, 9], [12, 9]), "waves": ([70, 150], [70, 150]), "tiles": ([70, 150] + EMPTY, [70, 150] + EMPTY), "cut": ([5, 3], [1700, 1500])}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("infinity", [-np.inf, np.inf])
@pytest.mark.parametrize("kind,at", [(k, at) for k in ("short", "waves", "tiles") for at in (0, 1, 2, 3, 6)] + [("cut", at) for at in (0, 3, 128, 130, 1280, 1691)])
def test_one_infinite_element_of_k_is_a_weight_of_zero(gpu_device, dtype, heads, kv_heads, d, infinity, kind, at):
    """One element of K is infinite, and the queries' elements there have the sign that makes the score -inf: that key takes no
    part, rows that see others are finite, and a row that sees nothing else is 0 / 0.  An infinite value at the first sequence's
    last key sends the 16-bit types through the loop for what is not finite as well."""
    rng = np.random.default_rng(at + d)
    new, total = KINDS[kind]
    cu_q, cu_k = offsets(new), offsets(total)
    assert (cut_workspace(cu_q, cu_k, heads, kv_heads, d, dtype) > 0) == (kind == "cut")
    tensors = make(rng, dtype, cu_q[-1], cu_k[-1], heads, kv_heads, d)
    for h in range(heads):
        tensors[0][:, h * d + 7] = -np.sign(infinity) * (tensors[0][:, h * d + 7].abs() + 0.25)
    tensors[1][at, 7] = 0
    tensors[2][total[0] - 1, 5] = np.inf
    q, k, v = (t.double().numpy() for t in tensors)
    reach = serving.packed_attention_f64(q, k, v, cu_q, cu_k, heads, kv_heads)[2]          # of the finite scores
    tensors[1][at, 7] = infinity
    k[at, 7] = infinity
    with np.errstate(invalid="ignore"):
        o, spread, _, weight = serving.packed_attention_f64(q, k, v, cu_q, cu_k, heads, kv_heads)
    got = run(gpu_device, tensors, cu_q, cu_k, heads, kv_heads)
    group, first = heads // kv_heads, total[0] - new[0]
    hidden = np.zeros(o.shape, dtype=bool)                       # rows that see the infinite key and no other
    if at == 0 and first == 0:
        hidden[0, :group * d] = True
    assert np.array_equal(np.isnan(o), hidden) and np.array_equal(np.isnan(got), hidden)
    fine = np.isfinite(o)
    assert (~fine & ~hidden).sum() == group and np.array_equal(got[~fine & ~hidden], o[~fine & ~hidden])
    tol = serving.tolerance(dtype, (o, spread, reach, weight), max(total), d)
    worst = np.abs(got[fine] - o[fine]) / tol[fine]
    assert worst.max() <= 1.0, worst.max()


# ------------------------------------------------------------------------------------------------- weights of 16-bit types

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("kind,n", [("short", 31), ("waves", 900), ("tiles", 900), ("cut", 4000)])
def test_equal_weights_that_round_the_same_way(gpu_device, dtype, kind, n):
    """One key above n - 1 equal ones, whose weight lies just over half a step of the type above a representable one: rounded alike, all of them are off
    the same way.  The last row's V is constant, and the quotient gives it back: numerator and denominator hold the same
    weights, so only the fp32 sums (two steps a pair and add, 2^-22, over n / 2 in a row at most) and the output's rounding are left."""
    h = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]
    d = 64
    new, total = ([3], [n]) if kind == "cut" else ([n], [n])
    if kind == "tiles":
        new, total = new + EMPTY, total + EMPTY
    cu_q, cu_k = offsets(new), offsets(total)
    assert (cut_workspace(cu_q, cu_k, 1, 1, d, dtype) > 0) == (kind == "cut")
    # q = 8 (e_0 + .. + e_3), so that a score is the sum of four elements of K: 0 for the first key, ln(0.5 + 0.51 h) for the others, cut up over
    # the four, since one of them would not hold it exactly enough
    want = np.log(0.5 * (1 + 1.02 * h))
    q, k, v = (torch.zeros((rows, d)) for rows in (int(cu_q[-1]), n, n))
    q[:, :4] = 8
    rest = want
    for i in range(4):
        part = torch.tensor(rest).to(TYPES[dtype])
        k[1:, i] = part.float()
        rest -= float(part)
    assert abs(rest) < 1e-7
    v[:] = 1.0 + 12 * 2 ** -7                                     # exact in both types
    tensors = [t.to(TYPES[dtype]) for t in (q, k, v)]
    got = run(gpu_device, tensors, cu_q, cu_k, 1, 1)
    assert np.array_equal(got, np.full(got.shape, v[0, 0].item()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("kind,n", [("short", 31), ("waves", 700), ("tiles", 700), ("cut", 4000)])
def test_a_long_tail_below_one_large_weight(gpu_device, dtype, kind, n):
    """The first key has weight 1 and a value of 0, every other one a weight between 2^-29 and 2^-26 and a value of about 1000: what comes
    out is the tail alone.  fp16 numbers end at 2^-24.  Bound: as in serving.tolerance, but a weight is off by half a step of
    fp16 (2h, with the sum) or by 2^-33 of the largest weight, which is 1, whichever is more."""
    rng = np.random.default_rng(n)
    d, u, h = 64, 2.0 ** -24, {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]
    new, total = ([3], [n]) if kind == "cut" else ([n], [n])
    if kind == "tiles":
        new, total = new + EMPTY, total + EMPTY
    cu_q, cu_k = offsets(new), offsets(total)
    assert (cut_workspace(cu_q, cu_k, 1, 1, d, dtype) > 0) == (kind == "cut")
    q, k, v = (torch.zeros((rows, d)) for rows in (int(cu_q[-1]), n, n))
    q[:, 0] = 8
    k[1:, 0] = torch.from_numpy(rng.uniform(-29, -26, n - 1) * np.log(2)).float()
    v[1:] = torch.from_numpy(rng.uniform(800, 1200, (n - 1, d))).float()
    tensors = [t.to(TYPES[dtype]) for t in (q, k, v)]
    o, spread, reach, weight = serving.packed_attention_f64(*(t.double().numpy() for t in tensors), cu_q, cu_k, 1, 1)
    off = 2 * (d + 16) * u * reach + (160 + 2 * (n + 16)) * u + (0 if dtype == "float32" else 2 * h)
    tol = off * spread + h * np.abs(o) + (2.0 ** -25 + 2.0 ** -33 * (weight + n * np.abs(o)) if dtype == "float16" else 1e-37)
    assert (o[-1] > 3 * tol[-1]).all()                           # an answer without the tail is out of bounds
    worst = np.abs(run(gpu_device, tensors, cu_q, cu_k, 1, 1) - o) / tol
    assert worst.max() <= 1.0, worst.max()


# ------------------------------------------------------------------------------------------------------------ cut launches

@pytest.mark.gpu
@pytest.mark.parametrize("new,total", [([1], [1700]), ([3, 1], [1600, 5001]), ([300], [4096])], ids=str)
def test_the_join_is_handed_the_chunk_length(gpu_device, new, total):
    """It lies behind the states in the workspace: blocks times keys over the chunks aimed at (1024 of heads of 64), rounded up to 128."""
    cu_q, cu_k = offsets(new), offsets(total)
    heads, d = 2, 64
    need = cut_workspace(cu_q, cu_k, heads, heads, d, "bfloat16")
    tensors = [t.to(gpu_device) for t in make(np.random.default_rng(1), "bfloat16", cu_q[-1], cu_k[-1], heads, heads, d)]
    space = torch.full((need,), 85, dtype=torch.uint8, device=gpu_device)
    a, b = (torch.from_numpy(c).to(gpu_device) for c in (cu_q, cu_k))
    got = cmhsa.attention_packed_fwd(*tensors, a, b, heads, heads, workspace=space)
    each = sum(-(-n // 128) * t for n, t in zip(new, total)) / 512
    assert space[need - 16:].view(torch.int32)[0].item() == int(each * 1.0001 + 128) // 128 * 128
    assert torch.equal(got, op()(*tensors, a, b, heads, heads))


# ------------------------------------------------------------------------------------------------------ every key, once

EVERY = {"short": [([20, 32, 7], [20, 32, 7])], "waves": [([230, 300], [230, 300]), ([9], [600]), ([65], [129])],
         "tiles": [([230, 300] + EMPTY, [230, 300] + EMPTY), ([3, 1, 2] + EMPTY, [1000, 64, 65] + EMPTY), ([250] * 30, [257] * 30)],
         "cut": [([1], [1700]), ([3, 1], [1600, 5001]), ([1, 2, 1, 1, 1], [31, 1, 9000, 256, 1153])]}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 4, 64), (4, 4, 128)])
@pytest.mark.parametrize("kind,new,total", [(kind, *case) for kind in EVERY for case in EVERY[kind]], ids=str)
def test_every_key_counts_once(gpu_device, dtype, heads, kv_heads, d, kind, new, total):
    """q = 0: all weights are one number.  Each column of V holds 256 at one key and 0 elsewhere, a call after the other until every key has been
    marked: a row's output is 256 over the keys that it sees, exactly but for the quotient's and the output's roundings (3 u and
    h), or 0.  A key that is lost or taken twice changes one column by all of it."""
    cu_q, cu_k = offsets(new), offsets(total)
    assert (cut_workspace(cu_q, cu_k, heads, kv_heads, d, dtype) > 0) == (kind == "cut")
    off = 3 * 2.0 ** -24 + {"float32": 0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]
    columns, longest = kv_heads * d, max(total)
    a, b = (torch.from_numpy(c).to(gpu_device) for c in (cu_q, cu_k))
    q = torch.zeros((cu_q[-1], heads * d), dtype=TYPES[dtype], device=gpu_device)
    k = torch.randn((cu_k[-1], columns), device=gpu_device).to(TYPES[dtype])
    place = torch.cat([torch.arange(t) for t in total]).to(gpu_device)[:, None]            # of a key in its sequence
    last = torch.cat([torch.arange(t - n, t) for n, t in zip(new, total)]).to(gpu_device)[:, None]     # key that a row sees
    for at in range(0, longest, columns):
        mark = at + torch.arange(columns, device=gpu_device)[None]
        got = op()(q, k, (place == mark).to(TYPES[dtype]) * 256, a, b, heads, kv_heads).double()
        mark = mark.view(kv_heads, 1, d).expand(kv_heads, heads // kv_heads, d).reshape(1, -1)
        want = torch.where(mark <= last, 256 / (last + 1).double(), 0.0)
        assert ((got - want).abs() <= off * want).all(), at


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind,new,total", [(kind, *case) for kind in EVERY for case in EVERY[kind]], ids=str)
def test_one_key_with_all_of_the_weight(gpu_device, dtype, d, kind, new, total):
    """Each of four K/V heads has one key with a score of 64 where the others have 0, at every boundary of 32 keys in turn: rows that see it
    return its value (the others weigh exp(-64) each: 2^-92), rows before it the mean of theirs."""
    rng = np.random.default_rng(d)
    heads = 4
    cu_q, cu_k = offsets(new), offsets(total)
    assert (cut_workspace(cu_q, cu_k, heads, heads, d, dtype) > 0) == (kind == "cut")
    u, h = 2.0 ** -24, {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]
    a, b = (torch.from_numpy(c).to(gpu_device) for c in (cu_q, cu_k))
    s = int(np.argmax(total))                                    # the longest sequence
    n, t = new[s], total[s]
    rows = slice(int(cu_q[s]), int(cu_q[s + 1]))
    q = torch.zeros((cu_q[-1], heads, d), dtype=TYPES[dtype], device=gpu_device)
    q[:, :, 3] = 8
    v = torch.from_numpy(rng.uniform(1, 2, (cu_k[-1], heads, d)).astype(np.float32)).to(TYPES[dtype]).to(gpu_device)
    marks = sorted({x for y in range(0, t + 1, 32) for x in (y - 1, y) if 0 <= x < t} | {t - 1})
    for at in range(0, len(marks), heads):
        key = torch.tensor([marks[min(at + i, len(marks) - 1)] for i in range(heads)], device=gpu_device)
        k = torch.zeros((cu_k[-1], heads, d), dtype=TYPES[dtype], device=gpu_device)
        k[int(cu_k[s]) + key, torch.arange(heads, device=gpu_device), 3] = 64 * d ** 0.5 / 8
        got = op()(q.flatten(1), k.flatten(1), v.flatten(1), a, b, heads, heads).double().view(-1, heads, d)[rows]
        mine = v[int(cu_k[s]):int(cu_k[s + 1])].double()
        sums = mine.cumsum(0)[t - n:]
        seen = torch.arange(t - n, t, device=gpu_device)[:, None, None]
        want = torch.where(seen >= key[None, :, None], mine[key, torch.arange(heads, device=gpu_device)][None], sums / (seen + 1))
        # (the mean's sums: a step of fp32 a key at most)
        assert ((got - want).abs() <= (h + (t + 8) * u) * want + t * 2.0 ** -90).all(), marks[at]


# ------------------------------------------------------------------------------------------------------- skewed lengths

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,d,new,total", [(25, 25, 64, [1] * 16, [100] * 9 + [20000] + [100] * 6), (32, 8, 128, [1] * 32, [100] * 31 + [20000]), (16, 4, 64, [1] * 40, [500] * 40),
                                                        (16, 4, 64, [3, 1, 40, 1], [100, 90, 50, 17000])], ids=["25x64", "32/8x128", "even", "four"])
def test_one_long_sequence_among_short_ones(gpu_device, dtype, heads, kv_heads, d, new, total):
    """More than 16384 keys in all, whose average says little: sampled rows and heads against the oracle, each with its own sequence's
    length in the bound."""
    cu_q, cu_k = offsets(new), offsets(total)
    tensors = make(np.random.default_rng(7), dtype, cu_q[-1], cu_k[-1], heads, kv_heads, d)
    got = run(gpu_device, tensors, cu_q, cu_k, heads, kv_heads)
    q, k, v = (t.double().numpy() for t in tensors)
    for s in sorted({0, 1, int(np.argmax(total)), len(total) - 1}):
        for h in sorted({0, heads // 2, heads - 1}):
            x, y = slice(h * d, (h + 1) * d), slice(h // (heads // kv_heads) * d, (h // (heads // kv_heads) + 1) * d)
            rows, keys = slice(int(cu_q[s]), int(cu_q[s + 1])), slice(int(cu_k[s]), int(cu_k[s + 1]))
            want = serving.attention_rows(q[rows, x], k[keys, y], v[keys, y], total[s] - new[s])
            worst = np.abs(got[rows, x] - want[0]) / serving.tolerance(dtype, want, total[s], d)
            assert worst.max() <= 1.0, (s, h, worst.max())
