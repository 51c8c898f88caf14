"""Single-token attention over the paged 4-bit cache (include/cmhsa_kv4.h) where single keys decide: every key marked in turn, one key with all of
the weight at every boundary, scores of -inf.  Expected values are a few operations in 64 bits over numbers that the cache holds exactly."""
import numpy as np
import pytest
import torch

import cmhsa
from test_kv4_cache import TYPES, ints, offsets, ops, pool, table_of

HALF_STEP = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}      # of a rounded output (fp32: counted with the sums)

# lengths, width of the table in positions: one workgroup a sequence (eight waves, four, a wave for two steps) and cut into chunks
CASES = [([1, 0, 17, 300, 511], 512), ([int(x) for x in np.random.default_rng(1).integers(1, 700, 150)], 1024), ([6001, 7, 0, 1100], 6016), ([2049], 4096)]


def places(lengths, device):
    """(sequence, position) of every cached token, in the order in which they are appended."""
    s = torch.cat([torch.full((n,), i) for i, n in enumerate(lengths)]).to(device)
    return s, torch.cat([torch.arange(n) for n in lengths]).to(device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,d,page_size", [(16, 8, 64, 16), (4, 4, 128, 64), (34, 2, 128, 256)])
@pytest.mark.parametrize("lengths,width", CASES, ids=["few", "many", "cut", "cut in one"])
def test_every_key_counts_once(gpu_device, dtype, heads, kv_heads, d, page_size, lengths, width):
    """q = 0: all weights are 1.  Each column of V holds 256 at one position and 0 elsewhere, until every position has been marked: the output
    is 256 over the length, but for the quotient's and the output's roundings (3 u and h), or 0."""
    rng = np.random.default_rng(page_size)
    count = sum(-(-n // page_size) for n in lengths) + 2
    pages, table = pool(count, kv_heads, page_size, d, gpu_device, fill=255), table_of(rng, lengths, page_size, count, gpu_device, -(-width // page_size))
    seq, place = places(lengths, gpu_device)
    columns = kv_heads * d
    k = torch.randn((len(seq), columns), device=gpu_device)
    q = torch.zeros((len(lengths), heads * d), dtype=TYPES[dtype], device=gpu_device)
    n = ints(lengths, gpu_device)
    for at in range(0, max(lengths), columns):
        mark = at + torch.arange(columns, device=gpu_device)[None]
        ops().kv4_append(k, (place[:, None] == mark).float() * 256, pages, table, offsets(lengths, gpu_device), None)
        got = ops().kv4_decode(q, pages, table, n, heads).double()
        mark = mark.view(kv_heads, 1, d).expand(kv_heads, heads // kv_heads, d).reshape(1, -1)
        want = torch.where(mark < n[:, None], 256 / n[:, None].double(), 0.0)
        assert ((got - want).abs() <= (3 * 2.0 ** -24 + HALF_STEP[dtype]) * want).all(), at


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("d,page_size", [(64, 16), (128, 64)])
@pytest.mark.parametrize("lengths,width", CASES, ids=["few", "many", "cut", "cut in one"])
def test_one_key_with_all_of_the_weight(gpu_device, dtype, d, page_size, lengths, width):
    """Each K/V head of the longest sequence has one key with a score of 64 where the others have 0, at every boundary of 16 in turn:
    the output is its value (the others weigh 2^-92 each).  Sixteen heads, so sixteen keys a call."""
    rng = np.random.default_rng(d)
    heads = 16
    count = sum(-(-n // page_size) for n in lengths) + 2
    pages, table = pool(count, heads, page_size, d, gpu_device, fill=255), table_of(rng, lengths, page_size, count, gpu_device, -(-width // page_size))
    seq, place = places(lengths, gpu_device)
    s = int(np.argmax(lengths))
    first, t = sum(lengths[:s]), lengths[s]
    v = torch.from_numpy(rng.choice([1.0, 1.5, 2.0, 3.0, 4.0, 6.0], (len(seq), heads * d)).astype(np.float32)).to(gpu_device)
    v[:, ::32] = 6                                               # scale 1: every value is one of the format's
    q = torch.zeros((len(lengths), heads, d), dtype=TYPES[dtype], device=gpu_device)
    q[:, :, 3] = 16 if d == 64 else 16 * 2 ** 0.5
    marks = sorted({x for y in range(0, t + 1, 16) for x in (y - 1, y) if 0 <= x < t} | {t - 1})
    for at in range(0, len(marks), heads):
        key = torch.tensor([marks[min(at + i, len(marks) - 1)] for i in range(heads)], device=gpu_device)
        k = torch.zeros((len(seq), heads, d), device=gpu_device)
        k[first + key, torch.arange(heads, device=gpu_device), 3] = 32               # 32 * 16 / 8 = 64
        ops().kv4_append(k.flatten(1), v, pages, table, offsets(lengths, gpu_device), None)
        got = ops().kv4_decode(q.flatten(1), pages, table, ints(lengths, gpu_device), heads).double()[s].view(heads, d)
        want = v[first:first + t].double().view(t, heads, d)[key, torch.arange(heads, device=gpu_device)]
        assert ((got - want).abs() <= (HALF_STEP[dtype] + 4 * 2.0 ** -24) * want + 6 * t * 2.0 ** -89).all(), marks[at]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("lengths,width", [([100, 1, 33, 60], 128), ([3000, 400, 90, 2500], 3136)], ids=["one workgroup", "cut"])
def test_scores_of_minus_infinity(gpu_device, dtype, heads, kv_heads, d, lengths, width):
    """q . k passes fp32's range: the weight is 0 where another key's score is finite, and a sequence of nothing else is 0 / 0, as the formula
    gives; where no position has a page the output is 0 all the same."""
    page_size = 64
    count = sum(-(-n // page_size) for n in lengths) + 2
    pages, table = pool(count, kv_heads, page_size, d, gpu_device, fill=255), table_of(np.random.default_rng(3), lengths, page_size, count, gpu_device, width // page_size)
    seq, place = places(lengths, gpu_device)
    k, v = (torch.zeros((len(seq), kv_heads, d), device=gpu_device) for _ in range(2))
    low = ((seq == 0) & (place < 70)) | (seq == 1) | ((seq == 2) & (place >= 1)) | (seq == 3)
    k[low, :, 7] = -2.0 ** 120
    v[~low] = 4
    q = torch.zeros((4, heads, d), dtype=TYPES[dtype], device=gpu_device)
    q[:, :, 7] = 2.0 ** 15
    ops().kv4_append(k.flatten(1), v.flatten(1), pages, table, offsets(lengths, gpu_device), None)
    got = ops().kv4_decode(q.flatten(1), pages, table, ints(lengths, gpu_device), heads)
    assert (got[0] == 4).all() and (got[2] == 4).all()
    assert torch.isnan(got[1]).all() and torch.isnan(got[3]).all()
    table[3] = -1
    table[1] = count
    got = ops().kv4_decode(q.flatten(1), pages, table, ints(lengths, gpu_device), heads)
    assert (got[0] == 4).all() and (got[2] == 4).all() and (got[1] == 0).all() and (got[3] == 0).all()


@pytest.mark.gpu
def test_many_sequences_in_a_long_table(gpu_device):
    """More sequences than a look through all of their lengths pays for: not cut, and every key counts once all the same."""
    rng = np.random.default_rng(4)
    heads, kv_heads, d, page_size, width = 4, 2, 64, 64, 2112
    lengths = [int(x) for x in rng.integers(0, 300, 599)] + [2100]
    assert cmhsa.load_library().cmhsa_kv4_decode_workspace_bytes(600, width // page_size, page_size, heads, kv_heads, d) == 0
    assert cmhsa.load_library().cmhsa_kv4_decode_workspace_bytes(64, width // page_size, page_size, heads, kv_heads, d) > 0
    test_every_key_counts_once(gpu_device, "bfloat16", heads, kv_heads, d, page_size, lengths, width)
