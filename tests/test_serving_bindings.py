"""What the ctypes forms of the serving calls (cmhsa.attention_packed_fwd, cmhsa.kv4_*) check before they call the library.  Tensors on devices that
this machine need not have are stood in for: nothing here launches anything, but where marked."""
import ctypes

import pytest
import torch

import cmhsa


class On:
    """A CPU tensor that says it lies on a device."""

    def __init__(self, t, index):
        self._t, self.device, self.is_cuda = t, torch.device("cuda", index), True

    def __getattr__(self, name):
        return getattr(self._t, name)


@pytest.fixture
def no_library(monkeypatch):
    monkeypatch.setattr(cmhsa, "load_library", lambda: pytest.fail("the library was called"))


@pytest.mark.parametrize("other", ["pages and table", "pages", "table", "offsets", "starts"])
def test_a_pool_on_another_device_is_refused(no_library, other):
    """A pool on another GPU is not this call's to read or write; the torch ops refuse it as well."""
    at = lambda name: int(name in other)  # noqa: E731
    x = On(torch.zeros(4, 128), 0)
    pages, table = On(torch.zeros(3, 2, cmhsa.kv4_block_bytes(16, 64), dtype=torch.uint8), at("pages")), On(torch.zeros(1, 2, dtype=torch.int32), at("table"))
    cu, starts, lengths = On(torch.tensor([0, 4], dtype=torch.int32), at("offsets")), On(torch.zeros(1, dtype=torch.int32), at("starts")), On(torch.zeros(1, dtype=torch.int32), at("offsets"))
    with pytest.raises(ValueError, match="device"):
        cmhsa.kv4_append(x, x, pages, table, cu, starts)
    with pytest.raises(ValueError, match="device"):
        cmhsa.kv4_gather(pages, table, cu, starts, 64, (x, x))
    if other != "starts":
        with pytest.raises(ValueError, match="device"):
            cmhsa.kv4_decode(On(torch.zeros(1, 128), 0), pages, table, lengths, 2)


@pytest.mark.parametrize("src,dst", [([1 << 32], [1]), ([0], [(1 << 32) + 1]), ([-(1 << 32)], [1]), ([3], [1]), ([0], [-1])], ids=str)
@pytest.mark.parametrize("layers", [None, 2])
def test_page_numbers_are_not_cut_to_32_bits(no_library, src, dst, layers):
    shape = (3, 2, cmhsa.kv4_block_bytes(16, 64))
    with pytest.raises(ValueError, match="page numbers"):
        cmhsa.kv4_copy_pages(On(torch.zeros(shape if layers is None else (layers, *shape), dtype=torch.uint8), 0), src, dst)


def test_launches_of_too_many_threads_are_refused():
    """2^32 threads: an error of the launch itself would be left for the caller's next one to find.  (Nothing is read: the library
    refuses before it launches.)"""
    lib, at, block = cmhsa.load_library(), ctypes.c_void_p(0x1000), cmhsa.kv4_block_bytes(64, 64)
    packed = lambda seqs, rows, heads, dtype=1: lib.cmhsa_packed_fwd(at, at, at, at, *[heads * 64] * 4, at, at, seqs, rows, rows, heads, heads, 64, dtype, 1, None, 0, None)  # noqa: E731
    assert packed(1 << 22, 1 << 22, 4) == packed(1 << 24, 8, 1) == packed(1, 1 << 30, 2) == cmhsa.CMHSA_ERR_TOO_LARGE
    pool = (at, 2 * block, 4, 64, at, 1, 1)
    for rows_call, rest in ((lib.cmhsa_kv4_append, ()), (lib.cmhsa_kv4_gather, (1,))):
        for rows in (1 << 27, (1 << 31) - 1025):
            assert rows_call(at, at, 128, 128, 1, *pool, at, None, 1, rows, 2, 64, *rest, None) == cmhsa.CMHSA_ERR_TOO_LARGE
    assert lib.cmhsa_kv4_decode(at, at, 256, 256, 1, *pool, at, 1 << 23, 4, 2, 64, None, 0, None) == cmhsa.CMHSA_ERR_TOO_LARGE
    assert lib.cmhsa_kv4_copy_pages(at, 0, 1, 1 << 39, 2, 1 << 38, (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(1), 1, None) == cmhsa.CMHSA_ERR_TOO_LARGE


@pytest.mark.gpu
def test_a_single_row_has_no_stride(gpu_device):
    """One row, page or layer cut out of something wider: its stride is not used, so it is not held to anything."""
    d, block = 64, cmhsa.kv4_block_bytes(16, 64)
    one = torch.randn(3, 2 * d + 1, device=gpu_device)[:1, :2 * d]
    cu, n = torch.tensor([0, 1], dtype=torch.int32, device=gpu_device), torch.ones(1, dtype=torch.int32, device=gpu_device)
    out = torch.zeros(3, 2 * d + 1, device=gpu_device)[:1, :2 * d]
    # one key: its value, e V / e with e near 1: the part products left out are below 9 u of e V (u = 2^-24), sums, quotient and product 4 u
    got = cmhsa.attention_packed_fwd(one, one, one, cu, cu, 2, 2, out=out).double()
    assert ((got - one).abs() <= 13 * 2.0 ** -24 * one.abs()).all()
    pages = torch.zeros(3, 2 * block + 1, dtype=torch.uint8, device=gpu_device)[:1, :2 * block].view(1, 2, block)
    table = torch.zeros(1, 1, dtype=torch.int32, device=gpu_device)
    row = torch.full((3, 2 * d + 1), 1.5, device=gpu_device)[:1, :2 * d]
    cmhsa.kv4_append(row, row, pages, table, cu)
    back = tuple(torch.zeros(3, 2 * d + 1, device=gpu_device)[:1, :2 * d] for _ in range(2))
    cmhsa.kv4_gather(pages, table, cu, None, d, back)
    assert torch.equal(back[0], row) and torch.equal(back[1], row)
    got = cmhsa.kv4_decode(one, pages, table, n, 2, out=out).double()           # e 1.5 / e, e in three parts, no product left out: 4 u
    assert ((got - 1.5).abs() <= 6 * 2.0 ** -24).all()
    pool = torch.randint(0, 256, (2, 4 * 2 * block + 8), dtype=torch.uint8, device=gpu_device)[:1, :4 * 2 * block].view(1, 4, 2, block)
    want = pool[0, 1].clone()
    cmhsa.kv4_copy_pages(pool, [1], [3])
    assert torch.equal(pool[0, 3], want)
