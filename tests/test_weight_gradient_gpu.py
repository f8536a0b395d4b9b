"""The weight gradient from 8-bit rows: CTA pairs that hand rows to one another, and rows that
end where their storage ends."""
import zlib

import pytest
import torch

from grappa_b200 import _native

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF = torch.bfloat16


def cu():
    return _native.cuda()


def gen_for(*key):
    g = torch.Generator(device=DEV)
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def coded(g, n, k):
    """Codes, exponents and the rows that they stand for."""
    w = (k + 31) // 32 * 32
    q = torch.randint(-127, 128, (n, w), generator=g, dtype=torch.int8, device=DEV)
    e = torch.randint(118, 123, (n, w // 32), generator=g, device=DEV).to(torch.uint8)
    x = q.double() * torch.exp2(e.double() - 127).repeat_interleave(32, 1)
    return q, e, x[:, :k]


# truncations of at most 2048 rows, 16 at a time, then fp32 sums of chains and shares
def tolerance(n, size):
    return ((min(n, 2048) / 16 + 8) * 2.0 ** -23 + 256 * 2.0 ** -24) * size


@pytest.mark.parametrize("n,k,m", [(64, 512, 256), (50001, 512, 256), (60063, 300, 300), (123457, 136, 200)])
def test_pairs_repeat_bit_for_bit_over_other_data(n, k, m):
    """Two sets of rows in turn through the same kernel: what a block left in shared memory must
    not show in the next one's products."""
    sets = []
    for i in range(2):
        g = gen_for("pair", n, k, m, i)
        dy = torch.randn((n, (m + 7) // 8 * 8), generator=g, device=DEV).to(BF)[:, :m]
        q, e, x = coded(g, n, k)
        sets.append((dy, q, e, dy.double().t() @ x, dy.double().abs().t() @ x.abs()))
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    first = [None, None]
    for _ in range(20):
        for i, (dy, q, e, want, size) in enumerate(sets):
            gw = torch.full((m, k), float("nan"), device=DEV)
            cu().ckpt8_dw(dy, q, e, None, n, gw, err, accumulate=False)
            if first[i] is None:
                assert bool(((gw.double() - want).abs() <= tolerance(n, size)).all())
                first[i] = gw
            assert torch.equal(gw, first[i])
    assert int(err) == 0


@pytest.mark.parametrize("m", [1, 3, 5, 65, 130, 255])
@pytest.mark.parametrize("n,cap,k", [(1, 1, 40), (37, 37, 64), (2001, 2001, 136), (60063, 60063, 200)])
def test_rows_that_end_with_their_storage(n, cap, k, m):
    """The last row of dY ends where its storage ends, without columns to a multiple of 8."""
    g = gen_for("end", n, k, m)
    ld = (m + 7) // 8 * 8
    store = torch.randn((n - 1) * ld + m, generator=g, device=DEV).to(BF)
    dy = store.as_strided((n, m), (ld, 1))
    q, e, x = coded(g, n, k)
    gw = torch.full((m, k), float("nan"), device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    cu().ckpt8_dw(dy, q, e, None, cap, gw, err, accumulate=False)
    want, size = dy.double().t() @ x, dy.double().abs().t() @ x.abs()
    assert bool(((gw.double() - want).abs() <= tolerance(n, size)).all()) and int(err) == 0


def test_columns_past_m_do_not_count():
    """A NaN right behind the M columns, in the row that is read in parts and in the others."""
    g = gen_for("behind")
    n, k, m = 133, 96, 45
    dy = torch.full((n, 64), float("nan"), dtype=BF, device=DEV)
    dy[:, :m] = torch.randn((n, m), generator=g, device=DEV).to(BF)
    q, e, x = coded(g, n, k)
    gw = torch.zeros((m, k), device=DEV)
    cu().ckpt8_dw(dy, q, e, None, n, gw, torch.zeros(1, dtype=torch.int32, device=DEV), accumulate=False)
    want, size = dy[:, :m].double().t() @ x, dy[:, :m].double().abs().t() @ x.abs()
    assert bool(((gw.double() - want).abs() <= tolerance(n, size)).all())
