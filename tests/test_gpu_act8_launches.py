"""Matrices of more rows than one launch takes: what the later launches read and write, and the depth of dw's sums.

A thousand rows repeat, so the same call on those alone is the answer for all; the format is exact and every row's
arithmetic its own, so the answers are the same bits."""

import pytest
import torch

import nanopysche_amd as fm
from tests.act8_reference import kept
from tests.test_gpu_act8 import U32, activation, gen

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
N = 1000   # rows that repeat


@pytest.fixture(autouse=True)
def _memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def repeated(rows, T):
    return rows.repeat((T + N - 1) // N, 1)[:T]


def all_alike(got, one):
    """Rows of ``got`` are those of ``one``, over and over."""
    whole = got.shape[0] // N
    return (torch.equal(got[:whole * N].view(whole, N, -1), one.expand(whole, N, -1))
            and torch.equal(got[whole * N:], one[:got.shape[0] - whole * N]))


def test_rmsnorm_in_two_launches(dev):
    """A row of 257 to 512 columns takes a wave, four a workgroup: 2^25 rows a launch."""
    D, T = 264, 2 ** 25 + 4000
    rows, w = activation(gen(1), N, D), torch.rand(D, generator=gen(2), device="cuda")
    x = repeated(rows, T)
    y, k, r = fm.rmsnorm_compress(x, w)
    ys, ks, rs = fm.rmsnorm_compress(rows, w)
    assert all_alike(y, ys) and all_alike(r[:, None], rs[:, None])
    assert all_alike(k.data[:T * k.pitch].view(T, -1), ks.data[:N * k.pitch].view(N, -1))
    assert all_alike(k.data[T * k.pitch:].view(T, -1), ks.data[N * k.pitch:].view(N, -1))
    del y
    gx, gw = fm.rmsnorm_backward_8bit(x, k, w, r)
    gs, _ = fm.rmsnorm_backward_8bit(rows, ks, w, rs)
    assert all_alike(gx, gs)
    check_dw(gw, rows, rs, T, teams=8)


def check_dw(gw, rows, rs, T, teams):
    """512 slices; a slice's rows go around its teams, each adding its own in order; then the teams, 8 slices to a row of threads of the
    second launch, and its 64 rows of threads."""
    terms = rows.double() * kept(rows.double()) * rs.double()[:, None]
    ref = terms.sum(0) * (T // N) + terms[:T % N].sum(0)
    size = terms.abs().sum(0) * (T // N) + terms[:T % N].abs().sum(0)
    depth = -(-T // 512 // teams) + 1 + teams + 8 + 64
    # x r and its product with dy are rounded too: two more
    assert torch.all((gw.double() - ref).abs() <= (depth + 2) * U32 * size)


def test_dw_of_many_narrow_rows(dev):
    """Eight lanes a row, 64 teams to a workgroup: about a thousand rows one after the other."""
    T = 2 ** 25 + 4000
    rows, w = activation(gen(15), N, 8), torch.rand(8, generator=gen(16), device="cuda")
    x = repeated(rows, T)
    _, k, r = fm.rmsnorm_compress(x, w)
    _, gw = fm.rmsnorm_backward_8bit(x, k, w, r)
    check_dw(gw, rows, fm.rmsnorm_compress(rows, w).rstd, T, teams=64)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_restore_in_several_launches(dev, dtype):
    """2^30 eights of bf16, or fours of fp32, a launch: 2^19 or 2^18 rows of 16384."""
    cols, T = 16384, (2 ** 19 if dtype == BF else 2 ** 18) + 130
    rows = activation(gen(3), N, cols, dtype=dtype)
    ref = kept(rows.double()).to(dtype)
    t = fm.compress_activation(repeated(rows, T))
    assert all_alike(t.restore(), ref)
    del t
    few = fm.compress_activation(rows)
    index = (torch.arange(T, device="cuda") % N).int()
    index[-3:] = -1
    got = few.restore_rows(index)
    assert all_alike(got[:-3], ref) and not got[-3:].any()


def test_swiglu_in_two_launches(dev):
    """2^30 eights a launch: 2^19 rows of 16384."""
    cols, T = 16384, 2 ** 19 + 130
    g, u = activation(gen(4), N, cols), activation(gen(5), N, cols)
    gate, up = repeated(g, T), repeated(u, T)
    h, g8, u8 = fm.swiglu_compress(gate, up)
    hs, gs, us = fm.swiglu_compress(g, u)
    assert all_alike(h, hs)
    for big, small in ((g8, gs), (u8, us)):
        assert all_alike(big.data[:T * cols].view(T, -1), small.data[:N * cols].view(N, -1))
        assert all_alike(big.data[T * cols:].view(T, -1), small.data[N * cols:].view(N, -1))
    del h, gate
    dg, du = fm.swiglu_backward_8bit(up, g8, u8)
    dgs, dus = fm.swiglu_backward_8bit(u, gs, us)
    assert all_alike(dg, dgs) and all_alike(du, dus)
