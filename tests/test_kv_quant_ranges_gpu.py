"""Single tokens over the 8-bit cache where values differ most: rows of zeros with the highest scores, exponents as far apart as the format lets them be, many small weights
beside a large one, keys and queries whose powers of two are far apart. Against 64 bits."""
import math

import pytest
import torch

import plain_kv_quant as P

pytestmark = pytest.mark.gpu
KINDS = ["fp8_e4m3", "int8"]
HEADS = [(4, 1, 64), (12, 1, 64), (8, 1, 128), (16, 1, 128), (4, 1, 256), (16, 1, 256)]      # one and two column tiles of heads
BLOCKS = [0, 1, 3, 300, -2, -8]


def _run(dev, monkeypatch, q, kv, kind, blocks, scale, order=None, window=None):
    """One request over kv [keys, kv_heads, 2, head_dim] (pages in `order`); its output, the 64-bit one, and the sums of weight times |value|."""
    from infinilm_b200 import ops
    from infinilm_b200.engine.step import Workspace
    n, nkv, _, hd = kv.shape
    nh, pages = q.shape[0], (n + 15) // 16
    full = torch.cat([kv.double(), torch.zeros((pages * 16 - n, nkv, 2, hd), dtype=torch.float64)]).view(pages, 16, nkv, 2, hd).permute(0, 2, 3, 1, 4).contiguous()
    rec = P.make_records(full, kind)
    val = P.decode_records(rec, hd, kind)
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(5))
    placed = torch.empty_like(rec)
    placed[ids] = rec
    monkeypatch.setattr(ops, "_quant_blocks", lambda *a: blocks)
    out = torch.full((1, nh * hd), 3.0, dtype=torch.bfloat16, device=dev)
    ops.attention_decode_quant(q.reshape(1, -1).to(dev), out, placed.to(dev), kind, ids.to(torch.int32).view(1, -1).to(dev), torch.tensor([n], dtype=torch.int32, device=dev), 1, nh,
                               nkv, hd, scale, window, n, Workspace(dev, 16))
    ops.check_status(dev)
    rows = val.permute(0, 3, 1, 2, 4).reshape(pages * 16, nkv, 2, hd)[:n]
    want, mag = [], []
    for h in range(nh):
        k, v = rows[:, h // (nh // nkv), 0], rows[:, h // (nh // nkv), 1]
        p = torch.softmax(k @ q[h].double() * scale, 0)
        want.append(p @ v), mag.append(p @ v.abs())
    return out.cpu().double().view(nh, hd), torch.stack(want), torch.stack(mag)


def _check(got, want, mag, n):
    # the output's rounding; weights as halves, 2^-11 each, and, where they are subnormal, by 2^-25 of a unit: the largest weight is 2^7 units at least, its row's largest code half
    # of the largest there is, so 2^-31 of the largest column a key; exponentials, exponents and sums in 32 bits: 2^-15 together
    room = want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8) + mag * (2.0 ** -11 + 2.0 ** -15) + 2.0 ** -31 * n * mag.amax(-1, keepdim=True)
    off = (got - want).abs()
    assert (off <= room).all(), float((off / room.clamp(min=1e-300)).max())


def _toward(hd, g):
    u = torch.randn(hd, generator=g).double()
    return u / u.norm()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("blocks", BLOCKS)
@pytest.mark.parametrize("gap,size", [(10.0, 1.0), (8.0, 2.0 ** -4), (12.0, 2.0 ** -4), (0.0, 2.0 ** -14), (14.0, 2.0 ** -14)])
def test_a_row_of_zeros_takes_its_share_and_nothing_else(cuda_device, monkeypatch, kind, nh, nkv, hd, blocks, gap, size):
    """Values of zero at keys whose scores lie `gap` above the others': the sum of weights is theirs, what the others bring keeps its bits. Zeros of both signs."""
    g = torch.Generator().manual_seed(31)
    n, u = 500, _toward(hd, g)
    kv = 0.3 * torch.randn((n, nkv, 2, hd), generator=g).double()
    kv[:, :, 1] *= size / 0.3
    q = (math.sqrt(hd) * u + 0.1 * torch.randn((nh, hd), generator=g).double()).to(torch.bfloat16)
    for at, zero in ((37, 0.0), (290, -0.0)):
        kv[at, :, 0] = (gap * u)                  # q.K / sqrt(hd) is near `gap`
        kv[at, :, 1] = zero
    got, want, mag = _run(cuda_device, monkeypatch, q, kv, kind, blocks, 1.0 / math.sqrt(hd))
    _check(got, want, mag, n)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_zeros_alone_give_zeros(cuda_device, monkeypatch, kind):
    g = torch.Generator().manual_seed(32)
    kv = torch.randn((70, 1, 2, 128), generator=g).double()
    kv[:, :, 1] = 0.0
    got, _, _ = _run(cuda_device, monkeypatch, torch.randn((8, 128), generator=g).to(torch.bfloat16), kv, kind, 0, 0.1)
    assert not got.any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("blocks", BLOCKS)
@pytest.mark.parametrize("how", ["pair", "rising", "falling", "mixed", "zeros"])
def test_values_whose_exponents_lie_as_far_apart_as_they_can(cuda_device, monkeypatch, kind, nh, nkv, hd, blocks, how):
    """The sum of weights counts every key, however small its value beside another's: in one page, page after page of a warp, warp beside warp, block beside block."""
    g = torch.Generator().manual_seed(33)
    n = 400
    kv = torch.randn((n, nkv, 2, hd), generator=g).double()
    if how == "pair":
        e = torch.full((n,), -60.0)
        e[211] = 70.0
    elif how in ("rising", "falling"):
        e = torch.linspace(-90, 98, n).round()
        e = e if how == "rising" else e.flip(0)
    else:
        e = torch.randint(-95, 99, (n,), generator=g).float()
    kv[:, :, 1] *= torch.exp2(e.double())[:, None, None]
    if how == "zeros":
        kv[5::7, :, 1] = 0.0
    q = torch.randn((nh, hd), generator=g).to(torch.bfloat16)
    got, want, mag = _run(cuda_device, monkeypatch, q, kv, kind, blocks, 1.0 / math.sqrt(hd))
    _check(got, want, mag, n)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("blocks", [0, 7, -8])
def test_many_small_weights_beside_a_large_one(cuda_device, monkeypatch, kind, nh, nkv, hd, blocks):
    """16,384 keys of 2^-26 of the largest weight each bring 2^-12 together, in a column of their own."""
    g = torch.Generator().manual_seed(34)
    n, u = 16385, _toward(hd, g)
    kv = torch.zeros((n, nkv, 2, hd)).double()
    kv[6000, :, 0] = 26 * math.log(2.0) * u
    kv[:, :, 1, 1] = 1.0
    kv[6000, :, 1, 1], kv[6000, :, 1, 0] = 0.0, 1.0
    q = (math.sqrt(hd) * u).to(torch.bfloat16).expand(nh, hd).contiguous()
    got, want, mag = _run(cuda_device, monkeypatch, q, kv, kind, blocks, 1.0 / math.sqrt(hd))
    assert (want[:, 1] > 2.0 ** -13).all()
    _check(got, want, mag, n)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("up", [1, -1])
def test_large_keys_with_small_queries(cuda_device, monkeypatch, kind, nh, nkv, hd, up):
    """Scores of ordinary size from keys near 2^106 and queries near 2^-98, and the other way round."""
    g = torch.Generator().manual_seed(35)
    n, sign = 150, torch.sign(torch.randn(hd, generator=g)).double()
    kv = torch.randn((n, nkv, 2, hd), generator=g).double()
    k_size, q_size = (2.0 ** 106, 2.0 ** -98) if up > 0 else (2.0 ** -85, 2.0 ** 93)
    kv[:, :, 0] = k_size * sign * (1 + 0.2 * torch.rand((n, nkv, hd), generator=g).double()) * (0.5 + 0.5 * torch.rand((n, 1, 1), generator=g).double())
    q = (q_size * sign * (1 + 0.1 * torch.rand((nh, hd), generator=g).double())).to(torch.bfloat16)
    got, want, mag = _run(cuda_device, monkeypatch, q, kv, kind, 0, 8.0 / (hd * 2.0 ** 8))
    _check(got, want, mag, n)
