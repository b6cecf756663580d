"""Steps over the 8-bit cache that mix single tokens and prompt portions, by every path that such a step can take, against attention in 64 bits."""
import math

import pytest
import torch

import plain_kv_quant as P
from test_parts_gpu import _ctx

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind", ["fp8_e4m3", "int8"])
@pytest.mark.parametrize("nh,nkv,hd,prefill", [(4, 2, 64, "mma"), (4, 2, 128, "mma"), (2, 1, 256, "mma"), (4, 2, 128, "auto"), (132, 1, 64, "auto"), (70, 1, 64, "mma"), (4, 2, 96, "auto")])
@pytest.mark.parametrize("window", [None, 24])
def test_single_tokens_beside_portions(cuda_device, kind, nh, nkv, hd, prefill, window):
    """Two requests with a token each, then portions of 5 and 40 tokens: every row is right, and the single tokens' bits are those of a step without portions."""
    from infinilm_b200 import ops
    from infinilm_b200.cache import PagedKVView
    from infinilm_b200.parts.attention import PagedAttend
    starts, qlens = [60, 29, 33, 10], [1, 1, 5, 40]
    kvlens = [s + n for s, n in zip(starts, qlens)]
    need = [(n + 15) // 16 for n in kvlens]
    g = torch.Generator().manual_seed(41)
    ids, rows, at = torch.randperm(sum(need) + 2, generator=g).tolist(), [], 0
    for n in need:
        rows.append(ids[at:at + n] + [-1] * (max(need) - n))
        at += n
    rec = P.make_records(torch.randn((sum(need) + 2, nkv, 2, 16, hd), generator=g), kind)
    val = P.decode_records(rec, hd, kind)
    q = torch.randn((sum(qlens), nh * hd), generator=g).to(torch.bfloat16)
    core = PagedAttend(torch.bfloat16, nh, nkv, hd, 1.0 / math.sqrt(hd), window, prefill_kernel=prefill)

    def go(entries):
        ctx = _ctx("bfloat16", starts[:entries], qlens[:entries])
        out = torch.full((sum(qlens[:entries]), nh * hd), 3.0, dtype=torch.bfloat16, device="cuda")
        core.run(q[:out.shape[0]].cuda(), out, ctx, PagedKVView(rec.cuda(), _i32(rows[:entries]), 16, True, max(need), quant=kind))
        return out.cpu()
    got = go(4)
    if hd in ops.QUANT_HEAD_DIMS:
        assert torch.equal(got[:2], go(2))
    t = 0
    for e in range(4):
        for i in range(qlens[e]):
            want, mag = P.attend(q[t].view(nh, hd), val, rows[e], starts[e] + i, 1.0 / math.sqrt(hd), window or 0)
            # one rounding of the output, one of each weight (bfloat16 at most: 2^-8, and its sum's), sums in 32 bits
            assert ((got[t].double().view(nh, hd) - want).abs() <= 2.0 ** -8 * (1 + 2.0 ** -7) * want.abs() + (2.0 ** -8 + 2.0 ** -14) * mag).all(), (e, i)
            t += 1
    ops.check_status("cuda:0")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_growing_prompt_leaves_captured_steps_as_they_are(cuda_device, dtype):
    """Decode steps are captured, then a long prompt comes in chunks beside them and after it more requests: the same graphs are replayed on."""
    from infinilm_b200 import ops
    from infinilm_b200.engine import StepEntry
    from test_kv_quant_engine_gpu import _config, _engine
    from tiny_configs import make_weights, random_ids
    eng = _engine(_config(64, dtype), make_weights(_config(64, dtype), 6), dtype, "int8")
    ws, room = eng.runner.ws, (eng.cache.groups[0].storage[0].shape[0] + ops.UNPACKED_SPARE) * 2 * 2 * 16 * 64
    assert ws.size("kv_unpacked", eng.dtype) == room          # held before the first request
    eng.enable_graphs()
    a, b = eng.open("a"), eng.open("b")
    eng.step([StepEntry(a, random_ids(20, 320, 1), [19])])
    for t in range(4):
        eng.step([StepEntry(a, [t], [0])])
    version, graphs = eng.runner.ws.version, {k: g.graph for k, g in eng.runner._graphs.items() if g.graph is not None}
    assert len(graphs) == 1
    for chunk in (17, 64, 130, 150):
        eng.step([StepEntry(b, random_ids(chunk, 320, chunk), [chunk - 1])])
        eng.step([StepEntry(a, [3], [0])])
    for i in range(5):
        c = eng.open(("c", i))
        eng.step([StepEntry(a, [5], [0]), StepEntry(c, random_ids(30 + i, 320, i), [0])])
    eng.synchronize()
    assert eng.runner.ws.version == version and all(eng.runner._graphs[k].graph is g for k, g in graphs.items())
