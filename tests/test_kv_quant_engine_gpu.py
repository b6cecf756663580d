"""The 8-bit cache under the attention mixer, the engine and the command line: every step against plain attention over the values the cache itself holds, whole models against the
plain model with its keys and values rounded, prompts cut anywhere, steps replayed as graphs."""
import math

import pytest
import torch

import plain_kv_quant as P
import plain_model
from test_parts_gpu import DT, _ctx
from tiny_configs import make_weights, random_ids

pytestmark = pytest.mark.gpu

from infinilm_b200.cache import CacheManager, PagedKVView  # noqa: E402
from infinilm_b200.parts import PartSpec, build_part  # noqa: E402

KINDS = ["fp8_e4m3", "int8"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("nh,nkv,hd,rot", [(6, 2, 64, 64), (4, 4, 128, 64), (20, 1, 64, 32), (3, 1, 256, 256), (6, 3, 48, 24), (4, 2, 16, 16)])
@pytest.mark.parametrize("window", [None, 24])
@pytest.mark.parametrize("normed", [False, True])
def test_attention_part_over_codes(cuda_device, kind, dtype, nh, nkv, hd, rot, window, normed):
    """A prompt portion for two requests, then a single token for one beside a further portion of the other, then a token each; head sizes with kernels of their own over codes and
    without. What is expected is made from the mixer's input and from what the cache holds."""
    from infinilm_b200 import ops
    H = 96
    params = {"hidden": H, "n_heads": nh, "n_kv_heads": nkv, "head_dim": hd, "qkv_bias": True, "window": window, "kv_cache": kind,
              "position": PartSpec("rope", {"rot_dim": rot, "theta": 10000.0})}
    att = build_part("mixer", PartSpec("attention", params, "a"), DT[dtype])
    g = torch.Generator().manual_seed(1)
    w = {ws.name: (torch.randn(ws.shape, generator=g) * (0.15 if ws.role == "matrix" else 0.05)).bfloat16().float() for ws in att.weight_specs()}
    att.set_weights({k: v.cuda() for k, v in w.items()})
    need = att.cache_need()
    assert need.quant == kind
    cm = CacheManager([need], 32, 8, 4, device="cuda", dtype=DT[dtype])         # pages of two kernel pages
    storage = cm.groups[0].storage[0]
    assert tuple(storage.shape) == (18, nkv, ops.kv_quant_record(hd)) and storage.dtype == torch.uint8 and cm.bytes_per_token(2) == nkv * (2 * hd + 2)
    xs = {"a": torch.randn(45, H, generator=g).to(DT[dtype]), "b": torch.randn(23, H, generator=g).to(DT[dtype])}
    seqs = {k: cm.open(k) for k in xs}
    # q, k and v in the compute dtype (one rounding of each), the weights' rounding, the output's and, in the product behind it, the attention's: steps of 2^-8 each in
    # bfloat16; the largest numbers of a row are what errors are measured by
    tol = {"float32": 2e-5, "bfloat16": 2.5e-2}[dtype]

    def step(parts):
        starts, qlens = [seqs[k].length for k, _ in parts], [n for _, n in parts]
        for k, n in parts:
            cm.reserve(seqs[k], seqs[k].length + n)
        ctx = _ctx(dtype, starts, qlens)
        tabs = [seqs[k].tables[0].array().tolist() for k, _ in parts]
        W = max(map(len, tabs))
        bt = torch.tensor([t + [-1] * (W - len(t)) for t in tabs], dtype=torch.int32).cuda()
        x = torch.cat([xs[k][s: s + n] for (k, n), s in zip(parts, starts)]).cuda()
        T = x.shape[0]
        arg = x
        if normed and dtype == "bfloat16" and att.accepts_normed(T):              # the norm's division inside the projection
            arg = ops.NormedInput(x, torch.full((T, H // 16), 4.0, device="cuda"), H, 0.0)
        y = att.forward(arg, ctx, PagedKVView(storage, bt, 16, True, W, quant=kind)).float().cpu()
        xd = x.double().cpu() / (math.sqrt(4.0 * (H // 16) / H) if arg is not x else 1.0)
        val = P.decode_records(storage.cpu(), hd, kind)
        q = xd @ w["q_proj.weight"].double().T + w["q_proj.bias"].double()
        pos = ctx.tok_pos.cpu()
        ang = pos.double()[:, None] * att.position.inv_freq.cpu().double()
        q = plain_model.apply_rope(q.view(T, nh, hd), ang.cos(), ang.sin(), rot)
        for t in range(T):
            e = int(ctx.tok_entry[t])
            o, _ = P.attend(q[t], val, bt[e].cpu().tolist(), int(pos[t]), 1.0 / math.sqrt(hd), window or 0)
            want = o.reshape(-1) @ w["o_proj.weight"].double().T
            assert (y[t].double() - want).abs().max() <= tol * want.abs().max(), (parts, t)
        # and what the cache holds is what was projected: v, not rotated, to within the codes' steps and the projection's rounding
        v = xd @ w["v_proj.weight"].double().T + w["v_proj.bias"].double()
        for t in (0, T - 1):
            e, p = int(ctx.tok_entry[t]), int(pos[t])
            got = val[int(bt[e, p // 16]), :, 1, p % 16]
            row = v[t].view(nkv, hd)
            room = row.abs().amax(-1, keepdim=True) * (2.0 ** -7 if dtype == "bfloat16" else 1e-5)
            assert ((got - row).abs() <= room + row.abs().amax(-1, keepdim=True) * (2.0 ** -6 if kind == "int8" else 2.0 ** -4)).all()
        for k, n in parts:
            cm.commit(seqs[k], seqs[k].length + n)
    step([("a", 30), ("b", 20)])
    step([("b", 1), ("a", 12)])
    step([("a", 1), ("b", 1)])
    step([("b", 1)])
    torch.cuda.synchronize()
    ops.check_status("cuda:0")


def _config(hd, dtype="float32"):
    return {"architectures": ["MiniCPMForCausalLM"], "model_type": "minicpm4", "num_hidden_layers": 3, "hidden_size": 256, "num_attention_heads": 8,
            "num_key_value_heads": 2, "head_dim": hd, "intermediate_size": 384, "vocab_size": 320, "rope_theta": 10000.0, "max_position_embeddings": 512,
            "scale_emb": 4.0, "dim_model_base": 128, "scale_depth": 1.4, "rms_norm_eps": 1e-5, "tie_word_embeddings": False, "torch_dtype": dtype,
            "eos_token_id": [1]}


def _engine(raw, w, dtype, kind, **kw):
    from infinilm_b200.config import config_from_json
    from infinilm_b200.engine import Engine
    return Engine.from_tensors(config_from_json(raw), w, dtype=dtype, page_size=16, num_pages=64, max_seqs=8, max_batch_tokens=512, kv_cache_dtype=kind, **kw)


def _plain(monkeypatch, raw, w, ids, kind, bf16):
    real = plain_model.attention_scores
    monkeypatch.setattr(plain_model, "attention_scores",
                        lambda q, k, v, window=None: real(q, P.encode(k.double(), kind)[0].float(), P.encode(v.double(), kind)[0].float(), window))
    out = plain_model.forward(raw, w, ids, round_embedding_bf16=bf16)
    monkeypatch.setattr(plain_model, "attention_scores", real)
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [64, 32])
def test_model_against_the_plain_one_with_rounded_keys_and_values(cuda_device, monkeypatch, kind, dtype, hd):
    """Whole prompts and prompts cut into portions and single tokens. A number next to the border between two codes may fall to the other side: a share of the row's codes of
    2^-24 / 2^-4 per unit of the last place in 32 bits, 2^-8 / 2^-4 in bfloat16, by a step of 2^-3 of the number each; over the row that is 2^-4 sqrt(2^-4) of the norm in bfloat16 at
    most, beside bfloat16's own 2.5e-2."""
    raw = _config(hd)
    w = make_weights(raw, 3)
    eng = _engine(raw, w, dtype, kind)
    ids = {"a": random_ids(70, 320, 5), "b": random_ids(33, 320, 6)}
    cuts = ([70], [33]), ([30, 1, 1, 38], [1, 20, 12])
    tol = {"float32": 4e-3, "bfloat16": 4e-2}[dtype]
    ref = {k: _plain(monkeypatch, raw, w, v, kind, dtype == "bfloat16") for k, v in ids.items()}
    from infinilm_b200.engine import StepEntry
    for cut_a, cut_b in cuts:
        seqs = {k: eng.open(k + str(len(cut_a))) for k in ids}
        got, at = {k: [] for k in ids}, {k: 0 for k in ids}
        for i in range(max(len(cut_a), len(cut_b))):
            entries, order = [], []
            for k, cut in (("a", cut_a), ("b", cut_b)):
                if i < len(cut):
                    entries.append(StepEntry(seqs[k], ids[k][at[k]:at[k] + cut[i]], list(range(cut[i]))))
                    order.append((k, cut[i]))
                    at[k] += cut[i]
            logits, a = eng.step(entries).float().cpu(), 0
            for k, n in order:
                got[k].append(logits[a:a + n])
                a += n
        for k in ids:
            g = torch.cat(got[k])
            off = (g - ref[k]).norm() / ref[k].norm()
            assert off <= tol, (kind, dtype, cut_a, k, float(off))
            eng.close(seqs[k])
    eng.synchronize()


@pytest.mark.parametrize("kind", KINDS)
def test_replayed_steps_are_the_eager_ones(cuda_device, kind):
    """Generation with graphs (decode steps, repeated prompt portions) and without: logits as near as sums in another order leave them."""
    from infinilm_b200.engine import StepEntry
    raw = _config(64, "bfloat16")
    w = make_weights(raw, 4)
    outs = []
    for graphs in (False, True):
        eng = _engine(raw, w, "bfloat16", kind)
        if graphs:
            eng.enable_graphs()
        rows = []
        for round_ in range(5):                   # prompts of one shape come back: from the third on their step is replayed
            seqs = [eng.open((round_, i)) for i in range(3)]
            prompts = [random_ids(25, 320, 10 * round_ + i) for i in range(3)]
            rows.append(eng.step([StepEntry(s, p, [24]) for s, p in zip(seqs, prompts)]).float().cpu().clone())
            for t in range(12):
                rows.append(eng.step([StepEntry(s, [(7 * t + i) % 320], [0]) for i, s in enumerate(seqs)]).float().cpu().clone())
            for s in seqs:
                eng.close(s)
        eng.synchronize()
        outs.append(torch.cat(rows))
    assert eng.runner.portion_replays > 0
    # the same K and V rows and codes come of the same kernels; only the attention's blocks differ: 2^-8 a layer, and what a code next to its border makes of that
    assert (outs[0] - outs[1]).norm() <= 3e-2 * outs[0].norm()


@pytest.mark.parametrize("kind", KINDS)
def test_generate_through_the_entry_point(cuda_device, kind):
    from infinilm_b200.config import config_from_json
    from infinilm_b200.llm import LLM, SamplingParams
    raw = _config(128, "bfloat16")
    w = make_weights(raw, 5)
    llm = LLM.from_tensors(config_from_json(raw), w, num_blocks=32, block_size=32, max_batch_size=4, kv_cache_dtype=kind, enable_graph=True)
    out = llm.generate(prompt_token_ids=[random_ids(n, 320, n) for n in (5, 40, 17)], sampling_params=SamplingParams(top_k=1, max_tokens=20, ignore_eos=True))
    assert [len(o.outputs[0].token_ids) for o in out] == [20, 20, 20] and llm.engine.kv_cache_dtype == kind
    half = llm.engine.cache.bytes_per_token(2)
    llm.close()
    full = LLM.from_tensors(config_from_json(raw), w, num_blocks=32, block_size=32, max_batch_size=4)
    assert half * 2 < full.engine.cache.bytes_per_token(2) * 1.02
    full.close()
