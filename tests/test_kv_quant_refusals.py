"""The 8-bit cache's entry points refuse what they cannot take before anything is launched (host checks: no GPU)."""
import pytest
import torch

from infinilm_b200 import ops
from infinilm_b200.engine.step import Workspace

NH, NKV, HD, T = 4, 2, 64, 3
REC = 32 * HD + 32


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _store(**kw):
    a = dict(qkv=torch.zeros((T, (NH + 2 * NKV) * HD), dtype=torch.bfloat16), q_out=torch.zeros((T, NH * HD), dtype=torch.bfloat16), tok_pos=_i(T), tok_entry=_i(T),
             block_table=_i(1, 2), cache=torch.zeros((2, NKV, REC), dtype=torch.uint8), kind="int8", n_heads=NH, n_kv_heads=NKV, head_dim=HD, rot_dim=HD,
             inv_freq=torch.zeros(HD // 2), mscale=1.0)
    a.update(kw)
    ops.rope_store_quant(**a)


def _unpack(**kw):
    a = dict(cache=torch.zeros((2, NKV, REC), dtype=torch.uint8), kind="fp8_e4m3", block_table=_i(2, 2), entry_kvlen=_i(2), pages=torch.zeros((4, 2, NKV, 16, HD)))
    a.update(kw)
    ops.kv_unpack(**a)


def _decode(**kw):
    a = dict(q=torch.zeros((2, NH * HD), dtype=torch.bfloat16), out=torch.zeros((2, NH * HD), dtype=torch.bfloat16), cache=torch.zeros((2, NKV, REC), dtype=torch.uint8),
             kind="int8", block_table=_i(2, 2), entry_kvlen=_i(2), n_decode=2, n_heads=NH, n_kv_heads=NKV, head_dim=HD, scale=1.0, window=None, max_kvlen=20,
             ws=Workspace("cpu", 8))
    a.update(kw)
    ops.attention_decode_quant(**a)


def _prefill(**kw):
    a = dict(q=torch.zeros((T, NH * HD), dtype=torch.bfloat16), out=torch.zeros((T, NH * HD), dtype=torch.bfloat16), cache=torch.zeros((2, NKV, REC), dtype=torch.uint8),
             kind="int8", block_table=_i(2, 2), entry_qstart=_i(3), entry_kvlen=_i(2), first_entry=0, n_entries=2, n_tiles_total=2, n_heads=NH, n_kv_heads=NKV, head_dim=HD,
             scale=1.0, window=None, ws=Workspace("cpu", 8))
    a.update(kw)
    ops.attention_prefill_quant(**a)


BF = torch.bfloat16
CASES = [
    (_store, dict(), "CUDA device"),
    (_store, dict(kind="fp8_e5m2"), "kind is one of"),
    (_store, dict(cache=torch.zeros((2, NKV, REC + 16), dtype=torch.uint8)), "cache uint8"),
    (_store, dict(cache=torch.zeros((2, NKV, REC), dtype=torch.int8)), "cache uint8"),
    (_store, dict(cache=torch.zeros((2, REC, NKV), dtype=torch.uint8).transpose(1, 2)), "contiguous"),
    (_store, dict(cache=torch.zeros((2, NKV + 1, REC), dtype=torch.uint8)), "cache uint8"),
    (_store, dict(qkv=torch.zeros((T, NH * HD), dtype=BF)), "qkv"),
    (_store, dict(q_out=torch.zeros((T, NH * HD))), "q_out"),
    (_store, dict(q_out=torch.zeros((T + 1, NH * HD), dtype=BF)), "q_out"),
    (_store, dict(q_out=torch.zeros((1, NH * HD), dtype=BF).expand(T, -1)), "overlap"),
    (_store, dict(tok_pos=torch.zeros(T, dtype=torch.int64)), "int32"),
    (_store, dict(tok_entry=_i(T - 1)), "tok_entry"),
    (_store, dict(block_table=_i(2)), "block_table"),
    (_store, dict(inv_freq=None), "inv_freq"),
    (_store, dict(inv_freq=torch.zeros(HD // 2, dtype=torch.float64)), "inv_freq"),
    (_store, dict(inv_freq=torch.zeros(HD)), "inv_freq"),
    (_unpack, dict(), "CUDA device"),
    (_unpack, dict(kind=0), "kind is one of"),
    (_unpack, dict(pages=torch.zeros((3, 2, NKV, 16, HD))), "room"),
    (_unpack, dict(pages=torch.zeros((4, 2, NKV, 32, HD))), "pages"),
    (_unpack, dict(pages=torch.zeros((4, 2, NKV, 16, HD + 16))), "cache uint8"),
    (_unpack, dict(pages=torch.zeros((4, 2, NKV, HD, 16)).transpose(3, 4)), "contiguous"),
    (_unpack, dict(table=_i(2, 3)), "table"),
    (_unpack, dict(packed=True), "a table"),
    (_unpack, dict(packed=True, table=_i(2, 2), pages=torch.zeros((0, 2, NKV, 16, HD))), "a page at least"),
    (_unpack, dict(first_entry=3), "first_entry"),
    (_unpack, dict(first_entry=-1), "first_entry"),
    (_unpack, dict(entry_kvlen=_i(1)), "entry_kvlen"),
    (_unpack, dict(entry_qstart=_i(2)), "entry_qstart"),
    (_unpack, dict(block_table=_i(2, 4)[:, :2]), "contiguous int32"),
    (_decode, dict(), "CUDA device"),
    (_decode, dict(q=torch.zeros((2, NH * HD))), "bfloat16"),
    (_decode, dict(out=torch.zeros((2, NH * HD), dtype=torch.float16)), "bfloat16"),
    (_decode, dict(head_dim=96), "head sizes"),
    (_decode, dict(n_kv_heads=3), "multiple"),
    (_decode, dict(n_decode=3), "n_decode"),
    (_decode, dict(q=torch.zeros((2, NH * HD - 8), dtype=BF)), "heads"),
    (_decode, dict(kind="int4"), "kind is one of"),
    (_decode, dict(block_table=_i(1, 2)), "block_table"),
    (_decode, dict(entry_kvlen=torch.zeros(2)), "int32"),
    (_prefill, dict(), "CUDA device"),
    (_prefill, dict(head_dim=80), "head sizes"),
    (_prefill, dict(n_heads=NKV * 129), "at most 128"),
    (_prefill, dict(q=torch.zeros((T, NH * HD - 8), dtype=BF)), "q "),
    (_prefill, dict(entry_qstart=_i(2)), "entry_qstart"),
    (_prefill, dict(block_table=_i(1, 2)), "block_table"),
    (_prefill, dict(first_entry=-1), "first_entry"),
    (_prefill, dict(out=torch.zeros((T + 1, NH * HD), dtype=BF)), "out"),
    (_prefill, dict(kind="fp4"), "kind is one of"),
]


@pytest.mark.parametrize("call,kw,says", CASES, ids=[f"{c.__name__[1:]}-{i}" for i, (c, _, _) in enumerate(CASES)])
def test_refused(call, kw, says):
    with pytest.raises(ops.KernelError, match=says):
        call(**kw)


def test_numbers_that_do_not_fit_are_refused_too(monkeypatch):
    monkeypatch.setattr(ops, "_on_one_device", lambda *a: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda d: 0)
    monkeypatch.setattr(ops, "_quant_fn", lambda *a: (lambda args: 0))
    with pytest.raises(ops.KernelError, match="out of range"):
        _unpack(window=1 << 40)


def test_nothing_to_do_is_no_call():
    _store(qkv=torch.zeros((0, (NH + 2 * NKV) * HD), dtype=BF), q_out=torch.zeros((0, NH * HD), dtype=BF))
    _decode(n_decode=0)
    _prefill(first_entry=2)


def test_record_bytes():
    assert ops.kv_quant_record(128) == 4128 and ops.kv_quant_record(64) == 2080


# ---- configuration ---
def test_names_of_the_option():
    from infinilm_b200.cli import build_parser
    from infinilm_b200.config.model_config import ConfigError, parse_kv_cache_dtype
    assert [parse_kv_cache_dtype(n) for n in (None, "auto", "fp8", "fp8_e4m3", "INT8")] == [None, None, "fp8_e4m3", "fp8_e4m3", "int8"]
    with pytest.raises(ConfigError, match="kv_cache_dtype 'int4'"):
        parse_kv_cache_dtype("int4")
    assert build_parser().parse_args([]).kv_cache_dtype == "auto"
    assert build_parser().parse_args(["--kv-cache-dtype", "int8"]).kv_cache_dtype == "int8"
    with pytest.raises(SystemExit):
        build_parser().parse_args(["--kv-cache-dtype", "bf16"])


def test_a_model_whose_layers_have_no_such_cache_is_refused():
    from tiny_configs import tiny_b

    import gopitar_configs
    from infinilm_b200.config.model_config import ConfigError
    from infinilm_b200.config.registry import config_from_json, describe_model
    from infinilm_b200.models.causal_lm import CausalLM, quantise_caches
    spec = describe_model(config_from_json(tiny_b()))
    quantise_caches(spec, "int8")
    assert all(n.quant == "int8" for n in CausalLM(spec, torch.bfloat16).cache_needs())
    raw = gopitar_configs.gp_a()
    with pytest.raises(ConfigError, match="no 8-bit form"):
        quantise_caches(describe_model(config_from_json(raw)), "int8")
    with pytest.raises(ValueError, match="kv_cache is one of"):
        spec.layers[0].mixer.params["kv_cache"] = "int4"
        CausalLM(spec, torch.bfloat16)


def test_descriptions_that_share_a_part():
    """Another model made of the same part keeps its own kind of cache."""
    from dataclasses import replace

    from infinilm_b200.config.registry import config_from_json, describe_model
    from infinilm_b200.models.causal_lm import quantise_caches
    from tiny_configs import tiny_b
    one = describe_model(config_from_json(tiny_b()))
    two = replace(one, layers=list(one.layers))
    quantise_caches(one, "int8")
    assert one.layers[0].mixer.params["kv_cache"] == "int8" and two.layers[0].mixer.params.get("kv_cache") is None


def test_pages_of_such_a_cache():
    from infinilm_b200.cache.manager import CacheManager
    from infinilm_b200.parts.spec import CacheNeed
    need = CacheNeed("paged_kv", n_kv_heads=2, head_dim=64, quant="int8")
    cm = CacheManager([need, CacheNeed("paged_kv", n_kv_heads=2, head_dim=64)], 32, 4, 2)
    assert len(cm.groups) == 2 and cm.bytes_per_token(2) == 2 * (2 * 64 + 2) + 2 * 2 * 64 * 2
    with pytest.raises(ValueError, match="pages of 16"):
        CacheManager([need], 8, 4, 2)
