"""What the host does around the 8-bit cache's kernels (no GPU): which kernels a step takes and what it vouches for."""
import inspect
import os
import re
from types import SimpleNamespace

import pytest
import torch

from infinilm_b200 import ops
from infinilm_b200.cache import PagedKVView
from infinilm_b200.engine.step import Workspace
from infinilm_b200.parts.attention import PagedAttend

LAUNCHING = ("attention_decode_quant", "attention_prefill_quant", "kv_unpack", "attention_decode", "attention_plain", "attention_prefill", "attention_prefill_tc5")
SIGNATURES = {name: inspect.signature(getattr(ops, name)) for name in LAUNCHING}
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "infinilm_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name), encoding="utf-8") as fh:
        return re.sub(r"//[^\n]*", "", fh.read())


def _step(monkeypatch, nh, nkv, hd, dtype=torch.bfloat16, n_dec=2, portions=(), quant="int8", prefill="auto"):
    """The kernels that an attention's step launches, as (name, arguments): n_dec requests of one token, then portions."""
    calls = []
    for name in LAUNCHING:
        def record(*a, _name=name, **kw):
            bound = SIGNATURES[_name].bind(*a, **kw)
            bound.apply_defaults()
            calls.append((_name, bound.arguments))
        monkeypatch.setattr(ops, name, record)
    monkeypatch.setattr(ops, "kv_tensor_map", lambda t: None)
    monkeypatch.setattr(ops, "attention_decode_resident_blocks", lambda *a: 296)
    E, T, pages, width = n_dec + len(portions), n_dec + sum(portions), 12, 3
    kvlen = [40] * n_dec + [max(p, 30) for p in portions]
    ctx = SimpleNamespace(n_decode=n_dec, n_entries=E, ws=Workspace("cpu", 64), h_kvlen=kvlen, entry_kvlen=torch.tensor(kvlen, dtype=torch.int32),
                          entry_qstart=torch.zeros(E + 1, dtype=torch.int32), tok_pos=torch.arange(T, dtype=torch.int32), tok_entry=torch.arange(T, dtype=torch.int32),
                          prompt_tiles=lambda n: max(1, len(portions)))
    storage = torch.zeros((pages, nkv, ops.kv_quant_record(hd)), dtype=torch.uint8) if quant else torch.zeros((pages, 2, nkv, 16, hd), dtype=dtype)
    view = PagedKVView(storage, torch.zeros((E, width), dtype=torch.int32), 16, max_pages=width, quant=quant)
    core = PagedAttend(dtype, nh, nkv, hd, 0.1, prefill_kernel=prefill)
    core.run(torch.zeros((T, nh * hd), dtype=dtype), torch.zeros((T, nh * hd), dtype=dtype), ctx, view)
    return calls


# ---- what is read before a kernel's wait ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [16, 32, 48, 80, 96, 112, 192])
def test_pages_read_back_are_not_read_early(monkeypatch, hd):
    """The decode kernel reads the block table and pages before its wait only where its caller says that the kernel in front wrote neither; kv_unpack in front writes both."""
    assert SIGNATURES["attention_decode"].parameters["cached_before"].default is False
    calls = _step(monkeypatch, 4, 2, hd)
    assert [c[0] for c in calls] == ["kv_unpack", "attention_decode"]
    assert calls[1][1]["block_table"].data_ptr() == calls[0][1]["table"].data_ptr() and calls[1][1]["cached_before"] is False
    calls = _step(monkeypatch, 4, 2, hd, quant=None)
    assert [c[0] for c in calls] == ["attention_decode"] and calls[0][1]["cached_before"] is True
    calls = _step(monkeypatch, 4, 2, 64)
    assert [c[0] for c in calls] == ["attention_decode_quant"] and calls[0][1]["cached_before"] is True


def test_the_decode_kernel_starts_early_only_where_it_may():
    text = _source("attn_decode.cu")
    launches = re.findall(r"(\w+)\(\s*\(?([^;]{0,40}?)attn_decode_kernel<", text)
    assert [(f, a.strip()) for f, a in launches if f.startswith("il_launch") or f == "IL_LAUNCH"] == [("il_launch_as", "early != 0,")]


def test_the_plain_kernels_do_not_declare_the_block_table_read_only():
    """They wait first, and the kernel in front may have written the table (kv_unpack does)."""
    found = 0
    for kernel in re.split(r"__global__", _source("attn_plain.cu"))[1:]:
        head, body = kernel.split("{", 1)
        if re.search(r"il_pdl_(?:wait|begin)\(", body):
            found += 1
            assert re.search(r"const int\s*\* block_table", head), head
    assert found == 2


# ---- a step's rows are attended to once --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("nh,nkv,prefill,behind", [(4, 2, "mma", "attention_prefill"), (132, 1, "auto", "attention_plain"), (70, 1, "mma", "attention_plain")])
def test_single_tokens_beside_portions_are_attended_to_once(monkeypatch, nh, nkv, prefill, behind):
    """Where portions have no kernel over codes, only their pages are read back, and only their rows go through the kernels over pages."""
    calls = _step(monkeypatch, nh, nkv, 64, n_dec=2, portions=(5, 9), prefill=prefill)
    assert [c[0] for c in calls] == ["attention_decode_quant", "kv_unpack", behind]
    unpack, last = calls[1][1], calls[2][1]
    assert unpack["first_entry"] == 2
    if behind == "attention_plain":
        assert last["qkv"].shape[0] == last["out"].shape[0] == 14 and last["tok_pos"].tolist() == last["tok_entry"].tolist() == list(range(2, 16))
        assert last["qkv"].is_contiguous() and last["out"].is_contiguous()
    else:
        assert (last["first_entry"], last["n_entries"]) == (2, 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_head_sizes_without_kernels_over_codes_read_all_entries_back(monkeypatch, dtype):
    calls = _step(monkeypatch, 4, 2, 48, dtype=dtype, portions=(5,))
    assert calls[0][0] == "kv_unpack" and calls[0][1]["first_entry"] == 0
    assert [c[0] for c in calls[1:]] == (["attention_plain"] if dtype is torch.float32 else ["attention_decode", "attention_prefill"])


# ---- arguments ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("packed,file,name", [("_STORE_ARGS", "kv_quant.cu", "KvqStoreArgs"), ("_UNPACK_ARGS", "kv_quant.cu", "KvqUnpackArgs"),
                                              ("_DECODE_ARGS", "attn_decode_quant.cu", "DqArgs"), ("_PAIR_ARGS", "attn_prefill_pair.cu", "PpArgs")])
def test_packed_arguments_are_as_long_as_the_struct_that_is_read(packed, file, name):
    """The entry points read a whole struct; its size stands in the source, where the compiler checks it, and follows from its members."""
    text = _source(file)
    size = int(re.search(r"static_assert\(sizeof\(%s\) == (\d+)," % name, text).group(1))
    body = re.search(r"struct %s \{(.*?)\n\};" % name, text, re.S).group(1)
    at, kind = 0, None
    for member in (m for statement in body.split(";") if statement.strip() for m in statement.split(",")):
        words = re.search(r"^\s*((?:const )?(?:void|float|int|long long|cudaStream_t))?\s*(\*?)\s*(\w+)\s*$", member)
        kind = words.group(1) or kind
        width = 8 if words.group(2) or kind in ("long long", "cudaStream_t") else 4
        at = (at + width - 1) // width * width + width
    assert (at + 7) // 8 * 8 == size == getattr(ops, packed).size


def test_an_occupancy_query_that_fails_is_asked_again(monkeypatch):
    answers = [0, 592]
    lib = SimpleNamespace(il_attn_decode_quant_resident_blocks=lambda kind, group: answers.pop(0))
    monkeypatch.setattr(ops.build, "load", lambda *a: lib)
    monkeypatch.setattr(ops, "_resident_quant", {})
    with pytest.raises(ops.KernelError, match="occupancy"):
        ops._quant_blocks(0, 128, 4, 64, 400, 0)
    assert ops._quant_blocks(0, 128, 4, 64, 400, 0) == 592 and not answers
    assert ops._quant_blocks(0, 128, 4, 64, 400, 0) == 592


@pytest.mark.parametrize("file,kernels", [("kv_quant.cu", 4), ("attn_decode_quant.cu", 1)])
def test_descriptors_that_the_kernel_in_front_may_write_are_not_declared_read_only(file, kernels):
    """Nothing says that lengths, tables, positions and entries are older than the kernel in front of these calls (but `cached_before`): their kernels wait first and read them then. The kernel
    that adds parts up stands behind one that has waited."""
    found = 0
    for kernel in re.split(r"__global__", _source(file))[1:]:
        head = kernel.split("{", 1)[0]
        if "merge_kernel" in head:
            continue
        found += 1
        assert re.findall(r"__restrict__ (\w+)", head) in ([], ["inv_freq"]), head
    assert found == kernels


# ---- workspaces ------------------------------------------------------------------------------------------------------------------
@pytest.fixture
def launches(monkeypatch):
    """The entry points with host tensors in place of the device's: everything up to the launch."""
    monkeypatch.setattr(ops, "_on_one_device", lambda *a: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda d: 0)
    monkeypatch.setattr(ops, "_status_ptr", lambda d: 0)
    monkeypatch.setattr(ops, "_quant_fns", {})
    monkeypatch.setattr(ops, "_quant_fn", lambda *a: (lambda args: 0))
    monkeypatch.setattr(ops, "_prefill_tc5_fn", lambda hd: (lambda *a: 0))
    monkeypatch.setattr(ops, "kv_tensor_map", lambda t: torch.zeros(ops.KV_MAP_BYTES, dtype=torch.uint8))
    monkeypatch.setattr(ops, "_has_third_map", lambda m: True)
    monkeypatch.setattr(ops, "attention_plain", lambda *a: None)
    monkeypatch.setattr(ops, "_resident_quant", {(0, 1, 64, wide): 592 for wide in (False, True)})


@pytest.mark.parametrize("dtype,nh", [(torch.bfloat16, 4), (torch.bfloat16, 132), (torch.float32, 4)])
def test_later_steps_leave_the_workspace_as_the_first_made_it(launches, dtype, nh):
    """Chunks of a growing prompt, more requests, wider tables: a buffer that was replaced would make every captured step stale."""
    nkv, hd, pages = (2 if nh < 9 else 1), 64, 300
    core = PagedAttend(dtype, nh, nkv, hd, 0.1)
    storage, ws, seen = torch.zeros((pages, nkv, ops.kv_quant_record(hd)), dtype=torch.uint8), Workspace("cpu", 512), []
    for lengths, portions, width in ([[5], [5], 1], [[80, 40], [75, 1], 5], [[2000, 300], [1000, 1], 125], [[4000] + [1] * 140, [64] + [1] * 140, 256], [[300] * 16, [1] * 16, 20]):
        order = sorted(range(len(portions)), key=lambda i: portions[i] != 1)
        kvlen, qlen = [lengths[i] for i in order], [portions[i] for i in order]
        n_dec, E, T = sum(q == 1 for q in qlen), len(qlen), sum(qlen)
        ctx = SimpleNamespace(n_decode=n_dec, n_entries=E, ws=ws, h_kvlen=kvlen, entry_kvlen=torch.tensor(kvlen, dtype=torch.int32), tok_pos=torch.zeros(T, dtype=torch.int32),
                              entry_qstart=torch.zeros(E + 1, dtype=torch.int32), tok_entry=torch.zeros(T, dtype=torch.int32), prompt_tiles=lambda n: sum((q + n - 1) // n for q in qlen[n_dec:]))
        core.run(torch.zeros((T, nh * hd), dtype=dtype), torch.zeros((T, nh * hd), dtype=dtype), ctx,
                 PagedKVView(storage, torch.zeros((E, width), dtype=torch.int32), 16, max_pages=width, quant="int8"))
        seen.append(ws.version)
    assert seen == [seen[0]] * len(seen), seen


def test_parts_have_room_for_a_wave_of_blocks_from_the_first_call_on(launches):
    nh, nkv, hd, ws, seen = 8, 2, 64, Workspace("cpu", 64), []
    cache = torch.zeros((2, nkv, ops.kv_quant_record(hd)), dtype=torch.uint8)
    for n, length in ((1, 4000), (2, 9000), (8, 30000), (8, 131072)):
        q = torch.zeros((n, nh * hd), dtype=torch.bfloat16)
        ops.attention_decode_quant(q, q.clone(), cache, "int8", torch.zeros((n, 2), dtype=torch.int32), torch.zeros(n, dtype=torch.int32), n, nh, nkv, hd, 0.1, None, length, ws)
        seen.append((ws.version, ws.size("quant_o_part", torch.float32)))
    assert seen == [(0, 592 * 32 * hd)] * 4, seen


def test_a_workspace_that_grows_does_not_keep_what_it_replaces(launches):
    import gc
    import weakref
    ws = Workspace("cpu", 64)
    ops._unpacked_map(ws, 10, 2, 64)
    old = weakref.ref(ws.whole("kv_unpacked", torch.bfloat16))
    gc.collect()
    alive = []
    real = torch.empty
    try:
        torch.empty = lambda *a, **kw: (alive.append(old() is not None), real(*a, **kw))[1]
        ops._unpacked_map(ws, 500, 2, 64)
    finally:
        torch.empty = real
    assert alive == [False] and ws.version == 1


def test_steps_are_padded_by_fewer_entries_than_room_is_held_for():
    from infinilm_b200.engine.step import _ENTRY_BUCKETS, _bucket
    assert max(_bucket(n, _ENTRY_BUCKETS) - n for n in range(1, 5000)) < ops.UNPACKED_SPARE
