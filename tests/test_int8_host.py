"""What the operators of 8-bit codes refuse, and their plain forms (no GPU)."""
import pytest
import torch

import int8_plain as plain

I8, F32, BF16, I32 = torch.int8, torch.float32, torch.bfloat16, torch.int32


def empty(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


def store_args(**change):
    a = dict(qkv=empty(5, 5 * 64, dtype=BF16), q=empty(5, 3 * 64, dtype=BF16), pos=empty(5, dtype=I32), seq=empty(5, dtype=I32),
             table=empty(2, 3, dtype=I32), cos=empty(9, 32), sin=empty(9, 32), k=empty(4, 1, 64, 64, dtype=I8), v=empty(4, 1, 64, 64, dtype=I8),
             ks=empty(4, 1, 64), vs=empty(4, 1, 64), heads=3, kv_heads=1, d=64, page=64)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,why", [
    (dict(), "CUDA tensors only"), (dict(qkv=empty(5, 5 * 64, dtype=torch.float16)), "float16"), (dict(q=empty(5, 3 * 64)), "q is"),
    (dict(q=empty(4, 3 * 64, dtype=BF16)), "q is"), (dict(k=empty(4, 1, 64, 64)), "k is"), (dict(v=empty(3, 1, 64, 64, dtype=I8)), "v is"),
    (dict(ks=empty(4, 1, 63)), "k_scales is"), (dict(vs=empty(4, 1, 64, dtype=BF16)), "v_scales is"), (dict(pos=empty(4, dtype=I32)), "each of 5 rows"),
    (dict(seq=empty(5, dtype=torch.int64)), "token_seq is"), (dict(table=empty(6, dtype=I32)), "page_table is"), (dict(sin=None), "cos and sin"),
    (dict(cos=empty(9, 31)), "cos is"), (dict(sin=empty(8, 32)), "sin is"), (dict(heads=0), "query head"), (dict(d=63), "even head sizes"),
    (dict(kv_heads=0), "even head sizes"), (dict(qkv=empty(5, 6 * 64, dtype=BF16)[:, 64:]), "not contiguous")])
def test_writing_refuses(change, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.rope_store_int8(*store_args(**change))


def read_args(**change):
    a = dict(k=empty(4, 2, 64, 64, dtype=I8), v=empty(4, 2, 64, 64, dtype=I8), ks=empty(4, 2, 64), vs=empty(4, 2, 64), table=empty(2, 3, dtype=I32),
             local=empty(2, 3, dtype=I32), ko=empty(5, 2, 64, 64, dtype=BF16), vo=empty(5, 2, 64, 64, dtype=BF16))
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,why", [
    (dict(), "CUDA tensors only"), (dict(k=empty(4, 2, 64, 64)), "k is"), (dict(k=empty(4, 64, 64, dtype=I8)), "k is int8"),
    (dict(vs=empty(4, 64, 2)), "v_scales is"), (dict(local=empty(2, 3, dtype=torch.int64)), "local_table is"), (dict(vo=empty(5, 2, 64, 64)), "v_out is"),
    (dict(ko=empty(5, 2, 64, 63, dtype=BF16)), "k_out is"), (dict(vo=empty(4, 2, 64, 64, dtype=BF16)), "v_out is"),
    (dict(ko=empty(5, 2, 64, 64, dtype=torch.float16)), "float16")])
def test_reading_refuses(change, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.read_pages_int8(*read_args(**change))


def attend_args(**change):
    a = dict(q=empty(5, 6 * 64, dtype=BF16), stride=6 * 64, k=empty(4, 2, 64, 64, dtype=I8), v=empty(4, 2, 64, 64, dtype=I8), ks=empty(4, 2, 64),
             vs=empty(4, 2, 64), pos=empty(5, dtype=I32), seq=empty(5, dtype=I32), table=empty(2, 3, dtype=I32), out=empty(5, 6 * 64, dtype=BF16),
             heads=6, kv_heads=2, d=64, window=0, scale=0.125, ws=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,why", [
    (dict(), "CUDA tensors only"), (dict(q=empty(5, 6 * 64)), "out is"), (dict(out=empty(5, 5 * 64, dtype=BF16)), "out is"), (dict(k=empty(4, 2, 64, 64)), "k is"),
    (dict(ks=empty(4, 2, 64, 1)), "k_scales is"), (dict(pos=empty(5)), "token_pos is"), (dict(table=empty(2, 3)), "page_table is"),
    (dict(q=empty(5, 6 * 64, dtype=torch.float16), out=empty(5, 6 * 64, dtype=torch.float16)), "float16")])
def test_attention_refuses(change, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.attention_int8(*attend_args(**change))


def product_args(**change):
    a = dict(x=empty(5, 40, dtype=BF16), w=empty(12, 48, dtype=I8), ws=empty(12), bias=None, out=empty(5, 12, dtype=BF16), mode=0, space=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,why", [
    (dict(), "CUDA tensors only"), (dict(x=empty(5, 40, dtype=torch.float16)), "float16"), (dict(w=empty(12, 40, dtype=I8)), "w is"), (dict(w=empty(12, 48)), "w is"),
    (dict(ws=empty(11)), "w_scales is"), (dict(bias=empty(12, dtype=BF16)), "bias is"), (dict(out=empty(5, 12)), "out is"), (dict(mode=1), "out is"),
    (dict(mode=3), "out is"), (dict(mode=7), "mode 7"), (dict(w=empty(11, 48, dtype=I8), mode=3), "no gate and up")])
def test_products_refuse(change, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.linear_int8(*product_args(**change))


@pytest.mark.parametrize("x,codes,scales,why", [
    (empty(3, 20), empty(3, 32, dtype=I8), empty(3), "CUDA tensors only"), (empty(3, 20), empty(3, 20, dtype=I8), empty(3), "codes is"),
    (empty(3, 20), empty(3, 32, dtype=I8), empty(4), "scales is"), (empty(20, 3).T, empty(3, 32, dtype=I8), empty(3), "beside one another"),
    (empty(3, 0), empty(3, 0, dtype=I8), empty(3), "k >= 1"), (empty(3, 20, dtype=torch.float16), empty(3, 32, dtype=I8), empty(3), "float16")])
def test_codes_of_rows_refuse(x, codes, scales, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.quantize_rows(x, codes, scales)


def test_codes_are_within_half_a_step():
    x = torch.randn((200, 64), generator=torch.Generator().manual_seed(0))
    codes, scales = plain.codes_of(x)
    assert codes.abs().amax() == 127
    assert ((codes.double() * scales.double()[:, None] - x.double()).abs() <= x.abs().amax(1, keepdim=True).double() / 254 * (1 + 2.0 ** -20)).all()


def test_codes_of_bfloat16_rows_are_the_exact_quotients():
    """Every pair of a value and a top of 8 significant bits: the code is the exact quotient's, ties to even; half of the top, 63.5 steps,
    may go either way."""
    top = torch.arange(128, 256, dtype=F32)
    for e in (1.0, 0.5, 0.25, 2.0 ** -6):
        x = torch.arange(128, 256, dtype=F32) * e
        rows = torch.stack((x[None].expand(128, -1), top[:, None].expand(-1, 128)), -1)
        rows = rows[(x[None] <= top[:, None])]
        codes, _ = plain.codes_of(rows)
        whole = (rows[:, 0].double() * 127).div(rows[:, 1].double(), rounding_mode="floor")
        part = rows[:, 0].double() * 127 - whole * rows[:, 1].double()  # (exact)
        up = (2 * part > rows[:, 1]) | ((2 * part == rows[:, 1]) & (whole % 2 == 1))
        half = 2 * rows[:, 0] == rows[:, 1]
        assert torch.equal(codes[~half, 0].double(), (whole + up)[~half])
        assert ((codes[half, 0] == 63) | (codes[half, 0] == 64)).all()


# ---- the cache, the model and the command line --------------------------------------------------
def test_pages_of_codes_are_copied_with_their_scales():
    from nnis_b200.cache import CacheManager, KVRequest
    cache = CacheManager([KVRequest(2, 8, codes=True)] * 3 + [KVRequest(2, 8)], F32, torch.device("cpu"), 64 * 8, 4, 1000)
    codes, wide = cache.groups
    assert (codes.k.dtype, wide.k.dtype, codes.k_scales.shape, wide.k_scales) == (I8, F32, (3, 8, 2, 64), None)
    view = cache.view(1)
    assert view.k_scales.shape == (8, 2, 64) and view.v_scales.data_ptr() == codes.v_scales[1].data_ptr() and cache.view(3).k_scales is None
    a = cache.acquire()
    cache.reserve([a], [70])
    cache.commit([a], [70])
    for t in codes.stores():
        t[:, cache.page_table(0, a)[1], :, :6] = 9
    b = cache.fork(a)
    cache.reserve([b], [71])
    cache.commit([b], [71])
    mine, copy = cache.page_table(0, a)[1], cache.page_table(0, b)[1]
    assert mine != copy and all((t[:, copy, :, :6] == 9).all() and (t[:, copy, :, 6:] == 0).all() for t in codes.stores())
    assert cache.kv_bytes_per_token() == 3 * 2 * (16 + 8) + 2 * 16 * 4
    assert cache.kv_bytes_read(10) == 10 * cache.kv_bytes_per_token()
    assert cache.usage()["kv_bytes"] == 8 * 64 * cache.kv_bytes_per_token()
    cache.check()


def test_a_cache_of_codes_without_values_is_refused():
    from nnis_b200.cache import CacheManager, KVRequest
    with pytest.raises(ValueError, match="keys and values"):
        CacheManager([KVRequest(1, 8, values=False, codes=True)], F32, torch.device("cpu"), 64, 1, 64)


def test_models_without_an_8_bit_form_are_refused():
    import nafezen_models
    from helpers import TINY_A
    from nnis_b200.config import config_from_dict
    from nnis_b200.engine.model import DecoderModel
    cpu = torch.device("cpu")
    llama, other = config_from_dict(TINY_A).to_spec(), config_from_dict(nafezen_models.CONFIGS["mixed"]).to_spec()
    model = DecoderModel(llama, F32, cpu, "int8", "int8")
    assert all(r is None or r.codes for r in model.cache_requests())
    assert not any(r is not None and r.codes for r in DecoderModel(llama, F32, cpu).cache_requests())
    for args, why in ((("int8", None), "no 8-bit cache"), ((None, "int8"), "no 8-bit product")):
        with pytest.raises(ValueError, match=why):
            DecoderModel(other, F32, cpu, *args)
    for args in (("fp8", None), (None, "int4")):
        with pytest.raises(ValueError, match="must be None or 'int8'"):
            DecoderModel(llama, F32, cpu, *args)


def test_pages_that_a_prompt_step_reads_back():
    from nnis_b200.config import config_from_dict
    from nnis_b200.csrc import ops
    from nnis_b200.engine.model import DecoderModel
    from helpers import TINY_A
    spec = config_from_dict(TINY_A).to_spec()
    mixer = DecoderModel(spec, BF16, torch.device("cpu"), "int8").blocks[0].mixer
    few, many = ops.INT8_ROWS_AT_ONCE[BF16], ops.INT8_ROWS_AT_ONCE[BF16] + 1
    name = mixer._read_back_name()
    assert name not in mixer.step_tables([few, 1], [100, 0])
    tables = mixer.step_tables([1, many, 64], [100, 64, 0])
    assert tables[name].tolist() == [[0, 1], [2, 3], [4, -1]] and tables[name + "/pages"].tolist() == [5]
    assert name not in mixer.step_tables([many], [0], tuple(tables))  # (another layer has asked)
    mixer.window = 70
    assert mixer._read_back_table([many, 20], [200, 63])[0].tolist() == [[-1, -1, 0, 1], [2, 3, -1, -1]]


def test_flags_of_the_command_line():
    from nnis_b200.cli.main import UsageError, parse_args
    from nnis_b200.cli.process import ProcessContractError, execute
    base = ["generate", "--model", "m", "--prompt-ids", "1,2"]
    a = parse_args([*base, "--cache-dtype", "int8"])
    assert (a.cache_dtype, a.weight_dtype) == ("int8", None) and parse_args([*base, "--weight-dtype", "int8"]).weight_dtype == "int8"
    for flag in ("--cache-dtype", "--weight-dtype"):
        with pytest.raises(UsageError, match="must be int8"):
            parse_args([*base, flag, "float32"])
    with pytest.raises((ProcessContractError, ValueError)):
        execute("m", prompt_ids=[1], cache_dtype="fp8")


@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_plans_of_attention_cover_every_key(d):
    """Slices cover the table, clusters and tiles are what the kernel takes, and records fit a call's buffer."""
    from nnis_b200.csrc import ops
    for n, seqs in ((1, 1), (7, 7), (64, 64), (80, 16), (300, 300), (5, 400), (3000, 7)):
        for heads, kv_heads in ((9, 3), (32, 32), (20, 1), (64, 1), (16, 2)):
            for cols in (1, 2, 3, 63, 64, 500, 4096):
                for window in (0, 1, 64, 5000):
                    slices, pieces, rows, cluster, eights = ops.attention_int8_plan(n, seqs, heads, kv_heads, d, cols, window, 148)
                    per_page = 1 if d <= 64 else 2
                    assert 1 <= slices <= 64 and slices * pieces >= per_page * cols and (slices - 1) * pieces < per_page * cols
                    assert cluster in (0, 1, 2, 4, 8) and (cluster > 0 or slices == 1) and eights in (1, 2)
                    assert 1 <= rows <= 64 and slices * cluster <= 65535


def test_norms_and_coded_rows_refuse():
    from nnis_b200.csrc import ops
    x, w, codes, scales = empty(3, 20), empty(20), empty(3, 32, dtype=I8), empty(3)
    for args, why in (((x, w, 1e-5, codes, scales, BF16), "CUDA tensors only"), ((x, w, 0.0, codes, scales, BF16), "positive eps"),
                      ((empty(3, 21), empty(21), 1e-5, codes, scales, BF16), "multiple of 4"), ((x, empty(21), 1e-5, codes, scales, BF16), "weight is"),
                      ((x, w, 1e-5, empty(3, 20, dtype=I8), scales, BF16), "codes is"), ((x.to(BF16), w, 1e-5, codes, scales, BF16), "x is")):
        with pytest.raises(ops.KernelError, match=why):
            ops.rmsnorm_int8(*args)
    m, ms = empty(12, 32, dtype=I8), empty(12)
    for args, why in (((codes, scales, 20, m, ms, None, empty(3, 12), 0), "CUDA tensors only"), ((codes, scales, 40, m, ms, None, empty(3, 12), 0), "codes is"),
                      ((codes, empty(4), 20, m, ms, None, empty(3, 12), 0), "scales is"), ((codes, scales, 20, m, ms, empty(11), empty(3, 12), 0), "bias is"),
                      ((codes, scales, 20, m, ms, None, empty(3, 12), 3), "out is"), ((codes, scales, 20, m, ms, None, empty(3, 12, dtype=BF16), 1), "out is"),
                      ((codes, scales, 20, m, ms, None, empty(3, 12), 9), "mode 9")):
        with pytest.raises(ops.KernelError, match=why):
            ops.linear_int8_coded(*args)


@pytest.mark.parametrize("change,why", [
    (dict(window=1 << 31), "a window of 0 or more"), (dict(scale=float("inf")), "a positive scale"), (dict(scale=float("nan")), "a positive scale"),
    (dict(table=empty(2, 0, dtype=I32)), "at least one page"), (dict(table=empty(0, 3, dtype=I32)), "at least one page"),
    (dict(k=empty(0, 2, 64, 64, dtype=I8), v=empty(0, 2, 64, 64, dtype=I8), ks=empty(0, 2, 64), vs=empty(0, 2, 64)), "at least one page")])
def test_attention_without_a_page_or_a_scale_is_refused(change, why, monkeypatch):
    """(with the tensors taken for a GPU's: what is refused for where it lies is refused first)"""
    from nnis_b200.csrc import ops
    monkeypatch.setattr(ops, "_wanted", lambda what, **tensors: None)
    with pytest.raises(ops.KernelError, match=why):
        ops.attention_int8(*attend_args(**change))


@pytest.mark.parametrize("change", [dict(table=empty(2, 0, dtype=I32)),
                                    dict(k=empty(0, 1, 64, 64, dtype=I8), v=empty(0, 1, 64, 64, dtype=I8), ks=empty(0, 1, 64), vs=empty(0, 1, 64))])
def test_writing_without_a_page_is_refused(change):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match="at least one page"):
        ops.rope_store_int8(*store_args(**change))


def test_operands_of_other_ranks_are_refused():
    from nnis_b200.csrc import ops
    for change in (dict(x=empty(5, 1, 40, dtype=BF16)), dict(x=empty(40, dtype=BF16)), dict(w=empty(48, dtype=I8))):
        with pytest.raises(ops.KernelError, match=r"x \[m, k\] and w"):
            ops.linear_int8(*product_args(**change))
    with pytest.raises(ops.KernelError, match=r"codes \[m, width\]"):
        ops.linear_int8_coded(empty(48, dtype=I8), empty(1), 40, empty(12, 48, dtype=I8), empty(12), None, empty(1, 12), ops.STORE)
    with pytest.raises(ops.KernelError, match=r"x \[n, width\]"):
        ops.rmsnorm_int8(empty(64), empty(64), 1e-5, empty(1, 64, dtype=I8), empty(1), BF16)


@pytest.fixture
def reached(monkeypatch):
    """Entries that were reached, with the operators' native checks taking the CPU's tensors for a GPU's and nothing launched."""
    import ctypes
    from nnis_b200.csrc import ops
    calls, lib = [], None
    ops._native("quantize_rows")
    lib = ops._build.load_locked()
    functions = {name: lib.nnis_host_function(ctypes.c_int(0), ctypes.py_object(ops._described(*lines, device_type=1)))
                 for name, lines in ops._CALLS8.items()}
    for name in ops._RECORDS8:
        functions[name] = lambda *values, name=name: calls.append((name, values)) or 0
    monkeypatch.setattr(ops, "_host_functions", functions)
    monkeypatch.setitem(ops._sm_count, 0, 148)
    monkeypatch.setattr(ops, "_status", {0: torch.zeros(1, dtype=I32)})
    return calls


def space():
    from nnis_b200.engine.workspace import Workspace
    return Workspace(torch.device("cpu"))


def coded_args(**change):
    a = dict(codes=empty(5, 48, dtype=I8), scales=empty(5), k=40, w=empty(12, 48, dtype=I8), ws=empty(12), bias=None, out=empty(5, 12, dtype=BF16), mode=0)
    a.update(change)
    return list(a.values())


def test_what_fits_is_passed_on(reached):
    from nnis_b200.csrc import ops
    at = lambda *tensors: tuple(t.data_ptr() for t in tensors)
    qkv, q, pos, seq, table, cos, sin, k, v, ks, vs = a = store_args()[:11]
    ops.rope_store_int8(*store_args(**dict(zip(("qkv", "q", "pos", "seq", "table", "cos", "sin", "k", "v", "ks", "vs"), a))))
    assert reached.pop() == ("nnis_rope_store_int8", (*at(*a), 1, 2, 3, 9, 4, 5, 3, 1, 64, 64, 0))
    ops.rope_store_int8(*store_args(cos=None, sin=None, k=k, qkv=empty(5, 320), q=empty(5, 192)))
    assert reached.pop()[1][5:8] == (0, 0, k.data_ptr())
    k, v, ks, vs, table, local, ko, vo = a = read_args(ko=empty(5, 2, 64, 64), vo=empty(5, 2, 64, 64))
    ops.read_pages_int8(*a)
    assert reached.pop() == ("nnis_read_pages_int8", (*at(*a), 3, 2, 3, 0, 4, 5, 2, 64, 64, 0))
    wide = empty(7, 500, dtype=BF16)
    for queries, stride, page in ((wide[:, 8:392], 500, 64), (wide[:1, 8:392], 999, 64), (empty(5, 384, dtype=BF16), 384, 16)):
        n = min(5, queries.shape[0])
        store = dict(k=empty(4, 2, page, 64, dtype=I8), v=empty(4, 2, page, 64, dtype=I8), ks=empty(4, 2, page), vs=empty(4, 2, page))
        a = attend_args(q=queries, stride=stride, out=empty(n, 384, dtype=BF16), ws=space(), **store)
        ops.attention_int8(*a)
        name, got = reached.pop()
        assert name == "nnis_attention_int8" and got[:5] == at(queries, *a[2:6]) and got[12:22] == (stride, 2, 3, 4, n, 6, 2, 64, page, 0)
        assert got[5:9] == at(a[6], a[7], a[8], a[9]) and got[22] == 0.125 and got[-2:] == (1, 0) and (got[24] > 0) == (page == 64)
    x = empty(5, 50, dtype=BF16)[:, :40]
    for change, want in ((dict(), (50, 5, 12, 40, 0, 1, 148, 0, 0)), (dict(mode=2, out=empty(5, 12)), (50, 5, 12, 40, 2, 1, 148, 0, 0)),
                         (dict(mode=3, out=empty(5, 6, dtype=BF16), bias=empty(12)), (50, 5, 6, 40, 3, 1, 148, 0, 0)),
                         (dict(x=empty(1, 40), out=empty(1, 12)), (40, 1, 12, 40, 0, 0, 148, 0, 0))):
        a = product_args(**{"x": x, "space": space(), **change})
        ops.linear_int8(*a)
        name, got = reached.pop()
        assert name == "nnis_linear_int8" and got[8:] == want and got[:3] == at(a[0], a[1], a[2]) and got[4] == a[4].data_ptr()
        assert got[3] == (a[3].data_ptr() if a[3] is not None else 0) and (got[5] == 0) == (want[1] == 1)
    for change, want in ((dict(), (0, 5, 12, 40, 0, 1, 148, 1, 0)), (dict(mode=1, out=empty(5, 12)), (0, 5, 12, 40, 1, 0, 148, 1, 0))):
        ops.linear_int8_coded(*coded_args(**change))
        assert reached.pop()[1][8:] == want
    ops.quantize_rows(x, empty(5, 48, dtype=I8), empty(5))
    assert reached.pop()[1][3:] == (50, 1, 5, 40, 0)
    ops.rmsnorm_int8(empty(5, 40), empty(40), 1e-5, empty(5, 48, dtype=I8), empty(5), BF16)
    assert reached.pop()[1][4:] == (5, 40, 1, 1e-5, 0)
    ops.linear_int8(*product_args(x=empty(0, 40, dtype=BF16), out=empty(0, 12, dtype=BF16)))
    ops.attention_int8(*attend_args(q=empty(0, 384, dtype=BF16), out=empty(0, 384, dtype=BF16)))
    assert not reached


REFUSED = [("rope_store_int8", store_args, change) for change, _ in test_writing_refuses.pytestmark[0].args[1] if change] + \
    [("read_pages_int8", read_args, change) for change, _ in test_reading_refuses.pytestmark[0].args[1] if change] + \
    [("attention_int8", attend_args, change) for change, _ in test_attention_refuses.pytestmark[0].args[1] if change] + \
    [("attention_int8", attend_args, change) for change, _ in test_attention_without_a_page_or_a_scale_is_refused.pytestmark[0].args[1]] + \
    [("rope_store_int8", store_args, change) for change in test_writing_without_a_page_is_refused.pytestmark[0].args[1]] + \
    [("linear_int8", product_args, change) for change, _ in test_products_refuse.pytestmark[0].args[1] if change] + \
    [("rope_store_int8", store_args, change) for change in (
        dict(cos=None), dict(cos=empty(9, 32).double()), dict(v=empty(4, 1, 64, 64, dtype=I8).transpose(2, 3)), dict(k=None), dict(pos=None),
        dict(heads=2), dict(page=32), dict(table=empty(3, 2, dtype=I32).t()), dict(qkv=[[0.0]]))] + \
    [("read_pages_int8", read_args, change) for change in (
        dict(local=empty(3, 3, dtype=I32)), dict(local=empty(2, 4, dtype=I32)), dict(ko=empty(5, 2, 64, 64)), dict(table=empty(2, 6, dtype=I32)[:, ::2]))] + \
    [("attention_int8", attend_args, change) for change in (
        dict(stride=383), dict(stride=385), dict(heads=5), dict(heads=7), dict(kv_heads=3), dict(window=-1), dict(scale=0.0), dict(scale=-1.0),
        dict(d=32), dict(q=empty(4, 384, dtype=BF16)), dict(q=empty(5, 768, dtype=BF16)[:, ::2], stride=768), dict(pos=empty(4, dtype=I32)),
        dict(out=empty(5, 768, dtype=BF16)[:, :384]), dict(vs=empty(2, 4, 64).transpose(0, 1)))] + \
    [("linear_int8", product_args, change) for change in (
        dict(mode=4), dict(mode=1), dict(mode=3), dict(mode=0.5), dict(w=empty(12, 40, dtype=I8)), dict(w=empty(12, 64, dtype=I8)), dict(bias=empty(11)),
        dict(bias=empty(12, dtype=BF16)), dict(x=empty(40, 5, dtype=BF16).t()), dict(ws=empty(24)[::2]), dict(out=empty(12, 5, dtype=BF16).t()))] + \
    [("linear_int8_coded", coded_args, change) for change in (
        dict(k=0), dict(k=50), dict(k=32), dict(k=133137), dict(mode=1), dict(mode=3), dict(mode=7), dict(codes=empty(5, 64, dtype=I8)),
        dict(scales=empty(6)), dict(out=empty(4, 12, dtype=BF16)), dict(w=empty(12, 48)))]


@pytest.mark.parametrize("name,args,change", REFUSED, ids=[f"{name}-{i}" for i, (name, _, _) in enumerate(REFUSED)])
def test_what_does_not_fit_reaches_no_entry(reached, name, args, change):
    from nnis_b200.csrc import ops
    with pytest.raises((ops.KernelError, AttributeError, TypeError)):
        getattr(ops, name)(*args(**change))
    assert not reached


def test_records_refuse_values_that_are_not_a_field_s():
    """The native caller of an entry: an entry that is not reached cannot fault, so a refusing one is called with no addresses."""
    from nnis_b200.csrc import ops
    call = ops._native("nnis_quantize_rows")
    assert call(0, 0, 0, 1, 1, 1, 1, 0) == -1 == call(0, 0, 0, 1 << 31, 1, 1, 1, 0) == call(0, 0, 0, 1) == call(0, 0, 0, "1", 1, 1, 1, 0)
    assert call(0, 0, 0, 1.5, 1, 1, 1, 0) == -1 == call(0, 0, 0, 1, 1, 1, 1, 0, 0)
    norm = ops._native("nnis_rmsnorm_int8")
    assert norm(0, 0, 0, 0, 1, 8, 1, "x", 0) == -1 == norm(0, 0, 0, 0, 1, 8, 1, 1e-5, 0)


def test_a_matrix_with_too_many_columns_is_refused():
    from nnis_b200.csrc import ops
    from nnis_b200.parts.linear import Int8Matrix
    with pytest.raises(ValueError, match="up to 133136 columns"):
        Int8Matrix.of(empty(1, ops.INT8_LONGEST + 1, dtype=BF16))


def test_entries_refuse_what_has_no_address():
    """Nothing is launched for a tensor without memory, whichever it is."""
    from nnis_b200.csrc import ops
    at = 1 << 20  # (looked at by nobody: an entry that refuses launches nothing)
    for name, places, sizes in (("nnis_rope_store_int8", 11, (0, 1, 1, 1, 1, 1, 1, 1, 64, 64)), ("nnis_read_pages_int8", 8, (1, 1, 1, 0, 1, 1, 1, 64, 64)),
                                ("nnis_attention_int8", 9, (0, 0, 0, 64, 1, 1, 1, 1, 1, 64, 64, 0, 0.5, 1, 0, 0, 0, 0, 0)),
                                ("nnis_quantize_rows", 3, (8, 0, 1, 8)), ("nnis_rmsnorm_int8", 4, (1, 8, 0, 1e-5))):
        for missing in range(places):
            assert ops._native(name)(*(0 if i == missing else at for i in range(places)), *sizes, 0) == -1, (name, missing)
    for missing in (1, 2, 4, 5, 6):
        assert ops._native("nnis_linear_int8")(*(0 if i in (missing, 3, 7) else at for i in range(8)), 0, 1, 16, 16, 0, 0, 148, 1, 0) == -1


def test_angles_of_no_position_write_nothing(reached):
    """Tables without a row have no address, and without an address nothing would be turned: no entry is reached."""
    from nnis_b200.csrc import ops
    ops.rope_store_int8(*store_args(cos=empty(0, 32), sin=empty(0, 32)))
    assert not reached
    with pytest.raises(ops.KernelError):
        ops.rope_store_int8(*store_args(cos=empty(0, 31), sin=empty(0, 31)))


def test_rows_at_any_distance_are_passed_on(reached):
    """Rows that are one row, that overlap, that lie further apart than 31 bits say; the entries take what they are passed."""
    from nnis_b200.csrc import ops
    for distance in (0, 1, 8, 39):
        x = empty(400, dtype=BF16).as_strided((5, 40), (distance, 1))
        ops.quantize_rows(x, empty(5, 48, dtype=I8), empty(5))
        assert reached.pop()[1][3:] == (distance, 1, 5, 40, 0)
        ops.linear_int8(*product_args(x=x, space=space()))
        assert reached.pop()[1][8:] == (distance, 5, 12, 40, 0, 1, 148, 0, 0)
    # (codes at an address that is refused after all else: nothing is launched)
    at = 1 << 20
    for distance in (0, 1, (1 << 31) + 8):
        assert ops._native("nnis_quantize_rows")(at, at + 1, at, distance, 1, 1, 40, 0) == ops._native("nnis_quantize_rows")(at, at + 1, at, 40, 1, 1, 40, 0) != -1
    assert ops._native("nnis_quantize_rows")(at, at, at, -1, 1, 1, 40, 0) == -1


@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_slices_share_what_a_window_shows(d):
    """The pieces that a run of rows can see, wherever its window begins, fall to all slices alike, and to no more of them than the plan has."""
    from nnis_b200.csrc import ops
    length, cut = 64 if d <= 64 else 32, 0
    for n, seqs in ((1, 1), (4, 4), (8, 8), (32, 32), (5, 1), (64, 16)):
        for heads, kv_heads in ((9, 3), (32, 8), (32, 32), (16, 2)):
            for cols in (1, 3, 64, 512, 4096):
                for window in (1, 63, 64, 1000, 4096, 5000):
                    slices, pieces, rows, cluster, _ = ops.attention_int8_plan(n, seqs, heads, kv_heads, d, cols, window, 148)
                    got = ops.attention_int8_slice(slices, pieces, rows, d, window)
                    # (window + rows - 1 keys in a row lie on so many pieces at most; equal parts of them are what a slice can have at best, and
                    # one more piece than there can be may be counted)
                    most = min((window + rows + length - 3) // length + 1, cols * 64 // length)
                    assert slices * got >= most and (slices == 1 or got <= -(-(most + 1) // slices))
                    cut += slices > 1
    assert cut > 20  # (some are cut)


def test_a_step_reads_back_what_long_sequences_have(monkeypatch):
    """Beside a prompt, sequences with few tokens and long contexts read the codes: their pages are not read back, no kernel of prompts has
    work for them, and their rows are named.  The bytes read back are bounded by that."""
    from nnis_b200.config import config_from_dict
    from nnis_b200.csrc import ops
    from nnis_b200.engine.model import DecoderModel
    from helpers import TINY_A
    spec = config_from_dict(TINY_A).to_spec()
    for dtype, many in ((BF16, 33), (F32, 65)):
        mixer = DecoderModel(spec, dtype, torch.device("cpu"), "int8").blocks[0].mixer
        name = mixer._read_back_name()
        counts, starts = [1, 5, many, 1, 200, 1], [500, 90, 0, 64, 130, 4000]
        both = mixer.step_tables(counts, starts)
        assert name + "/codes" not in both and both[name + "/pages"].tolist() == [8 + 2 + -(-many // 64) + 2 + 6 + 63]
        monkeypatch.setattr(ops, "INT8_READ_BACK", 0)
        tables = mixer.step_tables(counts, starts)
        assert tables[name + "/pages"].tolist() == [-(-many // 64) + 6] and tables[name].shape[1] == 6
        assert [row for row, line in enumerate(tables[name].tolist()) if max(line) >= 0] == [2, 4]
        assert tables[name + "/codes"].tolist() == [[0, 6], [6 + many, 7 + many], [207 + many, 208 + many]]
        for key in tables:
            if key.endswith("/units") or key == mixer.TILES_64 or key.startswith("prefill_f32"):
                assert set(tables[key][:, 0].tolist()) == {2, 4}
        assert set(mixer.step_tables(counts, starts, tuple(tables))) <= set(tables) - {name, name + "/pages", name + "/codes"}
        # contexts of few tokens that are no longer than the others' go with them
        assert name + "/codes" not in mixer.step_tables([1, many, 300], [100, 64, 1])
        monkeypatch.undo()
        # a server's step: 63 contexts of 4,000 and a prompt of 200 tokens, a layer of 32 heads of 64
        mixer.widest_row = 2048
        tables = mixer.step_tables([1] * 63 + [200], [4000] * 63 + [0])
        assert tables[name + "/pages"].tolist() == [4] and tables[name + "/codes"].tolist() == [[0, 63]]


def test_scratch_that_steps_lend_one_another():
    from nnis_b200.engine.workspace import Workspace
    own = Workspace(torch.device("cpu"))
    first, second, other = (Workspace(torch.device("cpu"), beside=own) for _ in range(3))
    a = first.lent("k", (3, 4), F32)
    first.frozen = True
    assert own.lent("k", (2, 4), F32).data_ptr() == a.data_ptr() == second.lent("k", (12,), F32).data_ptr() != second.get("k", (12,), F32).data_ptr()
    larger = second.lent("k", (13,), F32)  # (the first keeps what its graph holds)
    assert larger.data_ptr() != a.data_ptr() == first.lent("k", (12,), F32).data_ptr() and larger.data_ptr() == other.lent("k", (5,), F32).data_ptr()
    with pytest.raises(RuntimeError, match="would move"):
        first.lent("k", (13,), F32)
    assert own.lent("k", (13,), F32).data_ptr() == larger.data_ptr() and own.lent("k", (1,), BF16).dtype == BF16


def test_tensors_are_read_when_they_are_asked_for(tmp_path):
    """By file and role as the loader keeps them; what is still held is given out again, what nobody holds is read anew."""
    from helpers import TINY_A, make_model
    from nnis_b200.config import read_config
    from nnis_b200.engine.model import DecoderModel
    from nnis_b200.weights import TensorsOnDemand, WeightError, load_weights, open_weights
    made = make_model(str(tmp_path / "m"), TINY_A, 3)
    wanted = DecoderModel.weight_specs_of(read_config(made).to_spec())
    for dtype in (F32, BF16):
        eager = load_weights(made, wanted, dtype, torch.device("cpu"))
        with open_weights(made, wanted, dtype, torch.device("cpu")) as tensors:
            assert isinstance(tensors, TensorsOnDemand) and set(tensors) == set(eager) and len(tensors) == len(eager)
            for name, t in eager.items():
                assert tensors[name].dtype == t.dtype and torch.equal(tensors[name], t)
    reads = []
    lazy = TensorsOnDemand(wanted, lambda name: (reads.append(name), eager[name].clone())[1], BF16, torch.device("cpu"))
    name = next(n for n, w in wanted.items() if w.role == "matrix")
    held = lazy[name]
    assert lazy[name] is held and reads == [name]
    del held
    assert torch.equal(lazy[name], eager[name]) and reads == [name] * 2
    with pytest.raises(WeightError, match="missing"):
        with open_weights(made, {**wanted, "more": wanted[name]}, BF16, torch.device("cpu")):
            pass


def test_blocks_are_put_into_codes_one_after_another(monkeypatch):
    """A model in 8 bits holds the matrices of one block, at most, in 16."""
    import weakref
    from helpers import TINY_A
    from nnis_b200.config import config_from_dict
    from nnis_b200.csrc import ops
    from nnis_b200.engine.model import DecoderModel
    from nnis_b200.weights import TensorsOnDemand
    spec = config_from_dict({**TINY_A, "num_hidden_layers": 6}).to_spec()
    model = DecoderModel(spec, BF16, torch.device("cpu"), None, "int8")
    wanted, given, most, done = model.weight_specs(), [], [0], []
    monkeypatch.setattr(ops, "quantize_rows", lambda x, codes, scales: done.append(tuple(x.shape)))
    blocks = {n for n, w in wanted.items() if w.role == "matrix" and ".layers." in n}

    def read(name):
        t = torch.zeros(wanted[name].shape)
        if name in blocks:
            most[0] = max(most[0], 1 + sum(r() is not None for r in given))
        return t

    lazy = TensorsOnDemand(wanted, read, BF16, torch.device("cpu"))
    real = TensorsOnDemand.__getitem__
    monkeypatch.setattr(TensorsOnDemand, "__getitem__", lambda self, name: (lambda t: (given.append(weakref.ref(t)) if name in blocks else None, t)[1])(real(self, name)))
    model.load(lazy)
    assert most[0] <= len(blocks) // 6 and len(done) == 6 * 4  # (q, k, v in one; gate and up in one)
