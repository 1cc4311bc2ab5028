"""No-GPU checks of the paged-cache operators: what the library and the Python layer refuse, and the frequencies."""

import math

import pytest
import torch


@pytest.fixture(scope="module")
def native():
    from dram_attention_b200 import _native, build
    build.build()
    return _native


ROTATE = ["q", "k", "q_out", "k_out", "qs0", "qs1", "qs2", "ks0", "ks1", "ks2", "positions", "positions_64", "ps0", "ps1",
          "inv_freq", "rotary_dim", "interleaved", "transposed", "factor", "n_batch", "n_tokens", "n_q_heads", "n_kv_heads",
          "head_dim", "dtype", "stream"]
APPEND = ["q", "k", "v", "q_out", "qs0", "qs1", "ks0", "ks1", "vs0", "vs1", "pages", "page_stride", "page_head_stride",
          "page_size", "n_pages", "page_table", "table_stride", "table_columns", "lengths", "starts", "n_sequences", "n_rows",
          "inv_freq", "rotary_dim", "interleaved", "factor", "n_q_heads", "n_kv_heads", "head_dim", "dtype", "status", "stream"]
ATTEND = ["q", "qs0", "qs1", "pages", "page_stride", "page_head_stride", "page_size", "n_pages", "page_table", "table_stride",
          "table_columns", "lengths", "n_sequences", "window", "scale", "out", "lse", "workspace", "workspace_bytes", "status",
          "n_kv_heads", "rep", "head_dim", "dtype", "stream"]

ROTATE_OK = dict(q=256, k=256, q_out=256, k_out=256, positions=256, inv_freq=256, rotary_dim=64, factor=1.0, n_batch=1,
                 n_tokens=4, n_q_heads=8, n_kv_heads=2, head_dim=64, dtype=2)
APPEND_OK = dict(q=256, k=256, v=256, q_out=256, pages=256, page_size=16, n_pages=8, page_table=256, table_columns=4,
                 lengths=256, starts=256, n_sequences=2, n_rows=4, inv_freq=256, rotary_dim=64, factor=1.0, n_q_heads=8,
                 n_kv_heads=2, head_dim=64, dtype=2, status=256)
ATTEND_OK = dict(q=256, pages=256, page_size=16, n_pages=8, page_table=256, table_columns=4, lengths=256, n_sequences=2,
                 scale=0.1, out=256, workspace=256, workspace_bytes=1 << 30, status=256, n_kv_heads=2, rep=4, head_dim=64,
                 dtype=2)


def _call(native, which, fields, ok, **changes):
    values = {**dict.fromkeys(fields, 0), **ok, **changes}
    pack = {"da_rotate": native.PACK_ROTATE, "da_append_pages": native.PACK_APPEND, "da_paged_attention": native.PACK_ATTEND}
    return getattr(native.lib(), which)(pack[which](*(values[f] for f in fields)))


NULL, SHAPE, DTYPE, ALIGN, UNSUPPORTED, WORKSPACE = -1, -2, -3, -4, -5, -6


@pytest.mark.parametrize("changes,code", [
    (dict(q=0, k=0), NULL), (dict(positions=0), NULL), (dict(inv_freq=0), NULL), (dict(q_out=0), NULL), (dict(k_out=0), NULL),
    (dict(dtype=3), DTYPE), (dict(dtype=-1), DTYPE), (dict(rotary_dim=63), SHAPE), (dict(rotary_dim=66), SHAPE),
    (dict(rotary_dim=0), SHAPE), (dict(head_dim=1024, rotary_dim=64), SHAPE), (dict(n_tokens=0), SHAPE), (dict(n_batch=0), SHAPE),
    (dict(n_batch=1 << 20, n_tokens=1 << 20), SHAPE), (dict(n_q_heads=0), SHAPE), (dict(n_kv_heads=-1), SHAPE),
    (dict(q=257), ALIGN), (dict(positions=258), ALIGN), (dict(positions=260, positions_64=1), ALIGN), (dict(inv_freq=254), ALIGN),
])
def test_rotate_refuses(native, changes, code):
    assert _call(native, "da_rotate", ROTATE, ROTATE_OK, **changes) == code


@pytest.mark.parametrize("changes,code", [
    (dict(k=0), NULL), (dict(v=0), NULL), (dict(pages=0), NULL), (dict(page_table=0), NULL), (dict(lengths=0), NULL),
    (dict(status=0), NULL), (dict(q_out=0), NULL), (dict(inv_freq=0), NULL), (dict(dtype=5), DTYPE), (dict(starts=0), SHAPE),
    (dict(n_rows=0), SHAPE), (dict(n_sequences=0), SHAPE), (dict(page_size=0), SHAPE), (dict(n_pages=0), SHAPE),
    (dict(table_columns=0), SHAPE), (dict(table_columns=1 << 28), SHAPE), (dict(rotary_dim=65), SHAPE), (dict(rotary_dim=80), SHAPE),
    (dict(n_kv_heads=0), SHAPE), (dict(n_q_heads=0), SHAPE), (dict(head_dim=0), SHAPE), (dict(pages=255), ALIGN),
    (dict(page_table=254), ALIGN), (dict(starts=255), ALIGN), (dict(status=2), ALIGN),
])
def test_append_refuses(native, changes, code):
    assert _call(native, "da_append_pages", APPEND, APPEND_OK, **changes) == code


@pytest.mark.parametrize("changes,code", [
    (dict(q=0), NULL), (dict(pages=0), NULL), (dict(page_table=0), NULL), (dict(lengths=0), NULL), (dict(out=0), NULL),
    (dict(workspace=0), NULL), (dict(status=0), NULL), (dict(dtype=3), DTYPE), (dict(head_dim=72), UNSUPPORTED),
    (dict(head_dim=512), UNSUPPORTED), (dict(rep=257), UNSUPPORTED), (dict(rep=0), SHAPE), (dict(n_sequences=0), SHAPE),
    (dict(window=-1), SHAPE), (dict(page_size=0), SHAPE), (dict(table_columns=0), SHAPE), (dict(table_columns=1 << 28), SHAPE),
    (dict(q=264), ALIGN), (dict(qs0=4), ALIGN), (dict(page_stride=4), ALIGN), (dict(page_head_stride=12), ALIGN),
    (dict(lse=258), ALIGN), (dict(workspace=8), ALIGN), (dict(n_sequences=1 << 30, n_kv_heads=8), SHAPE),
])
def test_attend_refuses(native, changes, code):
    assert _call(native, "da_paged_attention", ATTEND, ATTEND_OK, **changes) == code


@pytest.mark.parametrize("rep,d,dtype", [(1, 64, 2), (4, 128, 1), (16, 128, 2), (17, 256, 2), (5, 80, 0), (256, 96, 0)])
def test_attend_workspace_has_to_be_as_large_as_stated(native, rep, d, dtype):
    need = native.lib().da_paged_attention_workspace_bytes(2, 2, rep, d, dtype)
    assert need > 0 and native.lib().da_paged_attention_workspace_bytes(200, 2, rep, d, dtype) > need
    assert _call(native, "da_paged_attention", ATTEND, ATTEND_OK, rep=rep, head_dim=d, dtype=dtype, workspace_bytes=need - 1) == WORKSPACE
    for bad in ((2, 2, 0, 64, 2), (2, 2, 257, 64, 2), (2, 2, 4, 72, 2), (2, 2, 4, 64, 3), (2, 2, -1, 64, 0), (0, 2, 4, 64, 0), (2, 0, 4, 64, 0)):
        assert native.lib().da_paged_attention_workspace_bytes(*bad) == 0


def test_null_argument_blocks_are_refused(native):
    for name in ("da_rotate", "da_append_pages", "da_paged_attention"):
        assert getattr(native.lib(), name)(None) == NULL


def test_classes_refuse_cpu_tensors_and_bad_pools(native):
    import dram_attention_b200 as da
    with pytest.raises(RuntimeError, match="CUDA"):
        da.Rotary(torch.ones(4))
    with pytest.raises(RuntimeError, match="CUDA"):
        da.PagedKVCache(2, 16, 1, 64, device="cpu")
    with pytest.raises(AssertionError, match="head_dim"):
        da.PagedKVCache(2, 16, 1, 72, device="cpu")
    with pytest.raises(TypeError, match="dtype"):
        da.PagedKVCache(2, 16, 1, 64, device="cpu", dtype=torch.float64)
    with pytest.raises(AssertionError, match="pages must be"):
        da.PagedKVCache.over(torch.zeros(2, 16, 1, 64))


# ---- frequencies ---------------------------------------------------------------------------

def _freq(*a, **k):
    from dram_attention_b200 import rotary_frequencies
    f, amplitude = rotary_frequencies(*a, device="cpu", **k)
    assert f.dtype == torch.float32
    return f.double(), amplitude


def test_plain_and_linear_frequencies():
    f, a = _freq(8, 10000.0)
    want = torch.tensor([10000.0 ** (-2 * i / 8) for i in range(4)], dtype=torch.float64)
    assert a == 1.0 and bool(((f - want).abs() <= want * 2.0 ** -24).all())
    g, a = _freq(8, 10000.0, {"type": "linear", "factor": 4.0})
    assert a == 1.0 and torch.equal(g, f / 4)


def test_ntk_keeps_the_fastest_pair_and_slows_the_slowest_by_the_factor():
    f, _ = _freq(64, 10000.0)
    g, a = _freq(64, 10000.0, {"type": "ntk", "factor": 8.0})
    assert a == 1.0 and g[0] == f[0] == 1.0
    assert math.isclose(float(f[-1] / g[-1]), 8.0, rel_tol=2.0 ** -22)


def test_llama3_scaling_by_turns():
    n, factor = 8192, 8.0
    f, _ = _freq(128, 500000.0)
    g, a = _freq(128, 500000.0, {"type": "llama3", "factor": factor, "original_length": n, "low": 1.0, "high": 4.0})
    assert a == 1.0
    for x, y in zip(f.tolist(), g.tolist()):
        wavelength = 2 * math.pi / x
        if wavelength < n / 4.0:
            want = x
        elif wavelength > n:
            want = x / factor
        else:
            smooth = (n / wavelength - 1.0) / 3.0
            want = (1 - smooth) * x / factor + smooth * x
        assert math.isclose(y, want, rel_tol=1e-6)


def test_yarn_scaling_and_amplitude():
    n, factor, base, d = 4096, 16.0, 10000.0, 128
    f, _ = _freq(d, base)
    g, a = _freq(d, base, {"type": "yarn", "factor": factor, "original_length": n})
    assert math.isclose(a, 0.1 * math.log(factor) + 1)
    turns = n * f / (2 * math.pi)
    assert torch.equal(g[turns > 40], f[turns > 40])                    # fast pairs as they were
    slow = turns < 0.8
    assert bool(((g[slow] * factor - f[slow]).abs() <= f[slow] * 1e-6).all())
    assert bool((g <= f * (1 + 1e-6)).all()) and bool((g >= f / factor * (1 - 1e-6)).all())
    _, a = _freq(d, base, {"type": "yarn", "factor": factor, "original_length": n, "attention_factor": 1.25})
    assert a == 1.25


@pytest.mark.parametrize("scaling", [
    {"type": "spiral", "factor": 2.0}, {"type": "linear", "factor": 0.0}, {"type": "linear", "factor": 2.0, "low": 1.0},
    {"type": "llama3", "factor": 2.0, "original_length": 100, "low": 4.0, "high": 1.0},
    {"type": "yarn", "factor": 2.0, "original_length": 100, "fast": 1.0, "slow": 2.0}])
def test_frequencies_refuse(scaling):
    with pytest.raises(AssertionError):
        _freq(16, 10000.0, scaling)
    with pytest.raises(AssertionError):
        _freq(7)
