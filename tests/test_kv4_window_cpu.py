"""Refusals of the 4-bit cache's and of windowed attention's entry points, on
the host: sizes, shapes, alignment and null pointers come back as statuses
before any device work (the pointers are never followed), wrong tensors raise
ValueError in the torch front end."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
OK, ARG, UNSUPPORTED = 0, -1, -2


def call(name, null=(), **values):
    """The entry point with valid-looking arguments but for those given."""
    from cache_eviction_b200 import capi
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "ce_api.h").read_text(), flags=re.S)
    params = re.search(r"\b" + name + r"\s*\(([^)]*)\)\s*;", text).group(1).split(",")
    default = dict(bs=1, num_q_heads=64, num_kv_heads=8, head_dim=64, page_size=16, pool_units=4, kv_capacity=4,
                   tokens=1, num_units=1, window=8, first=0, total_q=1, max_q=1, max_tokens=16, num_rows=1, layers=1, kv_heads=8,
                   table_width=16, r2u_width=16, pos_cap=16, max_cols=16, max_n=16, live=1, epoch=1,
                   workspace_bytes=1 << 40, hazard_bytes=1 << 20, score_sg=4,
                   q_sb=4096, q_sh=64, q_st=4096, o_sb=4096, o_sh=64, o_st=4096)
    args = []
    for p in params:
        key = re.findall(r"\w+", p)[-1]
        if key in values:
            x = values[key]
            args.append(C.c_void_p(x) if "*" in p else x)
        elif "*" in p:
            optional = key in ("err", "stream", "lse_out", "sinks", "rows", "mode_of_row", "swa_mapping", "uniforms",
                               "global_scores", "record_delta", "record_counts")
            args.append(None if key in null or optional else C.c_void_p(4096))
        elif "float" in p:
            args.append(0.125)
        else:
            args.append(default.get(key, 64 if re.search(r"_(st|sg|ou|og|ot)$", key) or "stride" in key else 0))
    status = getattr(capi.load(), name)(*args)
    return status, capi.load().ce_last_error().decode()


NAN, INF = float("nan"), float("inf")
REFUSALS = [
    ("ce_kv4_write", dict(tokens=-1), ARG), ("ce_kv4_write", dict(num_kv_heads=0), ARG),
    ("ce_kv4_write", dict(head_dim=128), UNSUPPORTED), ("ce_kv4_write", dict(page_size=1), UNSUPPORTED),
    ("ce_kv4_write", dict(k_st=60), ARG), ("ce_kv4_write", dict(v_sg=4), ARG), ("ce_kv4_write", dict(k=4104), ARG),
    ("ce_kv4_write", dict(v_pool=4100), ARG), ("ce_kv4_write", dict(pool_units=-1), ARG),
    ("ce_kv4_read", dict(num_units=-1), ARG), ("ce_kv4_read", dict(head_dim=32), UNSUPPORTED),
    ("ce_kv4_read", dict(page_size=32), UNSUPPORTED), ("ce_kv4_read", dict(k_ot=68), ARG),
    ("ce_kv4_read", dict(v_out=4098), ARG), ("ce_kv4_read", dict(k_pool=4097), ARG),
    ("ce_kv4_decode_attn_score", dict(bs=-1), ARG), ("ce_kv4_decode_attn_score", dict(head_dim=128), UNSUPPORTED),
    ("ce_kv4_decode_attn_score", dict(num_q_heads=32), UNSUPPORTED),
    ("ce_kv4_decode_attn_score", dict(num_q_heads=24, num_kv_heads=3), UNSUPPORTED),
    ("ce_kv4_decode_attn_score", dict(page_size=1), UNSUPPORTED), ("ce_kv4_decode_attn_score", dict(sm_scale=0.0), ARG),
    ("ce_kv4_decode_attn_score", dict(sm_scale=-1.0), ARG), ("ce_kv4_decode_attn_score", dict(sm_scale=NAN), ARG),
    ("ce_kv4_decode_attn_score", dict(pool_units=0), ARG), ("ce_kv4_decode_attn_score", dict(q_sh=65), ARG),
    ("ce_kv4_decode_attn_score", dict(q=4098), ARG), ("ce_kv4_decode_attn_score", dict(k_pool=4104), ARG),
    ("ce_kv4_decode_attn_score", dict(mode_of_row=4096, score_sg=3), ARG),
    ("ce_kv4_boundary", dict(page_size=1), UNSUPPORTED), ("ce_kv4_boundary", dict(head_dim=32), UNSUPPORTED),
    ("ce_kv4_boundary", dict(epoch=0), ARG),
    ("ce_window_decode", dict(window=0), ARG), ("ce_window_decode", dict(window=-2), ARG),
    ("ce_window_decode", dict(first=-1), ARG), ("ce_window_decode", dict(q=4098), ARG),
    ("ce_window_decode", dict(num_q_heads=56), UNSUPPORTED), ("ce_window_decode", dict(page_size=8), UNSUPPORTED),
    ("ce_window_decode", dict(page_size=1, num_q_heads=32, num_kv_heads=4), UNSUPPORTED),
    ("ce_window_decode", dict(head_dim=80), UNSUPPORTED), ("ce_window_decode", dict(q_sh=63), ARG),
    ("ce_window_prefill", dict(window=0), ARG), ("ce_window_prefill", dict(window=-3), ARG),
    ("ce_window_prefill", dict(first=-1), ARG), ("ce_window_prefill", dict(sm_scale=0.0), ARG),
    ("ce_window_prefill", dict(total_q=-1), ARG), ("ce_window_prefill", dict(max_tokens=-1), ARG),
    ("ce_window_prefill", dict(max_tokens=2 ** 31 - 1), UNSUPPORTED), ("ce_window_prefill", dict(bs=65536), UNSUPPORTED),
    ("ce_window_prefill", dict(head_dim=128), UNSUPPORTED), ("ce_window_prefill", dict(num_q_heads=8), UNSUPPORTED),
    ("ce_window_prefill", dict(page_size=128), UNSUPPORTED), ("ce_window_prefill", dict(page_size=24), UNSUPPORTED),
    ("ce_window_prefill", dict(pool_units=1 << 26), UNSUPPORTED), ("ce_window_prefill", dict(pool_units=0), ARG),
    ("ce_window_prefill", dict(q_st=2048), ARG), ("ce_window_prefill", dict(q_sh=68), ARG),
    ("ce_window_prefill", dict(o_st=4100), ARG), ("ce_window_prefill", dict(out=4104), ARG),
    ("ce_window_prefill", dict(v_pool=4100), ARG),
]


@pytest.mark.parametrize("name,values,want", REFUSALS, ids=[f"{n}-{v}" for n, v, _ in REFUSALS])
def test_refused_on_the_host(name, values, want):
    status, message = call(name, **values)
    assert status == want and message


@pytest.mark.parametrize("name,pointers", [
    ("ce_kv4_write", ["k", "v", "loc", "k_pool", "v_pool"]),
    ("ce_kv4_read", ["k_pool", "v_pool", "units", "k_out", "v_out"]),
    ("ce_kv4_decode_attn_score", ["q", "k_pool", "v_pool", "kv_indptr", "kv_indices", "kv_tokens", "out", "workspace"]),
    ("ce_window_decode", ["q", "k_pool", "v_pool", "kv_indptr", "kv_indices", "kv_tokens", "out", "workspace"]),
    ("ce_window_prefill", ["q", "k_pool", "v_pool", "qo_indptr", "kv_indptr", "kv_indices", "kv_tokens", "out"])])
def test_null_pointers_are_refused(name, pointers):
    for p in pointers:
        assert call(name, null=(p,))[0] == ARG, p


def test_empty_calls_do_nothing():
    assert call("ce_kv4_write", tokens=0)[0] == OK
    assert call("ce_kv4_read", num_units=0)[0] == OK
    assert call("ce_kv4_decode_attn_score", bs=0)[0] == OK
    assert call("ce_window_decode", bs=0)[0] == OK
    for none in (dict(bs=0), dict(max_q=0), dict(total_q=0)):
        assert call("ce_window_prefill", **none)[0] == OK
    assert call("ce_kv4_boundary", num_rows=0)[0] == OK


def test_workspace_queries():
    from cache_eviction_b200 import capi
    lib = capi.load()
    assert lib.ce_kv4_decode_workspace_bytes(-1, 1, 64, 8, 0) == -1
    assert lib.ce_kv4_decode_workspace_bytes(1, -1, 64, 8, 0) == -1
    four = lib.ce_kv4_boundary_workspace_bytes(32, 2, 8, 64, 16, 4096, 0, 0)
    assert 0 < four < lib.ce_boundary_workspace_bytes(32, 2, 8, 64, 16, 4096, 0, 0, 0)   # smaller pages to stage
    assert lib.ce_kv4_boundary_workspace_bytes(32, 2, 8, 64, 1, 4096, 0, 0) == -1        # 16-token pages only


def test_front_end_raises_on_wrong_tensors():
    from cache_eviction_b200 import kernels
    i32 = dict(dtype=torch.int32)
    pool = kernels.kv4_pool(4, 8, "cpu")
    rows = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    loc = torch.zeros(3, dtype=torch.int64)
    csr = (torch.zeros(2, **i32), torch.zeros(4, **i32), torch.zeros(1, **i32))
    q = torch.zeros((1, 64, 64), dtype=torch.bfloat16)
    bf = torch.zeros((4, 8, 16, 64), dtype=torch.bfloat16)
    wrong = [
        lambda: kernels.kv4_write(rows.float(), rows, pool, pool, loc),
        lambda: kernels.kv4_write(rows[:, :4], rows[:, :4], pool, pool, loc),
        lambda: kernels.kv4_write(rows, rows, pool, pool, loc.int()),
        lambda: kernels.kv4_write(rows, rows, pool, pool, loc[:2]),
        lambda: kernels.kv4_write(rows, rows, pool[:, :, :512], pool[:, :, :512], loc),
        lambda: kernels.kv4_write(rows, rows, pool, pool, loc),                        # not on a GPU
        lambda: kernels.kv4_read(pool, pool, loc),
        lambda: kernels.kv4_read(pool, pool, csr[1], k_out=rows),
        lambda: kernels.kv4_read(pool, pool[:2], csr[1]),
        lambda: kernels.kv4_decode_attn_score(q.float(), pool, pool, *csr, 0.125),
        lambda: kernels.kv4_decode_attn_score(q, bf, bf, *csr, 0.125),
        lambda: kernels.kv4_decode_attn_score(q, pool, pool, csr[0].long(), *csr[1:], 0.125),
        lambda: kernels.kv4_decode_attn_score(q, pool, pool, csr[0][:1], *csr[1:], 0.125),
        lambda: kernels.kv4_decode_attn_score(q, pool, pool, *csr, 0.125, out=q.float()),
        lambda: kernels.kv4_decode_attn_score(q, pool, pool, *csr, 0.125, scores=torch.zeros(8, 3)),
        lambda: kernels.kv4_decode_attn_score(q, pool, pool, *csr, 0.125, score_flags=7),
        lambda: kernels.window_decode(q, bf, bf, *csr, 0.125, 1, 8),
        lambda: kernels.window_decode(q, bf, bf[:2], *csr, 0.125, 16, 8),
        lambda: kernels.window_decode(q, bf, bf, *csr, 0.125, 16, 8, out=q[:, :32]),
        lambda: kernels.window_decode(q, bf, bf, *csr, 0.125, 16, 8, lse=torch.zeros(3)),
        lambda: kernels.window_decode(q, bf, bf, *csr, 0.125, 16, 8),                  # not on a GPU
        lambda: kernels.window_prefill(q, bf, bf, csr[0].long(), *csr, 0.125, 16, 1, 1, 8),
        lambda: kernels.window_prefill(q, bf, bf, csr[0][:1], *csr, 0.125, 16, 1, 1, 8),
        lambda: kernels.window_prefill(q[0], bf, bf, csr[0], *csr, 0.125, 16, 1, 1, 8),
        lambda: kernels.window_prefill(q, bf, bf, csr[0], *csr, 0.125, 16, 1, 1, 8, out=q.half()),
        lambda: kernels.window_prefill(q, bf, bf, csr[0], *csr, 0.125, 16, 1, 1, 8),   # not on a GPU
    ]
    for i, f in enumerate(wrong):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
