"""What node_attention, dropout_add and action_log_probs refuse, in Python and
behind the C boundary, and their argument blocks' layout.  No GPU."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from conftest import ROOT


def test_layout_matches_header(tmp_path):
    from trafficrl import _lib
    lines, structs = [], (("trx_node_attention_args", _lib.TrxNodeAttentionArgs),
                          ("trx_action_log_probs_args", _lib.TrxActionLogProbsArgs))
    for cname, cls in structs:
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        lines += [f'printf("%zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    lines.append('printf("%d %d\\n", TRX_ATT_MAX_CHANNELS, TRX_TOP_MAX);')
    src = tmp_path / "probe.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"trafficrl.h\"\nint main(){" + "".join(lines)
                   + "return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "probe")])
    vals = list(map(int, subprocess.check_output([str(tmp_path / "probe")]).split()))
    want = []
    for _, cls in structs:
        want += [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert vals == want + [_lib.ATT_MAX_CHANNELS, _lib.TOP_MAX]


def _qkv(rows=6, H=4, Hk=2, C=32, dt=torch.float32, nodes=None):
    nodes = rows if nodes is None else nodes
    return torch.zeros(rows, H, C, dtype=dt), torch.zeros(nodes, Hk, C, dtype=dt), torch.zeros(nodes, Hk, C, dtype=dt)


P = torch.tensor([0, 2, 6])


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(6, 128)), dict(q=torch.zeros(6, 4, 32, dtype=torch.float64)),
    dict(k=torch.zeros(6, 2, 32, dtype=torch.bfloat16)), dict(v=torch.zeros(6, 2, 64)), dict(k=torch.zeros(6, 3, 32)),
    dict(ptr=P.int()), dict(ptr=P.view(1, 3)), dict(ptr=P[:0]), dict(k_ptr=torch.tensor([0, 6])),
    dict(dist=torch.zeros(6, 6, dtype=torch.float64)), dict(dist=torch.zeros(3, 6, 6)), dict(dist=torch.zeros(36)),
    dict(dist=torch.zeros(6, 6, requires_grad=True)), dict(slope=torch.zeros(4)),
    dict(dist=torch.zeros(6, 6), slope=torch.zeros(3)), dict(dist=torch.zeros(6, 6), slope=torch.zeros(4).double()),
    dict(scale=math.nan), dict(scale=math.inf), dict(cap=-1.0), dict(cap=math.inf), dict(cap=1e-35), dict(max_nodes=-1),
], ids=lambda c: ",".join(c))
def test_node_attention_refuses(change):
    from trafficrl.models import node_attention
    q, k, v = _qkv()
    a = dict(q=q, k=k, v=v, ptr=P) | change
    with pytest.raises(ValueError, match="node_attention"):
        node_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("ptr"), **a)


@pytest.mark.parametrize("C", [0, 4, 12, 136])
def test_node_attention_refuses_channels(C):
    from trafficrl.models import node_attention
    with pytest.raises(ValueError, match="channels"):
        node_attention(*_qkv(C=C), P)


def test_no_cpu_fallback():
    from trafficrl.models import dropout_add, node_attention
    from trafficrl.rl import action_log_probs
    with pytest.raises(ValueError, match="HIP device"):
        node_attention(*_qkv(), P)
    with pytest.raises(ValueError, match="k_ptr"):
        node_attention(*_qkv(nodes=9), P)
    with pytest.raises(ValueError, match="HIP device"):
        dropout_add(torch.zeros(4), torch.zeros(2, dtype=torch.int64), 0.5)
    with pytest.raises(ValueError, match="HIP device"):
        action_log_probs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="tensors on"):
        dropout_add(torch.zeros(4), torch.zeros(2, dtype=torch.int64, device="meta"), 0.5)


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(4, dtype=torch.float64)), dict(x=torch.zeros(4, dtype=torch.int32)), dict(p=-0.1), dict(p=1.0),
    dict(p=0.999999), dict(p=math.nan), dict(rng=torch.zeros(2)), dict(rng=torch.zeros(3, dtype=torch.int64)),
    dict(residual=torch.zeros(5)), dict(residual=torch.zeros(4, dtype=torch.bfloat16)), dict(site=-1),
    dict(site=2 ** 32)], ids=lambda c: ",".join(c))
def test_dropout_add_refuses(change):
    from trafficrl.models import dropout_add
    a = dict(x=torch.zeros(4), rng=torch.zeros(2, dtype=torch.int64), p=0.5) | change
    with pytest.raises(ValueError, match="dropout_add"):
        dropout_add(a.pop("x"), a.pop("rng"), a.pop("p"), **a)


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(2, 5, dtype=torch.float64)), dict(logits=torch.zeros(2, 5, 1)), dict(logits=torch.zeros(10)),
    dict(row_ptr=torch.tensor([0, 5, 10])), dict(logits=torch.zeros(10), row_ptr=torch.tensor([0, 5, 10]).int()),
    dict(action=torch.zeros(3, dtype=torch.int64)), dict(action=torch.zeros(2)), dict(mask=torch.zeros(2, 4)),
    dict(top_k=17), dict(top_k=-1), dict(max_row=-1)], ids=lambda c: ",".join(c))
def test_action_log_probs_refuses(change):
    from trafficrl.rl import action_log_probs
    a = dict(logits=torch.zeros(2, 5), action=torch.zeros(2, dtype=torch.int64)) | change
    with pytest.raises(ValueError, match="action_log_probs"):
        action_log_probs(a.pop("logits"), a.pop("action"), **a)


def _attention_args():
    from trafficrl import _lib
    a = _lib.TrxNodeAttentionArgs()
    a.num_graphs, a.heads, a.kv_heads, a.channels, a.scale = 1, 4, 2, 32, 1.0
    a.num_queries = a.num_nodes = a.max_queries = a.max_nodes = 8
    for f in ("q", "k", "v", "q_ptr", "k_ptr", "out", "lse", "grad_out", "grad_q", "grad_k", "grad_v", "workspace"):
        setattr(a, f, 4096)      # never dereferenced: every case is refused first
    a.q_row, a.q_head, a.k_row, a.k_head, a.v_row, a.v_head = 128, 32, 64, 32, 64, 32
    a.workspace_bytes = 1 << 40
    return a


@pytest.mark.parametrize("field,value,code", [
    ("num_graphs", -1, -1), ("num_queries", -1, -1), ("num_nodes", 1 << 31, -3), ("dtype", 3, -1), ("kv_heads", 3, -1),
    ("kv_heads", 0, -1), ("heads", 2048, -3), ("channels", 33, -3), ("channels", 136, -3), ("channels", 0, -3),
    ("scale", math.nan, -1), ("cap", -1.0, -1), ("cap", 1e-35, -1), ("q", None, -1), ("v", None, -1), ("q_ptr", None, -1),
    ("k_ptr", None, -1), ("out", None, -1), ("q", 4100, -1), ("k_row", 65, -1), ("v_head", -32, -1),
    ("lse", None, -1), ("grad_out", None, -1), ("grad_k", None, -1), ("grad_v", 4104, -1),
    ("grad_slope", 4096, -1), ("workspace", None, -1), ("workspace_bytes", 4, -1), ("workspace", 4100, -1)])
def test_attention_boundary(field, value, code):
    from trafficrl import _lib
    L = _lib.load()
    a = _attention_args()
    setattr(a, field, value)
    assert L.trx_node_attention_backward(a, None) == code
    assert b"node_attention" in L.trx_last_error()
    assert L.trx_node_attention_backward(None, None) == L.trx_node_attention_forward(None, None) == -1
    assert L.trx_node_attention_workspace_bytes(None, 0) == -1


def test_attention_without_rows_is_no_call():
    from trafficrl import _lib
    a = _attention_args()
    a.num_queries = 0
    assert _lib.load().trx_node_attention_forward(a, None) == 0


def _log_probs_args():
    from trafficrl import _lib
    a = _lib.TrxActionLogProbsArgs()
    a.rows, a.row_len, a.row_stride, a.top_k = 3, 70000, 70000, 2
    for f in ("logits", "action", "log_prob", "entropy", "stats", "top_log_prob", "top_action", "grad_logits",
              "workspace"):
        setattr(a, f, 4096)
    a.workspace_bytes = 1 << 40
    return a


@pytest.mark.parametrize("field,value,code", [
    ("rows", -1, -1), ("rows", (1 << 23) + 1, -3), ("row_len", -1, -1), ("row_len", 1 << 31, -3), ("dtype", 3, -1),
    ("mask_dtype", 2, -1), ("top_k", 17, -3), ("top_k", -1, -3), ("logits", None, -1), ("action", None, -1),
    ("stats", None, -1), ("log_prob", None, -1), ("top_action", None, -1), ("top_log_prob", None, -1)])
def test_log_probs_boundary(field, value, code):
    from trafficrl import _lib
    L = _lib.load()
    a = _log_probs_args()
    setattr(a, field, value)
    assert L.trx_action_log_probs_forward(a, None) == code
    assert b"action_log_probs" in L.trx_last_error()
    a = _log_probs_args()
    a.grad_logits = None
    assert L.trx_action_log_probs_backward(a, None) == -1
    a.rows = 0
    assert L.trx_action_log_probs_forward(a, None) == L.trx_action_log_probs_backward(a, None) == 0
    assert L.trx_action_log_probs_workspace_bytes(None) == -1


def test_dropout_boundary():
    from trafficrl import _lib
    L = _lib.load()
    fwd, bwd = L.trx_dropout_add_forward, L.trx_dropout_add_backward
    assert fwd(-1, 0, 4096, None, 4096, 1, 0, 4096, 4096, None) == -1
    assert fwd(8, 3, 4096, None, 4096, 1, 0, 4096, 4096, None) == -1
    assert fwd(8, 0, None, None, 4096, 1, 0, 4096, 4096, None) == -1
    assert fwd(8, 0, 4096, None, None, 1, 0, 4096, 4096, None) == -1
    assert fwd(8, 0, 4096, None, 4096, 65536, 0, 4096, 4096, None) == -1
    assert fwd(8, 0, 4100, None, 4096, 1, 0, 4096, 4096, None) == -1
    assert fwd(8, 0, 4096, 4100, 4096, 1, 0, 4096, 4096, None) == -1
    assert bwd(8, 0, 4096, 4096, -1, 0, 4096, None) == -1
    assert bwd(8, 0, 4096, None, 1, 0, 4096, None) == -1
    assert fwd(0, 0, None, None, None, 1, 0, None, None, None) == bwd(0, 0, None, None, 1, 0, None, None) == 0
