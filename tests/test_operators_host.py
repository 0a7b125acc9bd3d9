"""The device operators without a GPU: the layout of their requests, and what the entry points
refuse before they touch a device."""
import ctypes as C
import os
import re
import struct

import numpy as np
import pytest
import torch

from poorgrad_b200 import abi, operators

INVALID, UNSUPPORTED = 6, 2
DESCS = {"tb_scan_desc": abi.TbScanDesc, "tb_rotate_desc": abi.TbRotateDesc,
         "tb_policy_desc": abi.TbPolicyDesc, "tb_preference_desc": abi.TbPreferenceDesc}


@pytest.mark.parametrize("name", sorted(DESCS))
def test_requests_mirror_the_header(name):
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(here, "include", "topos_b200.h")).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for statement in body.split(";"):
        for part in statement.strip().split(","):
            if part.strip():
                field, count = re.search(r"(\w+)(?:\[(\d+)\])?\s*$", part.strip()).groups()
                fields.append((field, int(count or 1)))
    desc = DESCS[name]
    mirrored = [(field, getattr(of, "_length_", 1) if issubclass(of, C.Array) else 1)
                for field, of in desc._fields_]
    assert fields == mirrored
    assert struct.calcsize(abi.request_format(desc)) == C.sizeof(desc) == 8 * sum(n for _, n in fields)


def scan_request(**changes):
    d = abi.TbScanDesc(element=0, form=0, batch=2, length=3, channels=4)
    for name in ("gate", "x", "h", "dh", "dgate", "dx"):
        getattr(d, name + "_strides")[:] = [12, 4]
        setattr(d, name, 256)
    for name, value in changes.items():
        if name.endswith("_strides"):
            getattr(d, name)[:] = value
        else:
            setattr(d, name, value)
    return bytes(d)


def rotate_request(**changes):
    d = abi.TbRotateDesc(element=0, style=0, batch=1, length=2, q_heads=2, k_heads=1, dim=8,
                         turned=8, table_rows=4, epsilon=1e-5)
    for name in ("q", "k", "q_out", "k_out", "dq", "dk"):
        getattr(d, name + "_strides")[:] = [32, 16, 8]
        setattr(d, name, 256)
    d.table = 256
    for name, value in changes.items():
        if name.endswith("_strides"):
            getattr(d, name)[:] = value
        else:
            setattr(d, name, value)
    return bytes(d)


def policy_request(**changes):
    d = abi.TbPolicyDesc(element=0, rows=2, vocab=5, logits_stride=5, gradient_stride=5, scale=1,
                         clip_low=0.2, clip_high=0.2, kl=0)
    for name in "logits targets old_logp advantages weights loss token_loss logp".split():
        setattr(d, name, 256)
    for name, value in changes.items():
        setattr(d, name, value)
    return bytes(d)


def preference_request(**changes):
    d = abi.TbPreferenceDesc(element=0, rows=2, vocab=5, pairs=1, logits_stride=5,
                             gradient_stride=5, scale=1, beta=0.1, smoothing=0,
                             workspace_bytes=1 << 20)
    for name in "logits targets offsets ref_logp loss ratios logp workspace".split():
        setattr(d, name, 256)
    for name, value in changes.items():
        setattr(d, name, value)
    return bytes(d)


NAN = float("nan")
REFUSED = (
    [("tb_gated_scan", scan_request(**c)) for c in (
        dict(element=2), dict(form=-1), dict(batch=-1), dict(length=1 << 31), dict(channels=-4),
        dict(gate=0), dict(x=0), dict(h=0), dict(gate=257), dict(state=258),
        dict(sequences=1, batch=1), dict(offsets=256), dict(sequences=1, offsets=256),
        dict(gate_strides=[-1, 4]), dict(h_strides=[12, 3]), dict(h_strides=[0, 4]),
        dict(h_strides=[4, 4]), dict(h_strides=[8, 4]), dict(h_strides=[4, 7]),
        dict(batch=1 << 40, length=1 << 30), dict(x_strides=[1 << 62, 4]),
        dict(channels=1 << 31, batch=1), dict(gate_strides=[0, 1 << 29]))]
    + [("tb_gated_scan_backward", scan_request(**c)) for c in (
        dict(dh=0), dict(dgate=0), dict(dx=0), dict(dgate_strides=[12, 1]),
        dict(dx_strides=[1, 4]), dict(dh=255), dict(x=0, form=1))]
    + [("tb_head_rotate", rotate_request(**c)) for c in (
        dict(element=5), dict(style=2), dict(dim=7), dict(dim=514), dict(turned=10),
        dict(turned=3), dict(turned=-2), dict(epsilon=-1.0), dict(epsilon=NAN), dict(q=0),
        dict(k_out=0), dict(table=0), dict(table=2), dict(length=-1), dict(q_heads=-1),
        dict(q_out_strides=[32, 16, 4]), dict(k_out_strides=[32, 0, 8]),
        dict(q_out_strides=[0, 8, 8]), dict(q_out_strides=[0, 8, 15]), dict(q=254),
        dict(q_weight=1))]
    + [("tb_head_rotate_backward", rotate_request(**c)) for c in (
        dict(dq=0), dict(dq_weight=256), dict(dq_weight=256, workspace=256, workspace_bytes=8),
        dict(dq_weight=256, workspace=260, workspace_bytes=1 << 30))]
    + [("tb_policy_loss", policy_request(**c)) for c in (
        dict(element=9), dict(rows=-1), dict(vocab=0), dict(scale=0.0), dict(scale=NAN),
        dict(scale=1e-60), dict(clip_low=-0.1), dict(clip_high=NAN), dict(kl=-1.0), dict(kl=0.1),
        dict(logits=0), dict(targets=0), dict(weights=0), dict(loss=0), dict(logp=2),
        dict(gradient=256, gradient_stride=4), dict(gradient=258), dict(logits_stride=-5))]
    + [("tb_preference_loss", preference_request(**c)) for c in (
        dict(pairs=0), dict(beta=0.0), dict(smoothing=1.0), dict(smoothing=-0.1), dict(offsets=0),
        dict(ref_logp=0), dict(workspace=0), dict(workspace_bytes=3), dict(workspace=264),
        dict(gradient=256, gradient_stride=0), dict(weights=1), dict(vocab=1 << 50))])


@pytest.mark.parametrize("entry,request_bytes", REFUSED)
def test_malformed_requests_are_refused_before_any_device_work(built, entry, request_bytes):
    lib = abi.load_library()
    assert getattr(lib, entry)(request_bytes, None) == INVALID
    assert entry.encode() in lib.tb_last_error()


def test_entry_points_without_a_request(built):
    lib = abi.load_library()
    for entry in ("tb_gated_scan", "tb_gated_scan_backward", "tb_head_rotate",
                  "tb_head_rotate_backward", "tb_policy_loss", "tb_preference_loss"):
        assert getattr(lib, entry)(None, None) == INVALID
    assert lib.tb_head_rotate_workspace(-2) == lib.tb_head_rotate_workspace(514) == 0
    assert lib.tb_preference_workspace(-1, 1) == lib.tb_preference_workspace(4, 0) == 0
    for bad in ((7, 256, 5, 256, 2, 5, 1.0, 256), (0, 0, 5, 256, 2, 5, 1.0, 256),
                (0, 256, 5, 0, 2, 5, 1.0, 256), (0, 256, 5, 256, 2, 5, -1.0, 256),
                (0, 256, 5, 256, -2, 5, 1.0, 256), (1, 257, 5, 256, 2, 5, 1.0, 256)):
        assert lib.tb_token_logp(*bad, None) == INVALID


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the device-less answers")
def test_well_formed_requests_without_a_device(built):
    lib = abi.load_library()
    for entry, request in (("tb_gated_scan", scan_request()),
                           ("tb_gated_scan", scan_request(h_strides=[4, 8])),
                           ("tb_head_rotate", rotate_request(q_out_strides=[0, 8, 16])),
                           ("tb_gated_scan_backward", scan_request()),
                           ("tb_head_rotate", rotate_request()),
                           ("tb_head_rotate_backward", rotate_request()),
                           ("tb_policy_loss", policy_request()),
                           ("tb_preference_loss", preference_request())):
        assert getattr(lib, entry)(request, None) == UNSUPPORTED


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 3)
    for call in (lambda: operators.gated_scan(x, x), lambda: operators.gated_scan_backward(x, x, x, x),
                 lambda: operators.head_rotate(x, x, x), lambda: operators.token_logp(x[0], x),
                 lambda: operators.policy_loss(x[0], x, x, x, x),
                 lambda: operators.preference_loss(x[0], x, x, x), lambda: operators.token_logp(3, 4)):
        with pytest.raises(ValueError):
            call()


def test_rotation_table_keeps_far_angles():
    t = operators.rotation_table(3, 8, first=1_000_000)
    assert t.shape == (3, 8) and t.dtype == np.float32
    for row in range(3):
        for i in range(4):
            angle = (1_000_000 + row) * 10000.0 ** (-i / 4)
            # one rounding to f32
            assert abs(t[row, i] - np.cos(angle)) <= 2.0 ** -24
            assert abs(t[row, 4 + i] - np.sin(angle)) <= 2.0 ** -24
    assert operators.rotation_table(5, 0).shape == (5, 0)
    with pytest.raises(ValueError):
        operators.rotation_table(5, 3)
