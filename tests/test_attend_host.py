"""The host side of the attention entry points, without a GPU: bias buckets and refusals before any launch."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import veckern_amd as vk
from tests.attend_plain import bucket


def test_buckets_against_whole_numbers():
    from veckern_amd import attention

    for buckets, max_distance, two_sided in ((32, 128, True), (32, 128, False), (20, 100, False), (64, 512, True), (2, 2, False),
                                             (3, 1024, False), (256, 1024, True), (256, 1024, False), (7, 40, False)):
        for x in list(range(-1100, 1101, 7)) + list(range(-140, 141)) + [-10**12, 10**12]:
            assert attention.bias_bucket(x, buckets, max_distance, two_sided) == bucket(
                max(-5000, min(5000, x)), buckets, max_distance, two_sided), (x, buckets, max_distance, two_sided)


def arguments(**given):
    a = vk._Attention()
    sizes = dict(type=1, batch=2, tokens=3, heads=4, kv_heads=2, head_dim=64, passages=5, length=20, bank=10, scale=1.0)
    for name, x in {**sizes, **given}.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("wrong", [dict(type=2), dict(head_dim=60), dict(head_dim=0), dict(head_dim=136), dict(kv_heads=3),
                                   dict(kv_heads=0), dict(bank=9), dict(scale=float("inf")), dict(scale=-1.0),
                                   dict(q_start=1 << 31), dict(batch=1 << 40), dict(tokens=1 << 30), dict(heads=0)], ids=str)
def test_wrong_arguments_are_refused(wrong):
    size = ctypes.c_size_t()
    lib = vk.library()
    assert lib.vk_attend_workspace(ctypes.byref(arguments()), ctypes.byref(size)) == vk.VK_OK
    for call in (lib.vk_attend_workspace, lib.vk_attend_backward_workspace):
        assert call(ctypes.byref(arguments(**wrong)), ctypes.byref(size)) == vk.VK_ERR_INVALID_ARGUMENT, lib.vk_last_error()
    assert lib.vk_attend(ctypes.byref(arguments(**wrong)), None, 0, None) == vk.VK_ERR_INVALID_ARGUMENT


def test_missing_tensors_and_workspaces_are_refused():
    lib, size = vk.library(), ctypes.c_size_t()
    invalid = vk.VK_ERR_INVALID_ARGUMENT
    assert lib.vk_attend(None, None, 0, None) == invalid
    assert lib.vk_attend_workspace(ctypes.byref(arguments()), None) == invalid
    assert lib.vk_bias_bucket(1, 32, 128, 1, None) == invalid
    a = arguments()
    assert lib.vk_attend(ctypes.byref(a), None, 0, None) == invalid and b"q is NULL" in lib.vk_last_error()
    # host addresses that are never read: the call is refused before a launch
    held = (ctypes.c_char * 4096)()
    base = (ctypes.addressof(held) + 15) // 16 * 16
    for t in (a.q, a.k, a.v, a.out):
        t.data, t.stride = base, (768, 256, 64)
    a.k.stride = (2560, 128, 4)
    assert lib.vk_attend(ctypes.byref(a), None, 0, None) == invalid and b"multiples of 8" in lib.vk_last_error()
    a.k.stride = (2560, 128, 64)
    a.v.stride = (2560, -128, 64)
    assert lib.vk_attend(ctypes.byref(a), None, 0, None) == invalid and b"not negative" in lib.vk_last_error()
    a.v.stride = (2560, 1 << 23, 64)
    assert lib.vk_attend(ctypes.byref(a), None, 0, None) == invalid and b"2^23" in lib.vk_last_error()
    a.v.stride = (2560, 128, 64)
    a.q.data = base + 8
    assert lib.vk_attend(ctypes.byref(a), None, 0, None) == invalid and b"aligned" in lib.vk_last_error()
    a.q.data = base
    assert lib.vk_attend_backward(ctypes.byref(a), None, None, 0, None) == invalid
    g = vk._AttentionGrad()
    for t in (g.d_out, g.d_q, g.d_k, g.d_v):
        t.data, t.stride = base, (2560, 128, 64)
    assert lib.vk_attend_backward(ctypes.byref(a), ctypes.byref(g), None, 0, None) == invalid and b"lse" in lib.vk_last_error()
    a.lse = base
    g.d_table = base
    assert lib.vk_attend_backward(ctypes.byref(a), ctypes.byref(g), None, 0, None) == invalid and b"d_table" in lib.vk_last_error()
    g.d_table = None
    assert lib.vk_attend_backward_workspace(ctypes.byref(a), ctypes.byref(size)) == vk.VK_OK and size.value > 0
    assert lib.vk_attend_backward(ctypes.byref(a), ctypes.byref(g), None, 0, None) == invalid and b"workspace" in lib.vk_last_error()
    assert lib.vk_attend_backward(ctypes.byref(a), ctypes.byref(g), base + 8, size.value, None) == invalid
    a.rows = base
    assert lib.vk_attend_backward(ctypes.byref(a), ctypes.byref(g), None, 0, None) == invalid and b"constants" in lib.vk_last_error()
