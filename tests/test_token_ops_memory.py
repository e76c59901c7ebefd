"""What the token-model operators refuse about memory and sizes, on the CPU: the checks of the native operators come
before any CUDA work."""

import pytest
import torch

from pararnn_b200 import _lib

ROWS, D = 3, 8


def step(q, k, v, decay, state, out, table=None):
    _lib.native().attention_step(q, k, v, decay, state, table, 1.0, out)


def parts(hq=2, hkv=2):
    return dict(q=torch.zeros(ROWS, hq, D), k=torch.zeros(ROWS, hkv, D), v=torch.zeros(ROWS, hkv, D),
                decay=torch.zeros(hkv), state=torch.zeros(ROWS, hkv, D, D), out=torch.zeros(ROWS, hq, D))


@pytest.mark.parametrize("name", ["q", "k"])
@pytest.mark.parametrize("shift", [-5, -1, 0, 1, 7, ROWS * 2 * D - 1])
def test_step_refuses_an_output_anywhere_inside_an_input(name, shift):
    n = ROWS * 2 * D
    flat = torch.zeros(3 * n)
    a = parts()
    a[name] = flat[n:2 * n].view(ROWS, 2, D)
    a["out"] = flat[n + shift:2 * n + shift].view(ROWS, 2, D)
    with pytest.raises(ValueError, match=f"out must not share memory with {name}"):
        step(**a)


def test_step_takes_a_neighbouring_output_and_v_itself():
    """No refusal: the call gets as far as the device, which the CPU does not have."""
    n = ROWS * 2 * D
    flat = torch.zeros(3 * n)
    a = parts()
    a["q"], a["out"] = flat[n:2 * n].view(ROWS, 2, D), flat[:n].view(ROWS, 2, D)
    with pytest.raises(RuntimeError) as e:
        step(**a)
    assert "share memory" not in str(e.value)
    a = parts()
    a["out"] = a["v"]
    with pytest.raises(RuntimeError) as e:
        step(**a)
    assert "share memory" not in str(e.value)
    # slices of one buffer that are not contiguous are copied first
    fused = torch.zeros(ROWS, 6, D)
    a = parts()
    a["q"], a["k"], a["v"] = fused[:, :2], fused[:, 2:4], fused[:, 4:]
    a["out"] = fused.view(-1)[:n].view(ROWS, 2, D)
    with pytest.raises(RuntimeError) as e:
        step(**a)
    assert "share memory" not in str(e.value)


def test_step_refuses_v_at_an_offset_or_with_other_heads():
    n = ROWS * 2 * D
    flat = torch.zeros(4 * n)
    a = parts()
    a["v"], a["out"] = flat[:n].view(ROWS, 2, D), flat[D:n + D].view(ROWS, 2, D)
    with pytest.raises(ValueError, match="with v"):
        step(**a)
    a = parts(hq=4)
    a["v"], a["out"] = flat[:n].view(ROWS, 2, D), flat[:2 * n].view(ROWS, 4, D)
    with pytest.raises(ValueError, match="with v"):
        step(**a)


def test_step_refuses_states_decays_and_tables_in_written_memory():
    pool = torch.zeros(ROWS * 2 * D * D + 64)
    a = parts()
    a["state"] = pool[64:].view(ROWS, 2, D, D)
    for name, match in (("out", "out must not share memory with state"), ("q", "state must not share memory with q"),
                        ("v", "state must not share memory with v")):
        b = dict(a)
        b[name] = pool[50:50 + ROWS * 2 * D].view(ROWS, 2, D)
        with pytest.raises(ValueError, match=match):
            step(**b)
    a = parts()
    a["decay"] = a["out"].view(-1)[4:6]
    with pytest.raises(ValueError, match="log_decay"):
        step(**a)
    a = parts()
    with pytest.raises(ValueError, match="block_table"):
        step(**a, table=a["out"].view(-1)[2:2 + ROWS].view(torch.int32))


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


BIG = 2 ** 32 + 3  # 3 in 32 bits


@pytest.mark.parametrize("change", [
    dict(state=(BIG, 1, 1, 1)), dict(q=(BIG, 1, 1), k=(BIG, 1, 1), v=(BIG, 1, 1), out=(BIG, 1, 1)),
    dict(q=(1, BIG, 1), out=(1, BIG, 1)),
])
def test_step_refuses_sizes_that_32_bits_would_cut(change):
    shapes = dict(q=(1, 1, 1), k=(1, 1, 1), v=(1, 1, 1), decay=(1,), state=(3, 1, 1, 1), out=(1, 1, 1))
    shapes.update(change)
    with pytest.raises(ValueError, match="32 bits"):
        step(**{n: meta(*s) for n, s in shapes.items()}, table=meta(1, dtype=torch.int32))


@pytest.mark.parametrize("shape", [(BIG, 1, 1, 1), (1, BIG, 1, 1), (1, 1, BIG, 1)])
def test_sequences_refuse_sizes_that_32_bits_would_cut(shape):
    x, g = meta(*shape), meta(shape[2])
    with pytest.raises(ValueError, match="32 bits"):
        _lib.native().attention_fwd(x, x, x, g, None, None, shape[0], shape[1], 1.0, False, False)
    with pytest.raises(ValueError, match="32 bits"):
        _lib.native().attention_bwd(x, x, x, g, x, None, None, None, shape[0], shape[1], 1.0, False, False)


class Captured:
    """A tensor as _offsets sees it, on a second GPU."""

    is_cuda, dtype, device = True, torch.int32, torch.device("cuda", 1)

    def is_contiguous(self):
        return True

    def dim(self):
        return 1

    def numel(self):
        return 3


def test_captured_offsets_have_to_lie_on_the_device_of_the_inputs(monkeypatch):
    from pararnn_b200 import attn_ops

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    cu = Captured()
    assert attn_ops._offsets(cu, 1, 5, torch.device("cuda", 1)) == (cu, 2, 5)
    with pytest.raises(RuntimeError, match="different devices"):
        attn_ops._offsets(cu, 1, 5, torch.device("cuda", 0))


def test_c_entry_points_refuse_states_in_place_that_others_still_read():
    """PRB_ERR_BAD_ARG before any launch.  The sizes need a workspace that is not given, so that the calls that stay
    allowed end in PRB_ERR_WORKSPACE instead of on a device."""
    import ctypes

    lib = _lib.lib()
    buf = ctypes.create_string_buffer(1024)
    p = (ctypes.addressof(buf) + 255) & ~255
    a, b, h, T = p, p + 256, ctypes.byref(_lib.Heads(p, 1, 1, 1)), 1 << 20

    def fwd(s_in, s_out, hq):
        return lib.prb_linear_attention(h, h, h, p, s_in, None, p, s_out, 1, T, 1, T, hq, 2, 8, 8, 1, 1.0, None, 0, None)

    def bwd(s_in, gs, g_state):
        return lib.prb_bwd_linear_attention(h, h, h, h, p, s_in, gs, None, p, p, p, g_state, 1, T, 1, T, 2, 2, 8, 8, 1,
                                            1.0, None, 0, None)

    bad, ws = -1, -2
    assert fwd(a, a, 4) == bad and fwd(a, a, 2) == ws and fwd(a, b, 4) == ws and fwd(None, None, 4) == ws
    assert bwd(a, None, a) == bad and bwd(None, a, a) == bad and bwd(b, b, a) == ws and bwd(None, None, None) == ws
