"""Refusals of the quantised decode operators and the 4-bit cache's host side (no GPU needed)."""
import ctypes

import pytest
import torch

import ds_kernels
from mla_cache import LatentKVCache4

bf16 = torch.bfloat16
P = ctypes.c_void_p
F = ctypes.c_float


def lib():
    return ds_kernels.library()


@pytest.mark.parametrize("call", [
    lambda: ds_kernels.int8_quantize(torch.zeros(2, 16, dtype=bf16)),
    lambda: ds_kernels.int8_linear(torch.zeros(2, 16, dtype=bf16), torch.zeros(8, 16, dtype=torch.int8), torch.ones(8)),
    lambda: ds_kernels.mla_cache4_append(torch.zeros(1, 1, 512, dtype=bf16), torch.zeros(1, 1, 64, dtype=bf16),
                                         LatentKVCache4(1, 4, "cpu"), torch.zeros(4, 64, dtype=bf16),
                                         torch.zeros(4, 64, dtype=bf16)),
    lambda: ds_kernels.mla_decode_attention4(torch.zeros(1, 16, 576, dtype=bf16), LatentKVCache4(1, 4, "cpu"), 1.0),
    lambda: ds_kernels.mla_cache4_get(LatentKVCache4(1, 4, "cpu"), 1),
    lambda: ds_kernels.mla_cache4_evict(LatentKVCache4(1, 4, "cpu"), 2),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="CUDA"):
        call()


C = [P(256 * i) for i in range(1, 16)]


@pytest.mark.parametrize("call,code", [
    # int8: K a multiple of 16 up to 131072, N of 8, aligned rows, a workspace
    (lambda L: L.ds_int8_quantize(C[0], 24, 2, 24, C[1], C[2], None), 1),
    (lambda L: L.ds_int8_quantize(C[0], 8, 2, 16, C[1], C[2], None), 1),
    (lambda L: L.ds_int8_quantize(C[0], 20, 2, 16, C[1], C[2], None), 1),
    (lambda L: L.ds_int8_quantize(P(258), 16, 2, 16, C[1], C[2], None), 1),
    (lambda L: L.ds_int8_quantize(None, 16, 2, 16, C[1], C[2], None), 1),
    (lambda L: L.ds_int8_linear(C[0], 24, C[1], C[2], C[3], 2, 8, 24, C[4], 1 << 20, None), 1),
    (lambda L: L.ds_int8_linear(C[0], 16, C[1], C[2], C[3], 2, 12, 16, C[4], 1 << 20, None), 1),
    (lambda L: L.ds_int8_linear(C[0], 131088, C[1], C[2], C[3], 2, 8, 131088, C[4], 1 << 20, None), 1),
    (lambda L: L.ds_int8_linear(C[0], 16, None, C[2], C[3], 2, 8, 16, C[4], 1 << 20, None), 1),
    (lambda L: L.ds_int8_linear(C[0], 16, C[1], C[2], C[3], 5, 8, 16, None, 0, None), 1),
    (lambda L: L.ds_int8_linear(C[0], 16, C[1], C[2], C[3], -1, 8, 16, C[4], 1 << 20, None), 1),
    (lambda L: L.ds_int8_linear(C[0], 16, P(520), C[2], C[3], 2, 8, 16, C[4], 1 << 20, None), 1),
    (lambda L: L.ds_int8_linear(C[0], 16, C[1], C[2], C[3], 5, 8, 16, C[4], 31, None), 5),
    # append: slots a multiple of 64, room, aligned rows
    (lambda L: L.ds_mla_cache4_append(C[0], 512, C[1], 64, 1, 1, None, C[2], C[3], 4, F(1e-6), C[4], C[5], C[6], C[7],
                                      C[8], C[9], 1, 63, None), 1),
    (lambda L: L.ds_mla_cache4_append(C[0], 512, C[1], 64, 1, 65, None, C[2], C[3], 4, F(1e-6), C[4], C[5], C[6], C[7],
                                      C[8], C[9], 1, 64, None), 1),
    (lambda L: L.ds_mla_cache4_append(C[0], 510, C[1], 64, 1, 1, None, C[2], C[3], 4, F(1e-6), C[4], C[5], C[6], C[7],
                                      C[8], C[9], 1, 64, None), 1),
    (lambda L: L.ds_mla_cache4_append(C[0], 512, C[1], 64, 1, 1, None, C[2], C[3], 0, F(1e-6), C[4], C[5], C[6], C[7],
                                      C[8], C[9], 1, 64, None), 1),
    (lambda L: L.ds_mla_cache4_append(C[0], 512, C[1], 64, 1, 1, None, C[2], C[3], 4, F(1e-6), C[4], None, C[6], C[7],
                                      C[8], C[9], 1, 64, None), 1),
    (lambda L: L.ds_mla_cache4_append(C[0], 512, C[1], 64, 1, 1, None, C[2], C[3], 4, F(1e-6), C[4], C[5], C[6], C[7],
                                      C[8], C[9], 65536, 64, None), 1),
    # get
    (lambda L: L.ds_mla_cache4_get(C[0], C[1], C[2], 1, 64, 65, C[3], C[4], None), 1),
    (lambda L: L.ds_mla_cache4_get(C[0], C[1], C[2], 1, 64, 4, None, C[4], None), 1),
    # attention: heads, bounds, pointers
    (lambda L: L.ds_mla_decode_attention4(C[0], 0, C[1], C[2], C[3], C[4], C[5], 1, 64, 4, F(1), 0, F(0), C[6], C[7],
                                          1 << 20, None), 1),
    (lambda L: L.ds_mla_decode_attention4(C[0], 129, C[1], C[2], C[3], C[4], C[5], 1, 64, 4, F(1), 0, F(0), C[6], C[7],
                                          1 << 20, None), 1),
    (lambda L: L.ds_mla_decode_attention4(C[0], 16, C[1], C[2], C[3], C[4], C[5], 1, 64, 65, F(1), 0, F(0), C[6], C[7],
                                          1 << 20, None), 1),
    (lambda L: L.ds_mla_decode_attention4(C[0], 16, C[1], C[2], C[3], C[4], C[5], 1, 64, 4, F(1), 0, F(0), C[6], None,
                                          0, None), 1),
    (lambda L: L.ds_mla_decode_attention4(P(260), 16, C[1], C[2], C[3], C[4], C[5], 1, 64, 4, F(1), 0, F(0), C[6], C[7],
                                          1 << 20, None), 1),
    # the decode step: heads, hidden, room for the token, pointers
    (lambda L: L.ds_mla_decode4_step(*C[:7], 4, 256, 0, F(1e-6), F(1), 0, F(0), *C[7:13], 1, 64, 4, C[13], C[14],
                                     1 << 20, None), 1),
    (lambda L: L.ds_mla_decode4_step(*C[:7], 4, 264, 16, F(1e-6), F(1), 0, F(0), *C[7:13], 1, 64, 4, C[13], C[14],
                                     1 << 20, None), 1),
    (lambda L: L.ds_mla_decode4_step(*C[:7], 4, 256, 16, F(1e-6), F(1), 0, F(0), *C[7:13], 1, 64, 65, C[13], C[14],
                                     1 << 20, None), 1),
    (lambda L: L.ds_mla_decode4_step(*C[:7], 4, 256, 16, F(1e-6), F(1), 0, F(0), *C[7:13], 1, 64, 4, C[13], None,
                                     0, None), 1),
    (lambda L: L.ds_mla_cache4_reset(None, 1, None), 1),
    (lambda L: L.ds_mla_cache4_reset(C[0], 65536, None), 1),
    # evict: budget, recent, the result shares all or nothing
    (lambda L: L.ds_mla_cache4_evict(*C[:6], 1, 64, 0, 0, *C[:6], 64, C[12], 1 << 20, None), 1),
    (lambda L: L.ds_mla_cache4_evict(*C[:6], 1, 64, 65, 0, *C[:6], 64, C[12], 1 << 20, None), 1),
    (lambda L: L.ds_mla_cache4_evict(*C[:6], 1, 64, 8, 9, *C[:6], 64, C[12], 1 << 20, None), 1),
    (lambda L: L.ds_mla_cache4_evict(*C[:6], 1, 64, 8, -1, *C[:6], 64, C[12], 1 << 20, None), 1),
    (lambda L: L.ds_mla_cache4_evict(*C[:6], 1, 64, 8, 0, C[0], *C[7:12], 64, C[12], 1 << 20, None), 1),
    (lambda L: L.ds_mla_cache4_evict(*C[:6], 1, 64, 8, 0, *C[6:11], C[5], 64, C[12], 1 << 20, None), 1),
    (lambda L: L.ds_mla_cache4_evict(*C[:6], 1, 64, 8, 0, *C[:6], 128, C[12], 1 << 20, None), 1),
    (lambda L: L.ds_mla_cache4_evict(*C[:6], 1, 64, 8, 0, *C[:6], 64, C[12], 16, None), 5),
])
def test_the_c_entries_refuse_before_any_launch(call, code):
    assert call(lib()) == code
    assert lib().ds_last_error().decode()


def test_zero_size_calls_are_no_ops():
    L = lib()
    assert L.ds_int8_quantize(None, 16, 0, 16, None, None, None) == 0
    assert L.ds_int8_linear(None, 16, None, None, None, 0, 8, 16, None, 0, None) == 0
    assert L.ds_mla_cache4_reset(None, 0, None) == 0
    assert L.ds_mla_cache4_get(None, None, None, 1, 64, 0, None, None, None) == 0


def test_cache_construction_and_host_bounds():
    for bad in (0, -1, 1.5):
        with pytest.raises(ValueError):
            LatentKVCache4(bad, 4, "cpu")
        with pytest.raises(ValueError):
            LatentKVCache4(1, bad, "cpu")
    c = LatentKVCache4(2, 100, "cpu")
    assert c.slots == 128 and c.codes.shape == (2, 128, 288) and c.scales.shape == (2, 5, 128)
    assert c.memory_bytes == 2 * 128 * 310 + 24
    assert c.current_len == 0 and c.remaining_capacity == 100
    c._check_room(100, 100)
    with pytest.raises(RuntimeError, match="overflow"):
        c._check_room(101, 1000)
    with pytest.raises(RuntimeError, match="RoPE"):
        c._check_room(10, 9)
    c._advance(60)
    with pytest.raises(RuntimeError, match="overflow"):
        c._check_room(41, 1000)
    d = LatentKVCache4(2, 32, "cpu")
    d._evicted(c, 32)
    assert d.current_len == 32 and d._seen == 60
    d.reset()
    assert d.current_len == 0 and d._seen == 0


def test_load_state_dict_checks_what_it_takes():
    c = LatentKVCache4(2, 64, "cpu")
    c.state[:2].copy_(torch.tensor([[3, 64], [5, 64]]))
    sd = c.state_dict()
    d = LatentKVCache4(2, 200, "cpu")
    d.load_state_dict(sd)
    assert d.lens.tolist() == [3, 64] and d.next_pos.tolist() == [5, 64] and d.current_len == 64
    e = LatentKVCache4(2, 200, "cpu")
    e.load_state_dict({k: sd[k] for k in ("codes", "scales", "rstd", "lens")})
    assert e.next_pos.tolist() == [3, 64] and e.pos[0, 190] == 190
    for key in ("codes", "scales", "rstd", "lens"):
        with pytest.raises(ValueError, match=key):
            LatentKVCache4(2, 64, "cpu").load_state_dict({k: v for k, v in sd.items() if k != key})
    with pytest.raises(ValueError, match="shape"):
        LatentKVCache4(3, 64, "cpu").load_state_dict(sd)
    with pytest.raises(ValueError, match="fit"):
        LatentKVCache4(2, 63, "cpu").load_state_dict(sd)       # 64 tokens do not fit 63
    sd["lens"] = torch.tensor([-1, 3], dtype=torch.int32)
    with pytest.raises(ValueError, match="fit"):
        LatentKVCache4(2, 64, "cpu").load_state_dict(sd)


def test_a_recorded_eviction_or_reset_keeps_the_bounds_of_what_the_cache_still_holds(monkeypatch):
    c, d = LatentKVCache4(2, 100, "cpu"), LatentKVCache4(2, 64, "cpu")
    c._advance(60)
    d._advance(20)
    with monkeypatch.context() as m:
        m.setattr(LatentKVCache4, "_recording", lambda self: True)
        d._evicted(c, 10)
        c._evicted(c, 32)
        c._check_room(68, 128)                  # behind the recorded eviction
        with pytest.raises(RuntimeError, match="overflow"):
            c._check_room(69, 1000)
    assert c.current_len == 60 and c.remaining_capacity == 40 and d.current_len == 20
    with pytest.raises(RuntimeError, match="overflow"):
        c._check_room(41, 1000)
    c.note_replay(1, budget=32)
    assert c.current_len == 33 and c._seen == 61
    c._check_room(67, 128)
    with monkeypatch.context() as m:
        m.setattr(LatentKVCache4, "_recording", lambda self: True)
        c.reset()
        c._check_room(100, 100)
        c._advance(5)
    assert c.current_len == 33
    with pytest.raises(RuntimeError, match="RoPE"):
        c._check_room(1, 61)
    c.note_replay(5, budget=0)
    assert c.current_len == 5 and c._seen == 5
    c.reset()
    assert c.current_len == 0 and c._seen == 0


def test_copies_have_arrays_of_their_own_and_arrays_are_not_replaced():
    import copy
    import pickle
    c = LatentKVCache4(2, 64, "cpu")
    c.state[:2].copy_(torch.tensor([[3, 4], [5, 6]]))
    c._advance(6)
    for d in (copy.deepcopy(c), pickle.loads(pickle.dumps(c))):
        assert not set(d._ptrs) & set(c._ptrs)
        assert d._ptrs == tuple(t.data_ptr() for t in (d.codes, d.scales, d.rstd, d.pos, d.mass, d.state))
        assert d.lens.tolist() == [3, 4] and d.next_pos.tolist() == [5, 6] and d.current_len == 6
        d.lens.zero_()
        assert d.state[0].tolist() == [0, 0] and c.lens.tolist() == [3, 4]
    for name in ("codes", "scales", "rstd", "pos", "mass", "state", "lens", "next_pos"):
        with pytest.raises(AttributeError):
            setattr(c, name, torch.zeros(2))


@pytest.mark.parametrize("slots", [64, 1024, 1088, 16384])
@pytest.mark.parametrize("which", ["mass", "pos"])
@pytest.mark.parametrize("in_place", [True, False])
def test_eviction_refuses_arrays_that_it_could_not_read_four_at_a_time(slots, which, in_place):
    src = list(C[:6])
    i = {"pos": 3, "mass": 4}[which]
    for off in (4, 8):
        src[i] = P(C[i].value + off)
        dst = src if in_place else C[6:12]
        assert lib().ds_mla_cache4_evict(*src, 1, slots, 8, 0, *dst, slots, C[12], 1 << 20, None) == 1
        assert "aligned" in lib().ds_last_error().decode()


@pytest.mark.parametrize("call", [
    lambda L: L.ds_mla_cache4_evict(*C[:6], 1, 64, 8, 0, *C[:6], 64, P(C[12].value + 2), 1 << 20, None),
    lambda L: L.ds_mla_cache4_get(C[0], P(C[1].value + 1), C[2], 1, 64, 4, C[3], C[4], None),
    lambda L: L.ds_mla_cache4_append(C[0], 512, C[1], 64, 1, 1, None, P(C[2].value + 1), C[3], 4, F(1e-6), *C[4:10], 1,
                                     64, None),
    lambda L: L.ds_mla_cache4_append(C[0], 512, C[1], 64, 1, 1, None, C[2], P(C[3].value + 1), 4, F(1e-6), *C[4:10], 1,
                                     64, None),
    lambda L: L.ds_mla_decode4_step(*C[:5], P(C[5].value + 1), C[6], 4, 256, 16, F(1e-6), F(1), 0, F(0), *C[7:13], 1,
                                    64, 4, C[13], C[14], 1 << 20, None),
    lambda L: L.ds_mla_decode4_step(*C[:6], P(C[6].value + 1), 4, 256, 16, F(1e-6), F(1), 0, F(0), *C[7:13], 1, 64, 4,
                                    C[13], C[14], 1 << 20, None),
])
def test_untyped_pointers_off_their_type_s_boundary_are_refused(call):
    assert call(lib()) == 1
    assert "aligned" in lib().ds_last_error().decode()


def recording(m):
    m.setattr(LatentKVCache4, "_recording", lambda self: True)


def test_eager_calls_behind_a_recorded_eviction_move_the_bounds_of_what_is_held(monkeypatch):
    monkeypatch.setattr("mla_cache._capturing", lambda: False)
    c = LatentKVCache4(2, 400, "cpu")
    c._advance(200)
    with monkeypatch.context() as m:
        recording(m)
        c._evicted(c, 100)
        c._advance(1)                            # the recorded step's token
    c.note_replay(-1)                            # recording appended nothing
    assert c.current_len == 200 and c.bound_for_launch == 200
    for i in range(150):                         # eager tokens: the eviction has not run
        c._check_room(1, 1000)
        c._advance(1)
        assert c.current_len == c.bound_for_launch == 201 + i
    c._advance(50)
    with pytest.raises(RuntimeError, match="overflow"):
        c._check_room(1, 1000)                   # the device holds 400 of 400
    with pytest.raises(RuntimeError, match="RoPE"):
        LatentKVCache4._check_room(c, 0, 399)
    c.note_replay(1, budget=100)
    assert c.current_len == 101 and c._seen == 401
    # the same behind a recorded reset, and behind replays of a graph that does not evict
    d = LatentKVCache4(2, 400, "cpu")
    d._advance(300)
    with monkeypatch.context() as m:
        recording(m)
        d.reset()
    d._advance(3)
    d.note_replay(2)
    assert d.current_len == 305
    d.note_replay(4, budget=0)
    assert d.current_len == 4 and d._seen == 4


def test_a_recorded_eviction_into_another_cache_bounds_whatever_its_source_holds_by_then(monkeypatch):
    import copy
    import pickle
    monkeypatch.setattr("mla_cache._capturing", lambda: False)
    src, dst = LatentKVCache4(2, 2000, "cpu"), LatentKVCache4(2, 1000, "cpu")
    src._advance(200)
    with monkeypatch.context() as m:
        recording(m)
        dst._evicted(src, 800)
        with pytest.raises(RuntimeError, match="overflow"):
            dst._check_room(201, 5000)           # a replay may leave 800
    assert src.current_len == 200 and dst.current_len >= 0
    src._advance(800)                            # 1000 by the replay: min(1000, 800) slots arrive
    dst.note_replay(0, 800)
    assert dst.current_len == dst.bound_for_launch == 800 and dst._seen == 1000
    with pytest.raises(RuntimeError, match="overflow"):
        dst._check_room(201, 5000)
    with pytest.raises(RuntimeError, match="RoPE"):
        dst._check_room(1, 1000)
    dst.reset()                                  # and again behind a reset of the result
    assert dst.current_len == 0
    src._advance(300)
    dst.note_replay(0, budget=800)
    assert dst.current_len == 800 and dst._seen == 1300
    dst.reset()
    dst.note_replay(2, 800, src=src)             # with the source named, its own bounds count
    assert dst.current_len == 802 and dst._seen == 1302
    short = LatentKVCache4(2, 2000, "cpu")
    short._advance(5)
    dst.reset()
    dst.note_replay(0, 800, src=short)
    assert dst.current_len == 5 and dst._seen == 5
    for d in (copy.deepcopy(dst), pickle.loads(pickle.dumps(dst))):  # no graph writes into a copy
        d.reset()
        d.note_replay(0, 800)
        assert d.current_len == 0 and d._seen == 0
    dst.note_replay(0, 5000)                     # more than there are slots
    assert dst.current_len == 1000
    del src                                      # the graph's memory is gone, the bounds stay usable
    dst.note_replay(0, 800)
    assert dst.current_len == 800


@pytest.mark.parametrize("next_pos", [[-1, 5], [2, 5], [3, -2 ** 31]])
def test_load_state_dict_refuses_positions_before_the_tokens_that_are_there(next_pos):
    c = LatentKVCache4(2, 64, "cpu")
    c.state[:2].copy_(torch.tensor([[3, 4], [3, 4]]))
    sd = c.state_dict()
    sd["next_pos"] = torch.tensor(next_pos, dtype=torch.int32)
    d = LatentKVCache4(2, 64, "cpu")
    with pytest.raises(ValueError, match="next_pos"):
        d.load_state_dict(sd)
    assert d.lens.tolist() == [0, 0] and d.current_len == 0
