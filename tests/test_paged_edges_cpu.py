"""Refusals of the paged-cache entry points that concern memory shared between a call's
arguments, without a GPU."""
import ctypes

import pytest

import dial_cuda as D
from dial_cuda import paged as P

# One address range per array, far apart; never dereferenced, as every call here is refused.
SLOT = 1 << 32
AT = {n: (i + 1) * SLOT for i, n in enumerate(
    "qkv q_norm k_norm cos sin positions k_pages v_pages k_scale v_scale block_table kv_len q_start q_out k_out v_out "
    "logits ids probs temperature accept sample out_ids n_out logprobs ws".split())}
T, HQ, HKV, PAGE, N_PAGES, B, MAX_PAGES, TABLE = 8, 32, 8, 64, 100, 2, 8, 50
ROWS, V = 8, 1000
POOL = N_PAGES * HKV * PAGE
SIZE = {"qkv": T * (HQ + 2 * HKV) * 256, "q_norm": 256, "k_norm": 256, "cos": TABLE * 256, "sin": TABLE * 256,
        "positions": T * 4, "k_pages": POOL * 128, "v_pages": POOL * 128, "k_scale": POOL * 4, "v_scale": POOL * 4,
        "block_table": B * MAX_PAGES * 4, "kv_len": B * 4, "q_start": (B + 1) * 4, "q_out": T * HQ * 256,
        "k_out": T * HKV * 256, "v_out": T * HKV * 256, "logits": ROWS * V * 2, "ids": ROWS * 4, "probs": ROWS * V * 4,
        "temperature": B * 4, "accept": ROWS * 4, "sample": B * 4, "out_ids": ROWS * 4, "n_out": B * 4, "logprobs": ROWS * 4}


def structs(at):
    kv = P._PagedKv(at["k_pages"], at["v_pages"], at["k_scale"], at["v_scale"], 3, HKV, 128, PAGE, N_PAGES)
    b = P._PagedBatch(at["block_table"], at["kv_len"], at["q_start"], B, MAX_PAGES, 4, 100)
    return ctypes.byref(kv), ctypes.byref(b)


def append(at):
    kv, b = structs(at)
    axes = ctypes.byref(P._RopeAxes(1, (ctypes.c_int32 * 4)(64), 0))
    return D.lib().dial_paged_kv_append(at["qkv"], at["q_norm"], at["k_norm"], at["cos"], at["sin"], TABLE, at["positions"],
                                        axes, kv, b, at["q_out"], D.F16, T, HQ, 1e-6, None)


def read(at):
    kv, b = structs(at)
    return D.lib().dial_paged_kv_read(kv, b, at["k_out"], at["v_out"], D.F16, T, None)


def attention(at):
    kv, b = structs(at)
    return D.lib().dial_paged_attention(at["qkv"], kv, b, at["q_out"], D.F16, T, HQ, 0.1, None)


def verify(at):
    need = D.lib().dial_verify_drafts_workspace_bytes(ROWS, V)
    return D.lib().dial_verify_drafts(at["logits"], D.F16, at["ids"], at["probs"], at["q_start"], B, at["temperature"],
                                      at["accept"], at["sample"], at["out_ids"], at["n_out"], at["logprobs"], ROWS, V, 4,
                                      at["ws"], need, None)


KV = ["k_pages", "v_pages", "k_scale", "v_scale"]
BATCH = ["block_table", "kv_len", "q_start"]
# (call, what it writes, what it reads or writes besides)
CASES = [(append, ["q_out"], ["qkv", "q_norm", "k_norm", "cos", "sin", "positions"] + KV + BATCH),
         (append, KV, ["qkv", "q_norm", "k_norm", "cos", "sin", "positions"] + KV + BATCH),
         (read, ["k_out", "v_out"], KV + BATCH + ["k_out", "v_out"]),
         (attention, ["q_out"], ["qkv"] + KV + BATCH),
         (verify, ["out_ids", "n_out", "logprobs", "ws"], ["logits", "ids", "probs", "q_start", "temperature", "accept",
                                                           "sample", "out_ids", "n_out", "logprobs", "ws"])]


@pytest.mark.parametrize("call,written,other", [(c, w, o) for c, ws, os in CASES for w in ws for o in os if w != o])
def test_results_that_overlap_another_argument_are_refused(call, written, other):
    size = dict(SIZE, qkv=T * HQ * 256) if call is attention else dict(SIZE)
    size["ws"] = D.lib().dial_verify_drafts_workspace_bytes(ROWS, V)
    for shift in (0, size[other] // 16 * 16 - 16, -(size[written] // 16 * 16) + 16):
        if shift and max(size[written], size[other]) < 48:
            continue
        at = dict(AT)
        at[written] = at[other] + shift
        assert call(at) == 1 and b"overlap" in D.lib().dial_last_error(), (shift, D.lib().dial_last_error())
