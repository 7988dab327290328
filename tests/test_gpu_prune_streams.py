"""The in-place prune spin-waits on lower slices, so the library keeps the condition that makes the wait safe: one grid in flight whatever the number of streams,
and no in-place grid on a stream whose CUs cannot hold it."""
import ctypes

import numpy as np
import pytest
import torch

from conftest import cu_mask_status
from oracle import qp_oracle as O

pytestmark = pytest.mark.gpu
D = 128
PAST, N, K, HKV = 2887, 5760, 2880, 4


@pytest.fixture(scope="module")
def ops():
    from quickvideo_amd.native import QuickPrefillOps
    return QuickPrefillOps(torch.device("cuda:0"))


@pytest.fixture(scope="module")
def case():
    rs = np.random.RandomState(12)
    keys, vals = (torch.from_numpy(rs.standard_normal((HKV, PAST + N, D)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(2))
    ko, vo = O.torch_bf16_to_bits(keys.cpu()).copy(), O.torch_bf16_to_bits(vals.cpu()).copy()
    idx, _ = O.prune_tail(ko, vo, PAST, N, K)
    return keys, vals, idx, torch.from_numpy(ko[:, :PAST + K].view(np.int16)).cuda(), torch.from_numpy(vo[:, :PAST + K].view(np.int16)).cuda()


def same(case, kc, vc, idx):
    _, _, ref, want_k, want_v = case
    return torch.equal(kc[:, :PAST + K].view(torch.int16), want_k) and torch.equal(vc[:, :PAST + K].view(torch.int16), want_v) and np.array_equal(idx.cpu().numpy(), ref)


def buffers(case):
    return case[0].clone(), case[1].clone(), torch.full((K,), -1, dtype=torch.int32, device="cuda")


def test_prune_tail_in_place_on_six_streams(ops, case):
    small = ops.prune_tail_workspace_bytes(N, K, HKV, D)
    assert small == -(-N * 2 // 256) * 256 + -(-((N + 15) // 16) * 4 // 256) * 256               # the in-place form's: 2.25 B per token
    assert ops.prune_workspace_bytes(N, K, HKV, D) >= small
    streams = [torch.cuda.Stream() for _ in range(6)]
    torch.cuda.synchronize()
    runs = []
    for _ in range(20):
        for st in streams:
            with torch.cuda.stream(st):
                kc, vc, idx = buffers(case)
                ws = torch.empty(small, dtype=torch.uint8, device="cuda")
                ops.prune_tail(kc, vc, (PAST + N) * D, PAST, N, K, HKV, D, idx, ws)
                runs.append((kc, vc, idx, ws))
    torch.cuda.synchronize()
    assert sum(not same(case, *r[:3]) for r in runs) == 0


def test_prune_tail_on_a_stream_of_few_cus(ops, case):
    """Two CUs of each of the eight XCDs cannot hold the grid of 360 workgroups: the size query for THAT stream gives the staged form's figure, prune_tail takes
    that form there and says so when handed only the in-place workspace."""
    from quickvideo_amd.native import QuickPrefillError
    words = [0x0000ffff] + [0] * 7
    if cu_mask_status(words):
        pytest.skip(f"hipExtStreamCreateWithCUMask: status {cu_mask_status(words)}")
    hip, raw = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p()
    assert hip.hipExtStreamCreateWithCUMask(ctypes.byref(raw), 8, (ctypes.c_uint32 * 8)(*words)) == 0
    small = ops.prune_tail_workspace_bytes(N, K, HKV, D)
    try:
        ext = torch.cuda.ExternalStream(raw.value)
        with torch.cuda.stream(ext):
            need = ops.prune_tail_workspace_bytes(N, K, HKV, D)
            assert need > small
            kc, vc, idx = buffers(case)
            with pytest.raises(QuickPrefillError, match="staged form"):
                ops.prune_tail(kc, vc, (PAST + N) * D, PAST, N, K, HKV, D, idx, torch.empty(small, dtype=torch.uint8, device="cuda"))
            ops.prune_tail(kc, vc, (PAST + N) * D, PAST, N, K, HKV, D, idx, torch.empty(need, dtype=torch.uint8, device="cuda"))
            ext.synchronize()
            assert same(case, kc, vc, idx)
    finally:
        torch.cuda.synchronize()
        hip.hipStreamDestroy(raw)
