"""Log probabilities that are written in the random numbers' place, through the C entry point."""
import pytest
import torch

from test_gpu_verify import inputs

pytestmark = pytest.mark.gpu


def test_logprobs_in_the_place_of_the_numbers(gpu):
    from dciknn_cuda_amd import _capi
    lib = _capi.lib()
    n, k, v, slots = 33, 4, 5000, 6
    z, drafts, u, ids, teacher = (t.cuda() for t in inputs(n, k, v, slots, "bf16", seed=1))
    want = gpu.verify_drafts(z, drafts, u, ids, teacher)
    need = lib.dcih_verify_work(n, k, v, 2)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    tokens, accepted = torch.empty(n, k + 1, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    assert lib.dcih_verify(z.data_ptr(), 2, n, k, v, v, drafts.data_ptr(), 8, u.data_ptr(), ids.data_ptr(), 8, teacher.data_ptr(), 0, slots, 1.0, tokens.data_ptr(), accepted.data_ptr(),
                           u.data_ptr(), work.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(tokens, want[0]) and torch.equal(accepted, want[1]) and torch.equal(u, want[2])
