"""mps_routed_check beside work on other streams and of other devices."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_check_is_of_the_stream_s_device(mps, cuda):
    class Elsewhere:
        device, cuda_stream = torch.device("cuda", 99), 0

    with pytest.raises(ValueError, match="stream: on cuda:99, expected cuda:0"):
        mps.routed_check(device=0, stream=Elsewhere())
    with pytest.raises(ValueError, match="stream: on cuda:99, expected cuda:0"):
        mps.routed_check(device=torch.device("cuda"), stream=Elsewhere())
    s = torch.cuda.Stream()
    for device in (None, 0, "cuda", "cuda:0", torch.device("cuda", 0)):
        for stream in (None, s):
            mps.routed_check(device=device, stream=stream)
