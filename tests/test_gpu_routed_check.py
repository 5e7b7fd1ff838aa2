"""mps_routed_check beside work on other streams and of other devices."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_report_made_after_a_check_is_not_wiped_out(mps, cuda):
    """A stream on which another thread keeps putting work: what a check there clears is cleared when it returns, and not after a
    call on another stream has reported something new."""
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    bad, rows = torch.full((8, 1), 99, dtype=torch.int32, device="cuda"), torch.ones(8, 16, device="cuda")
    mps.routed_combine(rows, bad)
    with pytest.raises(mps.MpsError):
        mps.routed_check()
    torch.cuda.synchronize()
    stop = threading.Event()

    def keep_busy():
        with torch.cuda.stream(side):
            for _ in range(4000):
                if stop.is_set():
                    return
                torch.cuda._sleep(200_000)  # about 0.1 ms
                if _ % 8 == 7:
                    side.synchronize()

    thread = threading.Thread(target=keep_busy)
    thread.start()
    try:
        for _ in range(40):
            mps.routed_combine(rows, bad, stream=side)
            with pytest.raises(mps.MpsError):
                mps.routed_check(stream=side)
            mps.routed_combine(rows, bad, stream=other)
            other.synchronize()
            side.synchronize()
            with pytest.raises(mps.MpsError):
                mps.routed_check(stream=other)
    finally:
        stop.set()
        thread.join()
    torch.cuda.synchronize()
    mps.routed_check()


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
