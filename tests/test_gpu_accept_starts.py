"""mtp_accept_sampled on cuda:0 where starts fall: the sequences before the fall come out as they would alone, at their own
temperatures, those from it on are impossible."""
import pytest
import torch

from tests.test_gpu_accept_int8 import Drafts, accept_reference, i32

pytestmark = pytest.mark.gpu


def expected(x, starts, T, most):
    """tokens, count, status: each sequence that may be served by itself, in 64 bits."""
    tokens, count, status = [], [], []
    rises = True
    for b, (t0, t1) in enumerate(zip(starts, starts[1:])):
        rises = rises and t1 >= t0
        if not (rises and 0 <= t0 and t1 <= T and t1 - t0 <= most):
            tokens.append(torch.full((most,), -1, dtype=torch.int32)), count.append(0), status.append(-1)
            continue
        one = accept_reference(x.logits, x.drafts, torch.tensor([t0, t1]), x.u, x.temperature[b:b + 1], most, x.draft_logits)
        tokens.append(one[0][0]), count.append(int(one[1][0])), status.append(int(one[2][0]))
    return torch.stack(tokens), count, status


@pytest.mark.parametrize("Vd", [0, 400])
@pytest.mark.parametrize("starts", [[0, 4, 2, 6], [0, 5, 3, 8], [4, 8, 0, 4], [0, 3, 3, 2, 6, 8], [6, 8, 5, 7], [-1, 3, 6, 4, 8], [0, 2, 2 ** 31 - 1, 4, 8], [0, 2, -2 ** 31, 4]])
def test_rows_of_two_sequences_are_the_first_ones(starts, Vd):
    for seed in range(6):
        x = Drafts([8], 500, Vd, seed=seed, near=0.3)
        B = len(starts) - 1
        x.n, x.starts = 6, i32(starts)
        x.temperature = torch.tensor([0.3, 3.0, 30.0, 0.05, 8.0][:B], device="cuda").roll(seed)
        tokens, count, status = x.run()
        want = expected(x, starts, 8, 6)
        assert torch.equal(tokens.cpu(), want[0]) and count.tolist() == want[1] and status.tolist() == want[2], (starts, seed)


@pytest.mark.parametrize("at", [1, 63, 64, 255, 256, 700, 999])
def test_a_falling_start_among_many(at):
    x = Drafts([2] * 1000, 40, 40, seed=at, temps=[0.2 + 0.01 * (i % 90) for i in range(1000)])
    ref = x.run()
    x.starts = x.starts.clone()
    x.starts[at] = x.starts[at - 1] - 1
    tokens, count, status = x.run()
    assert torch.equal(tokens[:at - 1], ref[0][:at - 1]) and torch.equal(count[:at - 1], ref[1][:at - 1]) and torch.equal(status[:at - 1], ref[2][:at - 1])
    assert (status[at - 1:] == -1).all() and (count[at - 1:] == 0).all() and (tokens[at - 1:] == -1).all()
