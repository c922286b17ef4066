"""Function G's loss over packed trajectories against the scores that generation uses: the recorded outputs of the reference's
own inference (the goldens of predict_g and of forward's candidate scores) and the framework's scoring kernel.

A row's loss for a target is logsumexp(z) - z[target] over all roads, so that over the candidates of a position softmax(-loss) is predict_g's
probability and differences of losses are differences of forward's scores.  Tolerances as where the scoring kernel meets
the same goldens: 1e-4 relative, 1e-5 absolute on scores (two losses: twice)."""
import numpy as np
import pytest
import torch

from tests._fixtures import GoldenRoadWorld, build_generator, load_json

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


@pytest.fixture(scope='module')
def road_model():
    return build_generator(GoldenRoadWorld(), DEV)


def losses(model, cases):
    """[case][candidate] losses at each case's last position, all of them packed into one call."""
    loc, tim, target, starts = [], [], [], [0]
    for c in cases:
        for cand in c['cand']:
            loc += c['loc']
            tim += c['tim']
            target += [-100] * (len(c['loc']) - 1) + [cand]
            starts.append(len(loc))
    g = model.function_g.train(False)
    with torch.no_grad():
        rows = g.trajectory_loss(torch.tensor(loc), torch.tensor(tim), torch.tensor(starts, dtype=torch.int32),
                                 target=torch.tensor(target), reduction='none').cpu()
    rows = rows[torch.tensor(starts[1:]) - 1]
    return torch.split(rows, [len(c['cand']) for c in cases])


def test_losses_over_the_candidates_are_predict_g(road_model):
    cases = load_json('g234_predict.json')['cases']
    for c, row in zip(cases, losses(road_model, cases)):
        np.testing.assert_allclose(torch.softmax(-row, 0).numpy(), c['g'], rtol=1e-4)


def test_losses_differ_as_the_recorded_scores_do(road_model):
    cases = load_json('g10_masked_batch.json')['logits']
    for c, row in zip(cases, losses(road_model, cases)):
        score = np.array(c['g_score'])
        np.testing.assert_allclose((row[0] - row).numpy(), score - score[0], rtol=1e-4, atol=2e-5 + 1e-4 * float(np.abs(score).max()))


def test_losses_at_every_prefix_are_the_scoring_kernels(road_model):
    """One trajectory of a golden, all of its prefixes by the scoring kernel, against one call over it."""
    case = max(load_json('g234_predict.json')['cases'], key=lambda c: len(c['loc']))
    loc, tim, cand = case['loc'], case['tim'], case['cand']
    n = len(loc)
    assert n >= 3
    g = road_model.function_g.train(False)
    rows = []
    for c in cand:
        with torch.no_grad():
            rows.append(g.trajectory_loss(torch.tensor(loc), torch.tensor(tim), torch.tensor([0, n], dtype=torch.int32),
                                          target=torch.full((n,), c), reduction='none').cpu())
    rows = torch.stack(rows)                                                  # [candidate][position]
    for i in range(n):
        p = g.predict_g(torch.LongTensor([loc[:i + 1]]).to(DEV), torch.LongTensor([tim[:i + 1]]).to(DEV), torch.LongTensor([case['des']]).to(DEV),
                        torch.LongTensor([cand]).to(DEV), torch.FloatTensor([case['dis']]).to(DEV))
        np.testing.assert_allclose(torch.softmax(-rows[:, i], 0).numpy(), p.cpu().numpy()[0], rtol=1e-4)
