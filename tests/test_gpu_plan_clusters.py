"""GPU: the step plan at its edges where clusters split the scan: more than 4096 requests, or 2^19
token rows and more (several clusters write the same results). Whole numbers, equal to the oracle's."""

import numpy as np
import pytest

from test_gpu_step import _check_plan, _i32, _step
from tq_mla import ops

pytestmark = pytest.mark.gpu
COLUMNS = 6
CASES = ["borders", "nothing new", "all empty", "negative", "short table", "cached past the table", "empty pool",
         "pool ends inside a request", "pool ends in the last request", "too many tokens", "count past the pool",
         "negative count", "no token rows", "everything at once"]


def batch(case, requests):
    """Lengths, table, free stack, count and number of token rows of an edge, ``requests`` of them."""
    rng = np.random.default_rng(len(case) + requests)
    edge_cached, edge_new = [0, 63, 64, 65, 128, 1, 127], [64, 1, 1, 63, 0, 127, 2]
    pick = np.resize(np.arange(7), requests)
    rng.shuffle(pick)
    cached, new = np.array(edge_cached)[pick], np.array(edge_new)[pick]
    some = rng.random(requests) < (0.02 if requests > 100 else 0.4)
    some[requests // 2] = some[-1] = True
    if case == "nothing new":
        new[:] = 0
    if case == "all empty":
        cached[:], new[:] = 0, 0
    if case in ("negative", "everything at once"):
        cached[some] = -cached[some] - 1
        new[np.roll(some, 3)] *= -1
    if case in ("short table", "everything at once"):
        new[np.roll(some, 1)] = 64 * COLUMNS + 77
    if case in ("cached past the table", "everything at once"):
        cached[np.roll(some, 2)] = 64 * COLUMNS + 1
    if case == "pool ends inside a request":
        new[some] = 200
    table, free = _step(rng, requests, cached, new, COLUMNS)
    first = np.minimum(-(-np.maximum(cached, 0) // 64), COLUMNS)
    last = np.minimum(-(-(np.maximum(cached, 0) + np.maximum(new, 0)) // 64), COLUMNS)
    need, count = last - first, len(free)
    if case == "empty pool":
        count = 0
    if case in ("pool ends inside a request", "everything at once"):
        # one page of a request that takes two
        two = np.flatnonzero(need >= 2)
        at = two[len(two) // 2]
        count = int(need[:at].sum()) + 1
    if case == "pool ends in the last request":
        new[-1], cached[-1] = 200, 0
        table, free = _step(rng, requests, cached, new, COLUMNS)
        first = -(-cached // 64)
        count = int((-(-(cached + new) // 64) - first).sum()) - 1
    tokens = int(np.maximum(new, 0).sum()) + 50
    if case in ("too many tokens", "everything at once"):
        tokens = int(np.maximum(new, 0).sum()) - 333 if requests > 100 else tokens
    if case == "count past the pool":
        count += 11
    if case == "negative count":
        count = -4
    if case == "no token rows":
        tokens = 0
    return cached, new, table, free, count, max(tokens, 0)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("requests", [4097, 9001])
def test_edges_of_many_requests(cuda_device, case, requests):
    _check_plan(cuda_device, *batch(case, requests))


@pytest.mark.parametrize("case", CASES)
def test_edges_over_several_clusters(cuda_device, case):
    """Many requests and 2^19 token rows, one of them with most of the tokens."""
    cached, new, table, free, count, tokens = batch(case, 4500)
    tokens = max(tokens, (1 << 19) + 5)
    if case == "too many tokens":
        new[1234] = tokens
    _check_plan(cuda_device, cached, new, table, free, count, tokens)


@pytest.mark.parametrize("case", CASES)
def test_edges_of_few_requests_over_many_token_rows(cuda_device, case):
    cached, new, table, free, count, _ = batch(case, 7)
    tokens = 1 << 19
    if case == "too many tokens":
        new[3] = tokens
    _check_plan(cuda_device, cached, new, table, free, count, tokens)


def test_lengths_near_the_type_border_in_a_cluster(cuda_device):
    top = 2 ** 31 - 1
    requests = 5000
    cached, new = np.zeros(requests, np.int64), np.ones(requests, np.int64)
    cached[[0, 2500, 4999]], new[[0, 2500, 4999]] = [top, 5, top - 1], [3, top, 2]
    table = np.arange(requests * 3).reshape(requests, 3)
    free = np.arange(requests * 3, requests * 6)
    got = ops.step_plan(_i32(cached, cuda_device), _i32(new, cuda_device), _i32(table, cuda_device),
                        _i32(free, cuda_device), _i32([len(free)], cuda_device), tokens=3000)
    starts = np.minimum(np.concatenate([[0], np.cumsum(new)]), 3000)
    assert got.q_start.tolist() == starts.tolist()
    assert got.kv_len[[0, 1, 2500, 4999]].tolist() == [192, 1, 192, 192]
    assert got.q_pos[:4].tolist() == [top] * 3 + [0]       # positions past 31 bits stay at the top
    assert got.q_pos[2502:2504].tolist() == [5, 6]
