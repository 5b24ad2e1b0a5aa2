"""The manager's leader lease within one pass over the jobs."""
from dgl_operator_amd.operator_plane.cluster import FakeCluster
from dgl_operator_amd.operator_plane.manager import Manager
from test_operator import GRAPHSAGE_YAML


class Leased(FakeCluster):
    """Grants the lease a given number of times; then another one holds it."""

    def __init__(self, grants):
        super().__init__()
        self.grants, self.asked = grants, 0

    def try_acquire_lease(self, namespace, name, identity, ttl_seconds=15):
        self.asked += 1
        return self.asked <= self.grants


def passes(grants, fails):
    cluster = Leased(grants)
    mgr = Manager(cluster=cluster, leader_elect=True)
    for i in range(4):
        mgr.submit(GRAPHSAGE_YAML.replace("graphsage-dist", f"job{i}"))
    seen = []

    def reconcile(job):
        seen.append(job.name)
        if job.name in fails:
            raise RuntimeError("kubectl: time limit")

    mgr.reconciler.reconcile = reconcile
    mgr.reconcile_once()
    return mgr, cluster, seen


def test_failing_jobs_renew_the_lease_too():
    jobs = ["job0", "job1", "job2", "job3"]
    for fails in ([], jobs[:2], jobs):
        mgr, cluster, seen = passes(100, fails)
        assert seen == jobs and mgr.is_leader
        assert cluster.asked == 5, "before the pass and after each job"


def test_a_lost_lease_ends_the_pass():
    for fails in ([], ["job0"], ["job1"], ["job0", "job1", "job2", "job3"]):
        mgr, cluster, seen = passes(2, fails)
        assert seen == ["job0", "job1"] and not mgr.is_leader
        assert cluster.asked == 3
