"""What a CTA of the streamed loss does when one of its waits has run out, read from the source: no wait runs out on purpose."""
import os

import _native as N


def test_copies_in_flight_are_waited_for_once_no_warp_can_issue_any():
    with open(os.path.join(N._CSRC, 'streamed_ce.cu')) as f:
        text = f.read()
    body = text[text.index('streamed_ce_kernel('):text.index('streamed_ce_join_kernel(')]
    last_barrier, leave = body.rindex('__syncthreads();'), body.rindex('cluster_sync();')
    # between the CTA's last barrier, when every warp is done, and the pair's, after which shared memory and TMEM may go away
    assert last_barrier < body.index('if (*abort_flag && threadIdx.x == 0)') < body.index('while (globaltimer_ns() - t0') < leave
    assert body.count('while (globaltimer_ns() - t0') == 1 and body.index('tmem_dealloc_pair(') > leave
