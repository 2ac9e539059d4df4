#!/bin/bash
# round 3, first GPU call: the whole GPU suite
R=$PWD
mkdir -p gpurun_out
timeout -k 10 900 python -u -m pytest tests -m gpu -x -q --timeout 300 --timeout-method thread > gpurun_out/r3_t1.log 2>&1
rc=$?
tail -n 15 gpurun_out/r3_t1.log
[ $rc -ne 0 ] && exit $rc
exit 0
