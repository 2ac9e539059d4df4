#!/bin/bash
# round 3, second GPU call: spectral tests, kernel timings of the product build and two variants
mkdir -p gpurun_out
timeout -k 10 300 python -u -m pytest tests/test_gpu_spectral_quant.py -x -q --timeout 200 --timeout-method thread > gpurun_out/r3_t2.log 2>&1
rc=$?; tail -n 6 gpurun_out/r3_t2.log; [ $rc -ne 0 ] && exit $rc
for rep in 1 2; do
timeout -k 10 200 python -u scratch/tk.py reps=20 >> gpurun_out/r3_tk_base.log 2>&1 || { tail -n 20 gpurun_out/r3_tk_base.log; exit 1; }
DPD_HIP_LIBRARY=$PWD/scratch/lib_q88w4.so timeout -k 10 100 python -u scratch/tk.py q88 reps=20 >> gpurun_out/r3_tk_base.log 2>&1 || { tail -n 20 gpurun_out/r3_tk_base.log; exit 1; }
DPD_HIP_LIBRARY=$PWD/scratch/lib_specnarrow.so timeout -k 10 100 python -u scratch/tk.py spec reps=20 >> gpurun_out/r3_tk_base.log 2>&1 || { tail -n 20 gpurun_out/r3_tk_base.log; exit 1; }
done
cat gpurun_out/r3_tk_base.log
exit 0
