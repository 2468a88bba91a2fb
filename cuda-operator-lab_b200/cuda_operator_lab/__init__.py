"""cuda-operator-lab for B200: sm_100a kernels behind the reference's Python API.

``cuda_operator_lab.bindings`` mirrors the reference module of the same name;
``cuda_operator_lab.benchmarking`` mirrors its timing helpers;
``cuda_operator_lab.sharding`` adds the multi-GPU (one process per GPU)
partitioning of the large workloads; ``cuda_operator_lab.fp8`` quantises to
e4m3 with a scale for each block of 128 and multiplies such operands;
``cuda_operator_lab.grouped`` multiplies rows sorted by expert with their
experts' weights, with the gradients of the bf16 form.
"""
