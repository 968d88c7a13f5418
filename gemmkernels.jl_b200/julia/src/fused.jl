# Layer-level operators over gk_gemm_fused and gk_activation_gradient: products with a fused bias, activation and
# residual, products grouped by expert, and their gradients.  No counterpart in the reference.
# Not executed in this repository's environment (no Julia); the executable mirror is gemmkernels_b200/fused.py.

# include/gemmkernels_b200.h, field for field
struct GkFusedDesc
    struct_size::UInt32; form::Int32; bias_axis::Int32; activation::Int32
    bias::CuPtr{Float32}; z::CuPtr{Cvoid}; ldz::Int64; reserved::NTuple{2, Int32}
end
struct GkGroupDesc
    struct_size::UInt32; ragged::Int32; groups::Int32; offsets_dtype::Int32
    offsets::CuPtr{Cvoid}; stride_a::Int64; stride_bias::Int64; stride_c::Int64; stride_d::Int64
end
struct GkActivationGradientDesc
    struct_size::UInt32; dtype::Int32; m::Int64; n::Int64
    ld_dd::Int64; ld_z::Int64; ld_dz::Int64; ld_db::Int64
    activation::Int32; groups::Int32; offsets_dtype::Int32; reserved::Int32
    offsets::CuPtr{Cvoid}
end

gk_activation(::Nothing) = Int32(0)
gk_activation(::Transform.ReLU) = Int32(1)
gk_activation(::Transform.GELU) = Int32(2)
gk_activation(::Transform.SiLU) = Int32(3)

const CU_NONE = reinterpret(CuPtr{Cvoid}, CU_NULL)
ptr_or_null(x::Nothing) = CU_NONE
ptr_or_null(x) = reinterpret(CuPtr{Cvoid}, pointer(x))

# Epilogue -> GkFusedDesc.  `groups` > 0: the bias is a matrix, one column per group.
function fused_desc(e::Epilogue.BiasActivationResidual, groups)
    axis = e.bias === nothing ? 0 : e.axis === :row ? 1 : 2
    GkFusedDesc(sizeof(GkFusedDesc), 1, axis, gk_activation(e.activation), reinterpret(CuPtr{Float32}, ptr_or_null(e.bias)),
                ptr_or_null(e.preactivation), e.preactivation === nothing ? 0 : stride(e.preactivation, 2), (0, 0))
end
fused_desc(e::Epilogue.ActivationGradient, groups) =
    GkFusedDesc(sizeof(GkFusedDesc), 2, 0, gk_activation(e.activation), CuPtr{Float32}(0), ptr_or_null(e.preactivation),
                stride(e.preactivation, 2), (0, 0))
fused_desc(::Epilogue.Default, groups) =
    GkFusedDesc(sizeof(GkFusedDesc), 0, 0, 0, CuPtr{Float32}(0), CU_NONE, 0, (0, 0))

function product_desc(conf::Config, a, b, c, d, alpha, beta)
    la, lb, lc = conf.global_a_layout, conf.global_b_layout, conf.global_c_layout
    op, compute = op_kind(conf.operator)
    Layout.is_zero(lc) && (beta = 0.0)
    first2(x) = x === nothing ? nothing : ndims(x) == 3 ? view(x, :, :, 1) : x
    ldim(x) = (v = first2(x); v === nothing ? Int64(1) : Int64(max(stride(v, 2), size(v, 1), 1)))
    M, N, K = conf.matmul_shape.M, conf.matmul_shape.N, conf.matmul_shape.K
    GkGemmDesc(sizeof(GkGemmDesc), 0, M, N, K, !Layout.col_major(la), !Layout.col_major(lb),
               gk_dtype(eltype(a)), gk_dtype(eltype(b)), gk_dtype(eltype(d)), gk_dtype(eltype(d)), compute, op,
               ldim(a), ldim(b), c === nothing ? ldim(d) : ldim(c), ldim(d), 0, 0, 0, 0, 0, 0, c === nothing ? 1 : 0, 0,
               alpha, beta, conf.tile_n, conf.cta_group, conf.stages, conf.raster_group, 0, 0, 0, 0, 0, conf.k_blocks_per_stage, 0, 0, 0, 0)
end

# The query has no addresses and takes them to be 16-byte aligned: an operand that is not is asked for with a leading
# dimension that is no multiple of 8.
function query_desc(desc, a, b)
    off(x) = x !== nothing && UInt(reinterpret(UInt, pointer(x))) % 16 != 0
    odd(ld) = ld + (ld % 8 == 0)
    fields = map(fieldnames(GkGemmDesc)) do f
        f === :lda && off(a) ? odd(desc.lda) : f === :ldb && off(b) ? odd(desc.ldb) : getfield(desc, f)
    end
    GkGemmDesc(fields...)
end

function enqueue_fused(desc, fused, groups, a, b, c, d)
    g = groups === nothing ? Ptr{GkGroupDesc}(0) : groups
    plan = Ref(GkGemmPlan(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0))
    gk_check(ccall((:gk_gemm_fused_query, libgk), Cint, (Ptr{Cvoid}, Ref{GkGemmDesc}, Ref{GkFusedDesc}, Ptr{GkGroupDesc}, Ref{GkGemmPlan}),
                   gk_handle(), query_desc(desc, a, b), fused, g, plan))
    bytes = plan[].workspace_bytes
    ws = bytes > 0 ? reinterpret(CuPtr{Cvoid}, pointer(lent_workspace(bytes))) : CU_NONE
    gk_check(ccall((:gk_gemm_fused, libgk), Cint,
                   (Ptr{Cvoid}, Ref{GkGemmDesc}, Ref{GkFusedDesc}, Ptr{GkGroupDesc}, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{Cvoid},
                    CuPtr{Cvoid}, CuPtr{Cvoid}, Int64, Ptr{Cvoid}),
                   gk_handle(), desc, fused, g, ptr_or_null(a), ptr_or_null(b), ptr_or_null(c), ptr_or_null(d), ws, bytes,
                   CUDA.stream().handle))
end

"D = act(alpha*A*B + bias) + beta*C, or (alpha*A*B + beta*C) .* act'(Z): `matmul` with a layer-level epilogue."
matmul_fused(conf::Config, a, b, c, d, epilogue; alpha = 1.0, beta = 1.0) =
    enqueue_fused(product_desc(conf, a, b, c, d, alpha, beta), fused_desc(epilogue, 0), nothing, a, b, c, d)

group_stride(x) = x === nothing || size(x, 3) == 1 ? Int64(0) : Int64(stride(x, 3))

"D[:, J_g] = epilogue(A[:, :, g] * B[:, J_g]) with J_g = offsets[g] + 1 : offsets[g + 1] (offsets on the device, zero-based)."
function matmul_grouped(conf::Config, a, b, c, d, offsets; epilogue = Epilogue.Default(), alpha = 1.0, beta = 1.0)
    fused = fused_desc(epilogue, size(a, 3))
    sb = epilogue isa Epilogue.BiasActivationResidual && epilogue.bias !== nothing && size(a, 3) > 1 ? Int64(stride(epilogue.bias, 2)) : Int64(0)
    groups = Ref(GkGroupDesc(sizeof(GkGroupDesc), 1, size(a, 3), gk_dtype(eltype(offsets)), ptr_or_null(offsets), group_stride(a), sb, 0, 0))
    GC.@preserve groups enqueue_fused(product_desc(conf, a, b, c, d, alpha, beta), fused, Base.unsafe_convert(Ptr{GkGroupDesc}, groups), a, b, c, d)
end

"D[:, :, g] = alpha * A[:, J_g] * B[J_g, :] + beta * C[:, :, g]: the weight gradient of every group."
function matmul_grouped_outer(conf::Config, a, b, c, d, offsets; alpha = 1.0, beta = 1.0)
    groups = Ref(GkGroupDesc(sizeof(GkGroupDesc), 2, size(d, 3), gk_dtype(eltype(offsets)), ptr_or_null(offsets), 0, 0, group_stride(c), group_stride(d)))
    GC.@preserve groups enqueue_fused(product_desc(conf, a, b, c, d, alpha, beta), fused_desc(Epilogue.Default(), 0),
                                      Base.unsafe_convert(Ptr{GkGroupDesc}, groups), a, b, c, d)
end

"dZ = dD .* act'(Z) and, with `bias_gradient`, its sums over the columns (of each group)."
function activation_gradient!(dz, dd, z, activation = nothing; bias_gradient = nothing, offsets = nothing)
    M, N = size(dd)
    ldim(x) = x === nothing ? Int64(max(M, 1)) : Int64(max(stride(x, 2), M, 1))
    ldb = bias_gradient === nothing || ndims(bias_gradient) == 1 ? Int64(max(M, 1)) : Int64(max(stride(bias_gradient, 2), M, 1))
    desc = GkActivationGradientDesc(sizeof(GkActivationGradientDesc), gk_dtype(eltype(dd)), M, N, ldim(dd), ldim(z), ldim(dz), ldb,
                                    gk_activation(activation), offsets === nothing ? 1 : length(offsets) - 1,
                                    offsets === nothing ? 5 : gk_dtype(eltype(offsets)), 0, ptr_or_null(offsets))
    bytes = Ref{Int64}(0)
    bias_gradient === nothing ||
        gk_check(ccall((:gk_activation_gradient_query, libgk), Cint, (Ptr{Cvoid}, Ref{GkActivationGradientDesc}, Ref{Int64}), gk_handle(), desc, bytes))
    ws = bytes[] > 0 ? reinterpret(CuPtr{Cvoid}, pointer(lent_workspace(bytes[]))) : CU_NONE
    gk_check(ccall((:gk_activation_gradient, libgk), Cint,
                   (Ptr{Cvoid}, Ref{GkActivationGradientDesc}, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{Cvoid}, Int64, Ptr{Cvoid}),
                   gk_handle(), desc, ptr_or_null(dd), ptr_or_null(z), ptr_or_null(dz), ptr_or_null(bias_gradient), ws, bytes[], CUDA.stream().handle))
    dz
end
